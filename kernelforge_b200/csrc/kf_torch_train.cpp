// Torch side of the training operators (kf_moe.h, "training"): argument checks,
// outputs and scratch from torch's caching allocator, launches on the current
// stream of the tensors' device, and the autograd functions.  Scratch is taken per
// call, so calls on several streams and captured graphs never share any.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <string>
#include <tuple>

#include "kf_moe.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == KF_OK, what, " failed: ", kf_moe_error_string(rc), " (code ", rc, ")");
}

void check_cuda(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor on a B200 (sm_100a); no CPU fallback");
}

int dtype_of(at::ScalarType type, const char* name) {
  switch (type) {
    case at::kBFloat16: return KF_DTYPE_BF16;
    case at::kHalf: return KF_DTYPE_F16;
    case at::kFloat: return KF_DTYPE_F32;
    default: TORCH_CHECK(false, name, " must be bfloat16, float16 or float32, got ", type);
  }
}
int dtype_of(const Tensor& t, const char* name) { return dtype_of(t.scalar_type(), name); }

// A 2-D row tensor of a supported type whose rows are dense (a copy is made of any other).
Tensor expect_rows(const Tensor& t, const char* name) {
  check_cuda(t, name);
  dtype_of(t, name);
  TORCH_CHECK(t.dim() == 2, name, " must be 2-dimensional, got shape ", t.sizes());
  TORCH_CHECK(t.size(1) >= 1 && t.size(1) <= KF_SORT_MAX_WIDTH, name, " must have 1 to ", KF_SORT_MAX_WIDTH,
              " columns, got ", t.size(1));
  return t.stride(1) == 1 || t.size(1) == 1 ? t : t.contiguous();
}

Tensor expect(const Tensor& t, const char* name, at::ScalarType dtype, at::IntArrayRef shape, const at::Device& dev) {
  TORCH_CHECK(t.scalar_type() == dtype, name, " must be ", dtype, ", got ", t.scalar_type());
  TORCH_CHECK(t.sizes() == shape, name, " must have shape ", shape, ", got ", t.sizes());
  TORCH_CHECK(t.device() == dev, name, " is on ", t.device(), ", expected ", dev);
  return t.contiguous();
}

void check_tokens(int64_t T, const char* what) {
  TORCH_CHECK(T <= KF_MOE_MAX_TOKENS, what, " ", T, " above ", KF_MOE_MAX_TOKENS);
}
void check_num_rows(int64_t R, const char* what) {
  TORCH_CHECK(R <= KF_SORT_MAX_ROWS, what, " ", R, " above ", KF_SORT_MAX_ROWS);
}

void* stream_of(const at::Device& dev) { return at::cuda::getCurrentCUDAStream(dev.index()).stream(); }

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// An output or scratch tensor, straight from the caching allocator: at decode sizes the
// dispatcher's share of at::empty (half a microsecond a tensor) is a tenth of a call.
Tensor new_tensor(at::IntArrayRef shape, at::ScalarType dtype, const at::Device& dev) {
  return Tensor(at::detail::empty_cuda(shape, dtype, dev, std::nullopt));
}

bool wants_grad(const Tensor& t) { return at::GradMode::is_enabled() && t.requires_grad(); }

// During a stream capture a leaf whose gradient accumulator lives on the default stream
// -- an eager graph of the same leaf, made there, is still alive -- is refused: the
// backward pass makes that stream wait for the capturing one, which the legacy stream
// cannot, and invalidates the capture inside the autograd engine.  Any other stream joins
// the capture by waiting (a warm-up on a side stream whose graph is still alive), unless
// another capture holds it.  `t`: an argument as the caller gave it.
void refuse_shared_leaf(const Tensor& t) {
  if (!t.defined() || !t.is_cuda() || !t.is_leaf() || !wants_grad(t)) return;
  const c10::DeviceIndex dev = t.device().index();
  const at::cuda::CUDAStream now = at::cuda::getCurrentCUDAStream(dev);
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  unsigned long long capture = 0, other = 0;
  if (cudaStreamGetCaptureInfo(now.stream(), &cap, &capture) != cudaSuccess || cap == cudaStreamCaptureStatusNone) return;
  const auto acc = torch::autograd::impl::try_get_grad_accumulator(t);
  if (!acc || !acc->stream().has_value() || *acc->stream() == now.unwrap()) return;
  const at::cuda::CUDAStream its(*acc->stream());
  bool joins = its != at::cuda::getDefaultCUDAStream(dev);
  if (joins) {
    cap = cudaStreamCaptureStatusNone;
    joins = cudaStreamGetCaptureInfo(its.stream(), &cap, &other) == cudaSuccess &&
            (cap == cudaStreamCaptureStatusNone || (cap == cudaStreamCaptureStatusActive && other == capture));
  }
  TORCH_CHECK(joins,
              "a captured call on a leaf tensor whose eager autograd graph is still alive on the default stream (or in "
              "another capture): release that graph first, or capture a detached copy that requires grad");
}

// The operators have no forward-mode rule.  A tensor that carries a tangent need not require a gradient, so without
// this check it would take the way past the autograd function, and its tangent would be lost without an error.  (The
// tangent is undefined where forward mode is switched off.)
void refuse_tangent(const Tensor& t, const char* what) {
  TORCH_CHECK(!t.defined() || !t._fw_grad(/*level=*/0).defined(), what,
              " has no forward-mode derivative: an argument carries a tangent (torch.autograd.forward_ad)");
}
void refuse_tangent(const std::optional<Tensor>& t, const char* what) {
  if (t.has_value()) refuse_tangent(*t, what);
}

void refuse_double_backward(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, " is not twice differentiable (backward with create_graph=True)");
}

// ------------------------------------------------------------------ order --

struct Order {
  Tensor pair_row, row_pair;
};

// The token order's index tensors as a caller hands them back.
Order expect_order(const Tensor& pair_row, const Tensor& row_pair, const at::Device& dev) {
  TORCH_CHECK(pair_row.dim() == 2 && pair_row.size(1) >= 1 && pair_row.size(1) <= KF_SORT_MAX_TOP_K,
              "order.pair_row must be [T, K] with K from 1 to ", KF_SORT_MAX_TOP_K, ", got shape ", pair_row.sizes());
  TORCH_CHECK(row_pair.dim() == 1, "order.row_pair must be [R], got shape ", row_pair.sizes());
  check_tokens(pair_row.size(0), "number of tokens");
  check_num_rows(row_pair.size(0), "number of rows");
  return Order{expect(pair_row, "order.pair_row", at::kInt, pair_row.sizes(), dev),
               expect(row_pair, "order.row_pair", at::kInt, row_pair.sizes(), dev)};
}

// sum_k weight[t, k] * rows[pair_row[t, k]]; without a weight the gradient of sort_tokens.
Tensor combine_forward(const Tensor& rows, const Tensor& pair_row, const Tensor& weight) {
  const at::Device dev = rows.device();
  c10::cuda::CUDAGuard guard(dev);
  Tensor out = new_tensor({pair_row.size(0), rows.size(1)}, rows.scalar_type(), dev);
  check_rc(kf_combine_tokens(ptr(rows), dtype_of(rows, "rows"), rows.stride(0), static_cast<int32_t>(rows.size(0)),
                             pair_row.const_data_ptr<int32_t>(),
                             weight.defined() ? weight.const_data_ptr<float>() : nullptr,
                             static_cast<int32_t>(pair_row.size(0)), static_cast<int32_t>(pair_row.size(1)),
                             static_cast<int32_t>(rows.size(1)), ptr(out), stream_of(dev)),
           "kf_combine_tokens");
  return out;
}

std::tuple<Tensor, Tensor> combine_backward_impl(const Tensor& grad_out, const Tensor& rows, const Order& order,
                                                 const Tensor& weight, bool need_rows, bool need_weight) {
  const at::Device dev = grad_out.device();
  c10::cuda::CUDAGuard guard(dev);
  const int64_t T = order.pair_row.size(0), K = order.pair_row.size(1), R = order.row_pair.size(0);
  const int64_t H = grad_out.size(1);
  Tensor g = grad_out.contiguous();
  Tensor grad_rows, grad_weight;
  if (need_rows) grad_rows = new_tensor({R, H}, g.scalar_type(), dev);
  if (need_weight) grad_weight = new_tensor({T, K}, at::kFloat, dev);
  check_rc(kf_combine_backward(ptr(g), ptr(rows), dtype_of(g, "grad_output"), rows.defined() ? rows.stride(0) : H,
                               static_cast<int32_t>(R), order.pair_row.const_data_ptr<int32_t>(),
                               order.row_pair.const_data_ptr<int32_t>(),
                               weight.defined() ? weight.const_data_ptr<float>() : nullptr, static_cast<int32_t>(T),
                               static_cast<int32_t>(K), static_cast<int32_t>(H), ptr(grad_rows),
                               need_weight ? grad_weight.data_ptr<float>() : nullptr, stream_of(dev)),
           "kf_combine_backward");
  return {grad_rows, grad_weight};
}

// --------------------------------------------------------------- operators --

struct SortArgs {
  int64_t experts, offset, align, rows;
};

variable_list sort_forward(const Tensor& x, const Tensor& ids, const SortArgs& a) {
  const at::Device dev = x.device();
  c10::cuda::CUDAGuard guard(dev);
  const int64_t T = ids.size(0), K = ids.size(1), H = x.size(1);
  Tensor rows = new_tensor({a.rows, H}, x.scalar_type(), dev);
  Tensor pair_row = new_tensor({T, K}, at::kInt, dev), row_pair = new_tensor({a.rows}, at::kInt, dev),
         counts = new_tensor({a.experts}, at::kInt, dev), starts = new_tensor({a.experts + 1}, at::kInt, dev);
  const size_t need = kf_sort_workspace_bytes(static_cast<int32_t>(T), static_cast<int32_t>(K),
                                              static_cast<int32_t>(a.experts));
  Tensor ws;
  if (need) ws = new_tensor({static_cast<int64_t>(need)}, at::kByte, dev);
  check_rc(kf_sort_tokens(ptr(x), dtype_of(x, "x"), x.stride(0), ids.const_data_ptr<int32_t>(), static_cast<int32_t>(T),
                          static_cast<int32_t>(K), static_cast<int32_t>(H), static_cast<int32_t>(a.experts),
                          static_cast<int32_t>(a.offset), static_cast<int32_t>(a.align), static_cast<int32_t>(a.rows),
                          ptr(rows), pair_row.data_ptr<int32_t>(), row_pair.data_ptr<int32_t>(),
                          counts.data_ptr<int32_t>(), starts.data_ptr<int32_t>(), ptr(ws), need, stream_of(dev)),
           "kf_sort_tokens");
  return {rows, pair_row, row_pair, counts, starts};
}

struct SortFn : public torch::autograd::Function<SortFn> {
  static variable_list forward(AutogradContext* ctx, const Variable& x, const Variable& ids, int64_t experts,
                               int64_t offset, int64_t align, int64_t rows) {
    variable_list out = sort_forward(x, ids, SortArgs{experts, offset, align, rows});
    ctx->set_materialize_grads(false);   // no zeros in place of the integer outputs' gradients
    ctx->mark_non_differentiable({out[1], out[2], out[3], out[4]});
    ctx->save_for_backward({out[1]});
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_double_backward("sort_tokens");
    refuse_tangent(grads[0], "sort_tokens");
    Tensor dx;
    if (grads[0].defined())
      dx = combine_forward(expect_rows(grads[0], "grad of rows"), ctx->get_saved_variables()[0], Tensor());
    return {dx, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> sort_tokens(const Tensor& x_in, const Tensor& topk_idx,
                                                               int64_t num_experts, int64_t expert_offset,
                                                               int64_t row_align, std::optional<int64_t> max_rows) {
  refuse_tangent(x_in, "sort_tokens");
  refuse_shared_leaf(x_in);
  const Tensor x = expect_rows(x_in, "x");
  const int64_t T = x.size(0);
  TORCH_CHECK(topk_idx.dim() == 2 && topk_idx.size(0) == T && topk_idx.size(1) >= 1 &&
                  topk_idx.size(1) <= KF_SORT_MAX_TOP_K,
              "topk_idx must be [", T, ", K] with K from 1 to ", KF_SORT_MAX_TOP_K, ", got shape ", topk_idx.sizes());
  const Tensor ids = expect(topk_idx, "topk_idx", at::kInt, topk_idx.sizes(), x.device());
  check_tokens(T, "number of tokens");
  TORCH_CHECK(num_experts >= 1 && expert_offset >= 0 && num_experts <= KF_MOE_GLOBAL_EXPERTS &&
                  expert_offset <= KF_MOE_GLOBAL_EXPERTS - num_experts,
              "local experts [", expert_offset, ", ", expert_offset + num_experts, ") outside [0, ",
              KF_MOE_GLOBAL_EXPERTS, ")");
  TORCH_CHECK(row_align >= 1 && row_align <= KF_SORT_MAX_ALIGN, "row_align must be 1 to ", KF_SORT_MAX_ALIGN, ", got ",
              row_align);
  const int64_t pairs = T * ids.size(1);
  int64_t rows = (pairs + std::min(pairs, num_experts) * (row_align - 1)) / row_align * row_align;
  if (max_rows.has_value()) {
    TORCH_CHECK(*max_rows >= 0 && *max_rows % row_align == 0, "max_rows must be a multiple of row_align (", row_align,
                ") and not negative, got ", *max_rows);
    rows = *max_rows;
  }
  check_num_rows(rows, "number of rows");
  variable_list o = wants_grad(x) ? SortFn::apply(x, ids, num_experts, expert_offset, row_align, rows)
                                  : sort_forward(x, ids, SortArgs{num_experts, expert_offset, row_align, rows});
  return {o[0], o[1], o[2], o[3], o[4]};
}

Tensor sort_tokens_backward(const Tensor& grad_rows, const Tensor& pair_row, const Tensor& row_pair) {
  refuse_tangent(grad_rows, "sort_tokens_backward");
  const Tensor g = expect_rows(grad_rows, "grad_rows");
  const Order o = expect_order(pair_row, row_pair, g.device());
  TORCH_CHECK(g.size(0) == o.row_pair.size(0), "grad_rows has ", g.size(0), " rows, the order ", o.row_pair.size(0));
  return combine_forward(g, o.pair_row, Tensor());
}

struct CombineFn : public torch::autograd::Function<CombineFn> {
  static Variable forward(AutogradContext* ctx, const Variable& rows, const Variable& pair_row, const Variable& row_pair,
                          const std::optional<Tensor>& topk_weight) {
    const Tensor weight = topk_weight.value_or(Tensor());
    // the rows are needed for the weights' gradient only, the weights for the rows'
    const bool need_w = weight.defined() && weight.requires_grad();
    ctx->save_for_backward({need_w ? rows : Tensor(), pair_row, row_pair, weight});
    return combine_forward(rows, pair_row, weight);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_double_backward("combine_tokens");
    refuse_tangent(grads[0], "combine_tokens");
    Tensor dr, dw;
    if (grads[0].defined()) {
      const auto saved = ctx->get_saved_variables();
      const bool need_rows = ctx->needs_input_grad(0);
      const bool need_weight = saved[3].defined() && ctx->needs_input_grad(3);
      if (need_rows || need_weight)
        std::tie(dr, dw) = combine_backward_impl(expect_rows(grads[0], "grad of the output"), saved[0],
                                                 Order{saved[1], saved[2]}, saved[3], need_rows, need_weight);
    }
    return {dr, Tensor(), Tensor(), dw};
  }
};

Tensor expect_weight(const std::optional<Tensor>& w, const Order& o, const at::Device& dev) {
  return w.has_value() ? expect(*w, "topk_weight", at::kFloat, o.pair_row.sizes(), dev) : Tensor();
}

Tensor combine_tokens(const Tensor& rows_in, const Tensor& pair_row, const Tensor& row_pair,
                      const std::optional<Tensor>& topk_weight) {
  refuse_tangent(rows_in, "combine_tokens");
  refuse_tangent(topk_weight, "combine_tokens");
  refuse_shared_leaf(rows_in);
  if (topk_weight.has_value()) refuse_shared_leaf(*topk_weight);
  const Tensor rows = expect_rows(rows_in, "rows");
  const Order o = expect_order(pair_row, row_pair, rows.device());
  TORCH_CHECK(rows.size(0) == o.row_pair.size(0), "rows has ", rows.size(0), " rows, the order ", o.row_pair.size(0));
  const Tensor w = expect_weight(topk_weight, o, rows.device());
  if (wants_grad(rows) || (w.defined() && wants_grad(w))) 
    return CombineFn::apply(rows, o.pair_row, o.row_pair, w.defined() ? std::optional<Tensor>(w) : std::nullopt);
  return combine_forward(rows, o.pair_row, w);
}

std::tuple<Tensor, Tensor> combine_tokens_backward(const Tensor& grad_output, const Tensor& rows_in,
                                                   const Tensor& pair_row, const Tensor& row_pair,
                                                   const Tensor& topk_weight) {
  for (const Tensor* t : {&grad_output, &rows_in, &topk_weight}) refuse_tangent(*t, "combine_tokens_backward");
  const Tensor g = expect_rows(grad_output, "grad_output");
  const at::Device dev = g.device();
  const Order o = expect_order(pair_row, row_pair, dev);
  const Tensor rows = expect_rows(rows_in, "rows");
  TORCH_CHECK(rows.device() == dev && rows.scalar_type() == g.scalar_type() && rows.size(1) == g.size(1) &&
                  rows.size(0) == o.row_pair.size(0),
              "rows must be ", g.scalar_type(), " [", o.row_pair.size(0), ", ", g.size(1), "] on ", dev, ", got ",
              rows.scalar_type(), " ", rows.sizes(), " on ", rows.device());
  TORCH_CHECK(g.size(0) == o.pair_row.size(0), "grad_output has ", g.size(0), " rows, the order ", o.pair_row.size(0),
              " tokens");
  return combine_backward_impl(g, rows, o, expect_weight(topk_weight, o, dev), true, true);
}

Tensor route_backward(const Tensor& routing_logits, const Tensor& topk_idx, const Tensor& grad_weight,
                      double routed_scaling_factor) {
  refuse_tangent(routing_logits, "route_backward");
  refuse_tangent(grad_weight, "route_backward");
  check_cuda(routing_logits, "routing_logits");
  const at::Device dev = routing_logits.device();
  TORCH_CHECK(routing_logits.dim() == 2, "routing_logits must be [T, 256]");
  const int64_t T = routing_logits.size(0);
  check_tokens(T, "number of tokens");
  const Tensor logits = expect(routing_logits, "routing_logits", at::kFloat, {T, KF_MOE_GLOBAL_EXPERTS}, dev);
  const Tensor ids = expect(topk_idx, "topk_idx", at::kInt, {T, KF_MOE_TOP_K}, dev);
  const Tensor g = expect(grad_weight, "grad_weight", at::kFloat, {T, KF_MOE_TOP_K}, dev);
  c10::cuda::CUDAGuard guard(dev);
  Tensor out = new_tensor({T, KF_MOE_GLOBAL_EXPERTS}, at::kFloat, dev);
  check_rc(kf_moe_route_backward(logits.const_data_ptr<float>(), ids.const_data_ptr<int32_t>(),
                                 g.const_data_ptr<float>(), static_cast<int32_t>(T),
                                 static_cast<float>(routed_scaling_factor), out.data_ptr<float>(), stream_of(dev)),
           "kf_moe_route_backward");
  return out;
}

variable_list route_forward(const Tensor& logits, const Tensor& bias, double rsf) {
  const at::Device dev = logits.device();
  c10::cuda::CUDAGuard guard(dev);
  const int64_t T = logits.size(0);
  Tensor ids = new_tensor({T, KF_MOE_TOP_K}, at::kInt, dev);
  Tensor w = new_tensor({T, KF_MOE_TOP_K}, at::kFloat, dev);
  check_rc(kf_moe_route(logits.const_data_ptr<float>(), bias.const_data_ptr(), static_cast<int32_t>(T),
                        static_cast<float>(rsf), ids.data_ptr<int32_t>(), w.data_ptr<float>(), stream_of(dev)),
           "kf_moe_route");
  return {ids, w};
}

struct RouteFn : public torch::autograd::Function<RouteFn> {
  static variable_list forward(AutogradContext* ctx, const Variable& logits, const Variable& bias, double rsf) {
    variable_list out = route_forward(logits, bias, rsf);
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({out[0]});
    ctx->save_for_backward({logits, out[0]});
    ctx->saved_data["rsf"] = rsf;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_double_backward("route");
    Tensor dl;
    if (grads[1].defined()) {
      const auto saved = ctx->get_saved_variables();
      dl = route_backward(saved[0], saved[1], grads[1], ctx->saved_data["rsf"].toDouble());
    }
    return {dl, Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor> route(const Tensor& routing_logits, const Tensor& routing_bias, double rsf) {
  refuse_tangent(routing_logits, "route");
  refuse_shared_leaf(routing_logits);
  check_cuda(routing_logits, "routing_logits");
  const at::Device dev = routing_logits.device();
  TORCH_CHECK(routing_logits.dim() == 2, "routing_logits must be [T, 256]");
  const int64_t T = routing_logits.size(0);
  check_tokens(T, "number of tokens");
  const Tensor logits = expect(routing_logits, "routing_logits", at::kFloat, {T, KF_MOE_GLOBAL_EXPERTS}, dev);
  const Tensor bias = expect(routing_bias.detach().reshape({-1}), "routing_bias", at::kBFloat16,
                             {KF_MOE_GLOBAL_EXPERTS}, dev);
  variable_list o = wants_grad(logits) ? RouteFn::apply(logits, bias, rsf) : route_forward(logits, bias, rsf);
  return {o[0], o[1]};
}

int64_t blocks_of(int64_t width) { return (width + KF_MOE_BLOCK - 1) / KF_MOE_BLOCK; }

std::tuple<Tensor, Tensor> pack8(const Tensor& x_in) {
  const Tensor x = expect_rows(x_in, "x");
  check_num_rows(x.size(0), "number of rows");
  c10::cuda::CUDAGuard guard(x.device());
  Tensor codes = new_tensor({x.size(0), x.size(1)}, at::kFloat8_e4m3fn, x.device());
  Tensor exps = new_tensor({x.size(0), blocks_of(x.size(1))}, at::kByte, x.device());
  check_rc(kf_pack8(ptr(x), dtype_of(x, "x"), x.stride(0), static_cast<int32_t>(x.size(0)),
                    static_cast<int32_t>(x.size(1)), ptr(codes), ptr(exps), stream_of(x.device())),
           "kf_pack8");
  return {codes, exps};
}

// Codes of `width` columns in `parts` halves whose blocks begin at their own first columns.
std::tuple<Tensor, Tensor> expect_kept(const Tensor& codes, const Tensor& exps, int64_t parts) {
  check_cuda(codes, "kept.codes");
  TORCH_CHECK(codes.dim() == 2 && codes.size(1) >= parts && codes.size(1) % parts == 0 &&
                  codes.size(1) <= parts * KF_SORT_MAX_WIDTH,
              "kept.codes must be [R, W]", parts == 2 ? " with an even W" : "", ", got shape ", codes.sizes());
  check_num_rows(codes.size(0), "number of rows");
  return {expect(codes, "kept.codes", at::kFloat8_e4m3fn, codes.sizes(), codes.device()),
          expect(exps, "kept.exponents", at::kByte, {codes.size(0), parts * blocks_of(codes.size(1) / parts)},
                 codes.device())};
}

Tensor restore8(const Tensor& codes_in, const Tensor& exps_in, at::ScalarType dtype,
                const std::optional<Tensor>& pair_row, const std::optional<Tensor>& row_pair) {
  auto [codes, exps] = expect_kept(codes_in, exps_in, 1);
  const at::Device dev = codes.device();
  c10::cuda::CUDAGuard guard(dev);
  int64_t out_rows = codes.size(0), K = 0;
  Tensor pairs, map;
  if (row_pair.has_value()) {
    const Order o = expect_order(*pair_row, *row_pair, dev);
    TORCH_CHECK(o.pair_row.size(0) == codes.size(0), "kept has ", codes.size(0), " rows, the order ",
                o.pair_row.size(0), " tokens");
    pairs = o.pair_row;
    map = o.row_pair;
    out_rows = map.size(0);
    K = o.pair_row.size(1);
  }
  const int code = dtype_of(dtype, "kept.dtype");
  Tensor out = new_tensor({out_rows, codes.size(1)}, dtype, dev);
  check_rc(kf_restore8(ptr(codes), ptr(exps), code, static_cast<int32_t>(codes.size(0)),
                       static_cast<int32_t>(codes.size(1)), pairs.defined() ? pairs.const_data_ptr<int32_t>() : nullptr,
                       map.defined() ? map.const_data_ptr<int32_t>() : nullptr,
                       static_cast<int32_t>(K), static_cast<int32_t>(out_rows), ptr(out), stream_of(dev)),
           "kf_restore8");
  return out;
}

std::tuple<Tensor, Tensor, Tensor> swiglu_forward(const Tensor& h_in, bool keep) {
  const Tensor h = expect_rows(h_in, "h");
  TORCH_CHECK(h.size(1) % 2 == 0, "h must be [R, 2 I] = [up | gate], got shape ", h.sizes());
  check_num_rows(h.size(0), "number of rows");
  const int64_t R = h.size(0), I = h.size(1) / 2;
  c10::cuda::CUDAGuard guard(h.device());
  Tensor act = new_tensor({R, I}, h.scalar_type(), h.device());
  Tensor codes, exps;
  if (keep) {
    codes = new_tensor({R, 2 * I}, at::kFloat8_e4m3fn, h.device());
    exps = new_tensor({R, 2 * blocks_of(I)}, at::kByte, h.device());
  }
  check_rc(kf_swiglu_pack8(ptr(h), dtype_of(h, "h"), h.stride(0), static_cast<int32_t>(R), static_cast<int32_t>(I),
                           ptr(act), ptr(codes), ptr(exps), stream_of(h.device())),
           "kf_swiglu_pack8");
  return {act, codes, exps};
}

std::tuple<Tensor, Tensor, Tensor> swiglu_pack8(const Tensor& h) { return swiglu_forward(h, true); }

std::tuple<Tensor, Tensor> swiglu_backward8(const Tensor& codes_in, const Tensor& exps_in, const Tensor& grad_act,
                                            bool need_act) {
  refuse_tangent(grad_act, "swiglu_backward8");
  auto [codes, exps] = expect_kept(codes_in, exps_in, 2);
  const Tensor g = expect_rows(grad_act, "grad_act");
  const int64_t R = codes.size(0), I = codes.size(1) / 2;
  TORCH_CHECK(g.device() == codes.device() && g.size(0) == R && g.size(1) == I, "grad_act must be [", R, ", ", I,
              "] on ", codes.device(), ", got ", g.sizes(), " on ", g.device());
  c10::cuda::CUDAGuard guard(g.device());
  Tensor grad_h = new_tensor({R, 2 * I}, g.scalar_type(), g.device()), act;
  if (need_act) act = new_tensor({R, I}, g.scalar_type(), g.device());
  check_rc(kf_swiglu_backward8(ptr(codes), ptr(exps), ptr(g), dtype_of(g, "grad_act"), g.stride(0),
                               static_cast<int32_t>(R), static_cast<int32_t>(I), ptr(grad_h), ptr(act),
                               stream_of(g.device())),
           "kf_swiglu_backward8");
  return {grad_h, act};
}

struct SwigluFn : public torch::autograd::Function<SwigluFn> {
  static Variable forward(AutogradContext* ctx, const Variable& h) {
    auto [act, codes, exps] = swiglu_pack8(h);
    ctx->save_for_backward({codes, exps});
    return act;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_double_backward("swiglu");
    if (!grads[0].defined()) return {Tensor()};
    const auto saved = ctx->get_saved_variables();
    return {std::get<0>(swiglu_backward8(saved[0], saved[1], grads[0], false))};
  }
};

Tensor swiglu(const Tensor& h) {
  refuse_tangent(h, "swiglu");
  refuse_shared_leaf(h);
  if (wants_grad(h)) return SwigluFn::apply(h);
  return std::get<0>(swiglu_forward(h, false));
}

}  // namespace

void register_train(pybind11::module_& m) {
  m.def("route", &route, "routing, differentiable in the logits (kf_moe_route, kf_moe_route_backward)");
  m.def("route_backward", &route_backward, "gradient of the routing weights (kf_moe_route_backward)");
  m.def("sort_tokens", &sort_tokens, "tokens' rows in expert order (kf_sort_tokens)");
  m.def("sort_tokens_backward", &sort_tokens_backward, "gradient of sort_tokens (kf_combine_tokens)");
  m.def("combine_tokens", &combine_tokens, "weighted sum of the experts' rows per token (kf_combine_tokens)");
  m.def("combine_tokens_backward", &combine_tokens_backward, "gradients of combine_tokens (kf_combine_backward)");
  m.def("pack8", &pack8, "rows in 8 bits (kf_pack8)");
  m.def("restore8", &restore8, "rows back from 8 bits (kf_restore8)");
  m.def("swiglu", &swiglu, "SwiGLU whose input is kept in 8 bits");
  m.def("swiglu_pack8", &swiglu_pack8, "SwiGLU and its input in 8 bits (kf_swiglu_pack8)");
  m.def("swiglu_backward8", &swiglu_backward8, "gradient of SwiGLU from its 8-bit input (kf_swiglu_backward8)");
}
