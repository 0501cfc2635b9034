// Tokens sorted by expert and back, for rows of bf16, fp16 or fp32.
//
//   order    a stable counting sort of the (token, choice) pairs by local expert:
//            per-chunk histograms, one scan over chunks and experts, and each
//            pair's row = its expert's segment start + its pairs in earlier chunks
//            + its pairs earlier in the chunk
//   gather   rows[r] = x[token of row_pair[r]], zeros for a row without a pair
//   combine  out[t] = sum_k w[t,k] rows[pair_row[t,k]], k ascending, fp32, one
//            rounding; without weights it is the gradient of the gather
//   combine_backward  drows[r] = w[p] dout[t], dw[t,k] = <dout[t], rows[pair_row[t,k]]>
//
// The reference sorts and combines inside its kernel() only, for its own FP8
// layer and without gradients (solution/triton/kernel.py:46-82, :1920-1925).
#include "kf_elem.cuh"
#include "kf_internal.cuh"

namespace kf {
namespace {

constexpr int kOrderThreads = 256;
constexpr int kOrderChunk = 1024;   // pairs per chunk of the counting sort
constexpr int kRowThreads = 256;
constexpr int kWarps = kRowThreads / 32;

__device__ __forceinline__ int local_expert(int id, int offset, int E) {
  const unsigned le = static_cast<unsigned>(id) - static_cast<unsigned>(offset);
  return id >= 0 && le < static_cast<unsigned>(E) ? static_cast<int>(le) : -1;
}

__global__ void __launch_bounds__(kOrderThreads) order_hist_kernel(const int32_t* __restrict__ ids, int n, int E,
                                                                   int offset, int32_t* __restrict__ hist) {
  __shared__ int32_t h[kEG];
  h[threadIdx.x] = 0;
  __syncthreads();
  const int p0 = blockIdx.x * kOrderChunk;
  for (int p = p0 + threadIdx.x; p < min(n, p0 + kOrderChunk); p += kOrderThreads) {
    const int e = local_expert(ids[p], offset, E);
    if (e >= 0) atomicAdd(&h[e], 1);
  }
  __syncthreads();
  if (threadIdx.x < E) hist[static_cast<size_t>(blockIdx.x) * E + threadIdx.x] = h[threadIdx.x];
}

// One block; thread e owns expert e.  hist[c][e] becomes the row of the first pair of expert e in chunk c.
__global__ void __launch_bounds__(kOrderThreads) order_scan_kernel(int32_t* __restrict__ hist, int nchunk, int E,
                                                                   int align, int rows, int32_t* __restrict__ counts,
                                                                   int32_t* __restrict__ starts) {
  __shared__ int64_t scan[kOrderThreads];
  const int e = threadIdx.x;
  int run = 0;
  if (e < E)
    for (int c = 0; c < nchunk; ++c) run += hist[static_cast<size_t>(c) * E + e];
  const int64_t padded = (static_cast<int64_t>(run) + align - 1) / align * align;
  scan[e] = padded;
  __syncthreads();
  for (int off = 1; off < kOrderThreads; off <<= 1) {
    const int64_t v = e >= off ? scan[e - off] : 0;
    __syncthreads();
    scan[e] += v;
    __syncthreads();
  }
  if (e >= E) return;
  const int64_t start = scan[e] - padded;
  counts[e] = run;
  starts[e] = static_cast<int32_t>(start < rows ? start : rows);
  if (e == E - 1) starts[E] = static_cast<int32_t>(scan[e] < rows ? scan[e] : rows);
  // past the buffer every pair is dropped, so a start there only has to stay past it
  int at = static_cast<int32_t>(start < rows ? start : rows);
  for (int c = 0; c < nchunk; ++c) {
    const int k = hist[static_cast<size_t>(c) * E + e];
    hist[static_cast<size_t>(c) * E + e] = at;
    at = at > rows - k ? rows : at + k;
  }
}

__global__ void __launch_bounds__(kOrderThreads) order_place_kernel(const int32_t* __restrict__ ids, int n, int E,
                                                                    int offset, const int32_t* __restrict__ first,
                                                                    int rows, int32_t* __restrict__ pair_row,
                                                                    int32_t* __restrict__ row_pair) {
  __shared__ int32_t at[kEG];                          // next row of each expert
  __shared__ int32_t warp_count[kOrderThreads / 32][kEG];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  at[tid] = tid < E ? first[static_cast<size_t>(blockIdx.x) * E + tid] : 0;
  const int p0 = blockIdx.x * kOrderChunk;
  for (int r = 0; r < kOrderChunk; r += kOrderThreads) {
    for (int w = 0; w < kOrderThreads / 32; ++w) warp_count[w][tid] = 0;
    __syncthreads();
    const int p = p0 + r + tid;
    const int e = p < n ? local_expert(ids[p], offset, E) : -1;
    const unsigned same = __match_any_sync(0xffffffffu, e);
    const int before = __popc(same & ((1u << lane) - 1u));
    if (e >= 0 && before == 0) warp_count[warp][e] = __popc(same);
    __syncthreads();
    int row = -1;
    if (e >= 0) {
      row = at[e] + before;
      for (int w = 0; w < warp; ++w) row += warp_count[w][e];
    }
    if (p < n) {
      if (row >= rows) row = -1;
      pair_row[p] = row;
      if (row >= 0) row_pair[row] = p;
    }
    __syncthreads();
    int sum = 0;
    for (int w = 0; w < kOrderThreads / 32; ++w) sum += warp_count[w][tid];
    at[tid] += sum;
    __syncthreads();
  }
}

// One warp per row of the buffer, 16-byte (or single-element) accesses.
template <typename T, bool kVec>
__global__ void __launch_bounds__(kRowThreads) gather_tokens_kernel(const T* __restrict__ x, int64_t stride, int T_,
                                                                    int K, int H, const int32_t* __restrict__ row_pair,
                                                                    int rows, T* __restrict__ out) {
  const int lane = threadIdx.x & 31;
  const int64_t r = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (r >= rows) return;
  const int p = row_pair[r];
  const int t = p >= 0 ? p / K : -1;
  const bool live = t >= 0 && t < T_;
  const T* src = x + (live ? static_cast<int64_t>(t) * stride : 0);
  T* dst = out + r * H;
  for (int c = 0; c < H; c += kSlice) {
    const Raw8<T> v = load_raw8<T, kVec>(src + c, live ? H - c : 0, lane);
    store_raw8<T, kVec>(dst + c, H - c, lane, v);
  }
}

// One warp per (token, slice of 256 columns); lane k of the warp holds pair k's row and weight.
template <typename T, bool kVec>
__global__ void __launch_bounds__(kRowThreads) combine_kernel(const T* __restrict__ rows, int64_t stride, int R,
                                                              const int32_t* __restrict__ pair_row,
                                                              const float* __restrict__ weight, int T_, int K, int H,
                                                              T* __restrict__ out) {
  const int lane = threadIdx.x & 31;
  const int slices = (H + kSlice - 1) / kSlice;
  const int64_t u = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int64_t t = u / slices;
  if (t >= T_) return;
  const int c = static_cast<int>(u % slices) * kSlice;
  int my_row = -1;
  float my_w = 1.f;
  if (lane < K) {
    my_row = pair_row[t * K + lane];
    if (my_row >= R) my_row = -1;
    if (weight) my_w = weight[t * K + lane];
  }
  float acc[8] = {};
  for (int k = 0; k < K; ++k) {
    const int row = __shfl_sync(0xffffffffu, my_row, k);
    const float w = __shfl_sync(0xffffffffu, my_w, k);
    if (row < 0) continue;
    float v[8];
    to_floats(load_raw8<T, kVec>(rows + static_cast<int64_t>(row) * stride + c, H - c, lane), v);
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = fmaf(w, v[j], acc[j]);
  }
  store_raw8<T, kVec>(out + t * H + c, H - c, lane, from_floats<T>(acc));
}

// Blocks [0, T): one per token.  Blocks past T: rows without a pair are zeroed.
template <typename T, bool kVec>
__global__ void __launch_bounds__(kRowThreads) combine_backward_kernel(
    const T* __restrict__ dout, const T* __restrict__ rows, int64_t stride, int R, const int32_t* __restrict__ pair_row,
    const int32_t* __restrict__ row_pair, const float* __restrict__ weight, int T_, int K, int H, T* __restrict__ drows,
    float* __restrict__ dweight) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (blockIdx.x >= T_) {
    if (!drows) return;
    const int64_t r = static_cast<int64_t>(blockIdx.x - T_) * kWarps + warp;
    if (r >= R) return;
    const int p = row_pair[r];
    if (p >= 0 && p < static_cast<int64_t>(T_) * K) return;
    Raw8<T> z = {};
    for (int c = 0; c < H; c += kSlice) store_raw8<T, kVec>(drows + r * H + c, H - c, lane, z);
    return;
  }
  __shared__ float part[kWarps][KF_SORT_MAX_TOP_K];
  const int64_t t = blockIdx.x;
  int my_row = -1;
  float my_w = 1.f;
  if (lane < K) {
    my_row = pair_row[t * K + lane];
    if (my_row >= R) my_row = -1;
    if (weight) my_w = weight[t * K + lane];
  }
  for (int k = 0; k < K; ++k) {
    const int row = __shfl_sync(0xffffffffu, my_row, k);
    const float w = __shfl_sync(0xffffffffu, my_w, k);
    float dot = 0.f;
    if (row >= 0) {
      for (int c = warp * kSlice; c < H; c += kWarps * kSlice) {
        float g[8];
        to_floats(load_raw8<T, kVec>(dout + t * H + c, H - c, lane), g);
        if (dweight) {
          float v[8];
          to_floats(load_raw8<T, kVec>(rows + static_cast<int64_t>(row) * stride + c, H - c, lane), v);
#pragma unroll
          for (int j = 0; j < 8; ++j) dot = fmaf(g[j], v[j], dot);
        }
        if (drows) {
#pragma unroll
          for (int j = 0; j < 8; ++j) g[j] *= w;
          store_raw8<T, kVec>(drows + static_cast<int64_t>(row) * H + c, H - c, lane, from_floats<T>(g));
        }
      }
    }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, off);
    if (lane == 0) part[warp][k] = dot;
  }
  if (!dweight) return;
  __syncthreads();
  if (threadIdx.x < K) {
    float s = 0.f;
    for (int w = 0; w < kWarps; ++w) s += part[w][threadIdx.x];
    dweight[t * K + threadIdx.x] = s;
  }
}

inline unsigned blocks(int64_t items, int per) { return static_cast<unsigned>((items + per - 1) / per); }

bool valid_shape(int32_t T, int32_t K, int64_t H, int32_t dtype) {
  return valid_tokens(T) && K >= 1 && K <= KF_SORT_MAX_TOP_K && H >= 1 && H <= KF_SORT_MAX_WIDTH && valid_dtype(dtype);
}

// Launch checks shared by the entry points: grids of one block per token or per few rows stay below 2^31.
int ready() {
  int sms = 0;
  return device_ready(&sms);
}

}  // namespace
}  // namespace kf

using namespace kf;

extern "C" {

size_t kf_sort_workspace_bytes(int32_t num_tokens, int32_t top_k, int32_t num_experts) {
  if (!valid_tokens(num_tokens) || top_k < 1 || top_k > KF_SORT_MAX_TOP_K || num_experts < 1 || num_experts > kEG)
    return 0;
  const int64_t n = static_cast<int64_t>(num_tokens) * top_k;
  const int64_t nchunk = (n + kOrderChunk - 1) / kOrderChunk;
  return static_cast<size_t>(nchunk > 0 ? nchunk : 1) * num_experts * sizeof(int32_t);
}

int kf_sort_tokens(const void* x, int32_t dtype, int64_t x_stride, const int32_t* topk_idx, int32_t num_tokens,
                   int32_t top_k, int32_t width, int32_t num_experts, int32_t expert_offset, int32_t row_align,
                   int32_t num_rows, void* rows, int32_t* pair_row, int32_t* row_pair, int32_t* counts,
                   int32_t* starts, void* workspace, size_t workspace_bytes, void* stream) {
  if (!valid_shape(num_tokens, top_k, width, dtype) || x_stride < 0) return KF_ERR_INVALID_ARGUMENT;
  if (num_experts < 1 || num_experts > kEG || expert_offset < 0 || expert_offset + num_experts > kEG)
    return KF_ERR_INVALID_ARGUMENT;
  if (row_align < 1 || row_align > KF_SORT_MAX_ALIGN || num_rows < 0 || num_rows > KF_SORT_MAX_ROWS ||
      num_rows % row_align)
    return KF_ERR_INVALID_ARGUMENT;
  if (!counts || !starts || (num_tokens > 0 && (!x || !topk_idx || !pair_row)) || (num_rows > 0 && (!rows || !row_pair)))
    return KF_ERR_INVALID_ARGUMENT;
  const size_t need = kf_sort_workspace_bytes(num_tokens, top_k, num_experts);
  if (!workspace) return KF_ERR_INVALID_ARGUMENT;
  if (workspace_bytes < need) return KF_ERR_WORKSPACE_TOO_SMALL;
  const int rc = ready();
  if (rc != KF_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int n = num_tokens * top_k;
  const int nchunk = (n + kOrderChunk - 1) / kOrderChunk;
  int32_t* hist = static_cast<int32_t*>(workspace);
  if (num_rows && cudaMemsetAsync(row_pair, 0xff, static_cast<size_t>(num_rows) * 4, s) != cudaSuccess) return KF_ERR_CUDA;
  if (nchunk) order_hist_kernel<<<nchunk, kOrderThreads, 0, s>>>(topk_idx, n, num_experts, expert_offset, hist);
  order_scan_kernel<<<1, kOrderThreads, 0, s>>>(hist, nchunk, num_experts, row_align, num_rows, counts, starts);
  if (nchunk)
    order_place_kernel<<<nchunk, kOrderThreads, 0, s>>>(topk_idx, n, num_experts, expert_offset, hist, num_rows,
                                                        pair_row, row_pair);
  if (cudaGetLastError() != cudaSuccess) return KF_ERR_CUDA;
  if (num_rows == 0) return KF_OK;
  const bool vec = vec_rows(x, x_stride, width, dtype) && vec_rows(rows, width, width, dtype);
  return dispatch_rows(dtype, vec, [&](auto t, auto v) {
           using E = std::remove_const_t<std::remove_pointer_t<decltype(t)>>;
           gather_tokens_kernel<E, decltype(v)::value><<<blocks(num_rows, kWarps), kRowThreads, 0, s>>>(
               static_cast<const E*>(x), x_stride, num_tokens, top_k, width, row_pair, num_rows, static_cast<E*>(rows));
           return cudaGetLastError();
         }) == cudaSuccess
             ? KF_OK
             : KF_ERR_CUDA;
}

int kf_combine_tokens(const void* rows, int32_t dtype, int64_t rows_stride, int32_t num_rows, const int32_t* pair_row,
                      const float* topk_weight, int32_t num_tokens, int32_t top_k, int32_t width, void* output,
                      void* stream) {
  if (!valid_shape(num_tokens, top_k, width, dtype) || num_rows < 0 || num_rows > KF_SORT_MAX_ROWS || rows_stride < 0)
    return KF_ERR_INVALID_ARGUMENT;
  if (num_tokens == 0) return KF_OK;
  if (!pair_row || !output || (num_rows > 0 && !rows)) return KF_ERR_INVALID_ARGUMENT;
  const int rc = ready();
  if (rc != KF_OK) return rc;
  const bool vec = vec_rows(rows, rows_stride, width, dtype) && vec_rows(output, width, width, dtype);
  const int64_t units = static_cast<int64_t>(num_tokens) * ((width + kSlice - 1) / kSlice);
  return dispatch_rows(dtype, vec, [&](auto t, auto v) {
           using E = std::remove_const_t<std::remove_pointer_t<decltype(t)>>;
           combine_kernel<E, decltype(v)::value><<<blocks(units, kWarps), kRowThreads, 0, static_cast<cudaStream_t>(stream)>>>(
               static_cast<const E*>(rows), rows_stride, num_rows, pair_row, topk_weight, num_tokens, top_k, width,
               static_cast<E*>(output));
           return cudaGetLastError();
         }) == cudaSuccess
             ? KF_OK
             : KF_ERR_CUDA;
}

int kf_combine_backward(const void* grad_output, const void* rows, int32_t dtype, int64_t rows_stride, int32_t num_rows,
                        const int32_t* pair_row, const int32_t* row_pair, const float* topk_weight, int32_t num_tokens,
                        int32_t top_k, int32_t width, void* grad_rows, float* grad_weight, void* stream) {
  if (!valid_shape(num_tokens, top_k, width, dtype) || num_rows < 0 || num_rows > KF_SORT_MAX_ROWS || rows_stride < 0)
    return KF_ERR_INVALID_ARGUMENT;
  if (num_tokens > 0 && (!grad_output || !pair_row)) return KF_ERR_INVALID_ARGUMENT;
  if (grad_weight && num_rows > 0 && !rows) return KF_ERR_INVALID_ARGUMENT;
  if (grad_rows && num_rows > 0 && !row_pair) return KF_ERR_INVALID_ARGUMENT;
  const int rc = ready();
  if (rc != KF_OK) return rc;
  const bool vec = vec_rows(grad_output, width, width, dtype) && (!grad_weight || vec_rows(rows, rows_stride, width, dtype)) &&
                   (!grad_rows || vec_rows(grad_rows, width, width, dtype));
  const unsigned grid = num_tokens + (grad_rows ? blocks(num_rows, kWarps) : 0u);
  if (grid == 0) return KF_OK;
  return dispatch_rows(dtype, vec, [&](auto t, auto v) {
           using E = std::remove_const_t<std::remove_pointer_t<decltype(t)>>;
           combine_backward_kernel<E, decltype(v)::value><<<grid, kRowThreads, 0, static_cast<cudaStream_t>(stream)>>>(
               static_cast<const E*>(grad_output), static_cast<const E*>(rows), rows_stride, num_rows, pair_row, row_pair,
               topk_weight, num_tokens, top_k, width, static_cast<E*>(grad_rows), grad_weight);
           return cudaGetLastError();
         }) == cudaSuccess
             ? KF_OK
             : KF_ERR_CUDA;
}

}  // extern "C"
