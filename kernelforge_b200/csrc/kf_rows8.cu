// Rows kept in 8 bits for the backward pass, and SwiGLU whose input is kept so.
//
// Per row and 128 columns, e is the smallest integer >= -126 with max|x| <= 448 * 2^e
// over the block's finite values; an element's code is e4m3(x * 2^-e), rounded to
// nearest even, and stands for code * 2^e.  A power of two makes both products
// exact, so each value is rounded once, by at most 2^-4 of itself (or 2^-10 * 2^e
// below the smallest normal code), and the result does not depend on how a division
// was rounded; the scale takes one byte (e + 127) per 128 columns.  A value that is
// not finite is kept as NaN, and its block's scale comes from the others.  Where
// 256 * 2^e is beyond the type's largest number the codes end at 240, so that
// restoring never makes an infinity.
//
// (The layer's input format, quantize_rows_kernel, has fp32 scales absmax / 448 as
// the reference fixes them, solution/triton/kernel.py:126-141, and no way back.)
#include <cuda_fp8.h>

#include "kf_elem.cuh"
#include "kf_fp8.cuh"
#include "kf_internal.cuh"

namespace kf {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

template <typename T>
constexpr int kTopExponent = 120;   // 256 * 2^120 = 2^128 is beyond bf16 and fp32
template <>
constexpr int kTopExponent<__half> = 8;   // 256 * 2^8 = 65536 is beyond fp16

__device__ __forceinline__ float pow2(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// Smallest e >= -126 with amax <= 448 * 2^e = 1.75 * 2^(e+8), amax finite and not negative.
__device__ __forceinline__ int block_exponent(uint32_t amax_bits) {
  const int e = static_cast<int>(amax_bits >> 23) - 135 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < -126 ? -126 : e;
}

// A slice of 256 columns = two blocks.  The vector form has a block per half-warp,
// the other form every lane in both (elements 0..3 and 4..7).
template <bool kVec>
__device__ __forceinline__ void block_max(const uint32_t (&m)[2], uint32_t (&out)[2]) {
  if (kVec) {
    uint32_t v = max(m[0], m[1]);
#pragma unroll
    for (int off = 8; off >= 1; off >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, off));
    out[0] = out[1] = v;
  } else {
    out[0] = __reduce_max_sync(0xffffffffu, m[0]);
    out[1] = __reduce_max_sync(0xffffffffu, m[1]);
  }
}

// Codes (byte j = element j) and exponents of this lane's eight elements.
template <typename T, bool kVec>
__device__ __forceinline__ uint2 encode8(const float (&v)[8], int (&e)[2]) {
  uint32_t m[2] = {0u, 0u};
#pragma unroll
  for (int j = 0; j < 8; ++j) m[j >> 2] = max(m[j >> 2], __float_as_uint(v[j]) & 0x7fffffffu);
  uint32_t a[2];
  block_max<kVec>(m, a);
  const bool odd = max(a[0], a[1]) >= 0x7f800000u;
  if (__any_sync(0xffffffffu, odd)) {   // a value that is not finite: the scale comes from the others
    m[0] = m[1] = 0u;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t b = __float_as_uint(v[j]) & 0x7fffffffu;
      if (b < 0x7f800000u) m[j >> 2] = max(m[j >> 2], b);
    }
    block_max<kVec>(m, a);
  }
  e[0] = block_exponent(a[0]);
  e[1] = block_exponent(a[1]);
  const float inv[2] = {pow2(-e[0]), pow2(-e[1])};
  float q[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) q[j] = v[j] * inv[j >> 2];
  if (e[0] == kTopExponent<T> || e[1] == kTopExponent<T>) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (e[j >> 2] == kTopExponent<T>) q[j] = fminf(fmaxf(q[j], -240.f), 240.f);
  }
  if (odd) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if ((__float_as_uint(v[j]) & 0x7fffffffu) >= 0x7f800000u) q[j] = __uint_as_float(0x7fffffffu);
  }
  return make_uint2(pack_fp8x4(q[0], q[1], q[2], q[3]), pack_fp8x4(q[4], q[5], q[6], q[7]));
}

template <bool kVec>
__device__ __forceinline__ void store_codes(uint8_t* __restrict__ slice, int n, int lane, uint2 c) {
  if (kVec) {
    if (lane * 8 < n) *reinterpret_cast<uint2*>(slice + lane * 8) = c;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (lane + 32 * j < n) slice[lane + 32 * j] = static_cast<uint8_t>((j < 4 ? c.x : c.y) >> (8 * (j & 3)));
  }
}

template <bool kVec>
__device__ __forceinline__ uint2 load_codes(const uint8_t* __restrict__ slice, int n, int lane) {
  uint2 c = make_uint2(0u, 0u);
  if (kVec) {
    if (lane * 8 < n) c = __ldg(reinterpret_cast<const uint2*>(slice + lane * 8));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (lane + 32 * j < n) (j < 4 ? c.x : c.y) |= static_cast<uint32_t>(__ldg(slice + lane + 32 * j)) << (8 * (j & 3));
  }
  return c;
}

// The slice's one or two exponent bytes.
template <bool kVec>
__device__ __forceinline__ void store_exponents(uint8_t* __restrict__ exps, int n, int lane, const int (&e)[2]) {
  if (kVec) {
    if ((lane & 15) == 0 && (lane >> 4) * kBlk < n) exps[lane >> 4] = static_cast<uint8_t>(e[0] + 127);
  } else {
    if (lane < 2 && lane * kBlk < n) exps[lane] = static_cast<uint8_t>(e[lane] + 127);
  }
}

// The values of eight codes (in [0, 448], exact) times their blocks' scales.
template <bool kVec>
__device__ __forceinline__ void decode8(uint2 c, const uint8_t* __restrict__ exps, int n, int lane, float (&v)[8]) {
  float s[2];
  if (kVec) {
    const int b = lane >> 4;
    s[0] = s[1] = b * kBlk < n ? __uint_as_float(static_cast<uint32_t>(__ldg(exps + b)) << 23) : 0.f;
  } else {
    s[0] = __uint_as_float(static_cast<uint32_t>(__ldg(exps)) << 23);
    s[1] = kBlk < n ? __uint_as_float(static_cast<uint32_t>(__ldg(exps + 1)) << 23) : 0.f;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t w = (j < 2 ? c.x : c.y) >> (16 * (j & 1));
    const float2 f = fp8x2_to_float2(static_cast<__nv_fp8x2_storage_t>(w & 0xffffu));
    v[2 * j] = f.x * s[j >> 1];
    v[2 * j + 1] = f.y * s[j >> 1];
  }
}

__device__ __forceinline__ float sigmoid(float x) { return 1.0f / (1.0f + expf(-x)); }

// One warp per (row, slice).
template <typename T, bool kVec>
__global__ void __launch_bounds__(kThreads) pack8_kernel(const T* __restrict__ x, int64_t stride, int R, int W,
                                                         uint8_t* __restrict__ codes, uint8_t* __restrict__ exps) {
  const int lane = threadIdx.x & 31;
  const int slices = (W + kSlice - 1) / kSlice, nb = (W + kBlk - 1) / kBlk;
  const int64_t u = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int64_t r = u / slices;
  if (r >= R) return;
  const int c = static_cast<int>(u % slices) * kSlice, n = W - c;
  float v[8];
  to_floats(load_raw8<T, kVec>(x + r * stride + c, n, lane), v);
  int e[2];
  const uint2 q = encode8<T, kVec>(v, e);
  store_codes<kVec>(codes + r * W + c, n, lane, q);
  store_exponents<kVec>(exps + r * nb + c / kBlk, n, lane, e);
}

// One warp per (row, slice); with row_pair, output row i is the row of pair row_pair[i] (zeros if it has none).
template <typename T, bool kVec>
__global__ void __launch_bounds__(kThreads) restore8_kernel(const uint8_t* __restrict__ codes,
                                                            const uint8_t* __restrict__ exps, int src_rows, int W,
                                                            const int32_t* __restrict__ row_pair, int K, int R,
                                                            T* __restrict__ out) {
  const int lane = threadIdx.x & 31;
  const int slices = (W + kSlice - 1) / kSlice, nb = (W + kBlk - 1) / kBlk;
  const int64_t u = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int64_t r = u / slices;
  if (r >= R) return;
  const int c = static_cast<int>(u % slices) * kSlice, n = W - c;
  int64_t src = r;
  if (row_pair) {
    const int p = row_pair[r];
    src = p >= 0 ? p / K : -1;
  }
  float v[8] = {};
  if (src >= 0 && src < src_rows)
    decode8<kVec>(load_codes<kVec>(codes + src * W + c, n, lane), exps + src * nb + c / kBlk, n, lane, v);
  store_raw8<T, kVec>(out + r * W + c, n, lane, from_floats<T>(v));
}

// h = [up | gate]: act = up * silu(gate), and h kept in 8 bits (each half's blocks begin at its own column 0).
template <typename T, bool kVec>
__global__ void __launch_bounds__(kThreads) swiglu_pack8_kernel(const T* __restrict__ h, int64_t stride, int R, int I,
                                                                T* __restrict__ act, uint8_t* __restrict__ codes,
                                                                uint8_t* __restrict__ exps) {
  const int lane = threadIdx.x & 31;
  const int slices = (I + kSlice - 1) / kSlice, nb = (I + kBlk - 1) / kBlk;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int64_t r = unit / slices;
  if (r >= R) return;
  const int c = static_cast<int>(unit % slices) * kSlice, n = I - c;
  float u[8], g[8], a[8];
  to_floats(load_raw8<T, kVec>(h + r * stride + c, n, lane), u);
  to_floats(load_raw8<T, kVec>(h + r * stride + I + c, n, lane), g);
#pragma unroll
  for (int j = 0; j < 8; ++j) a[j] = u[j] * (g[j] * sigmoid(g[j]));
  store_raw8<T, kVec>(act + r * I + c, n, lane, from_floats<T>(a));
  uint8_t* cr = codes + r * 2 * I + c;
  uint8_t* er = exps + r * 2 * nb + c / kBlk;
  int e[2];
  uint2 q = encode8<T, kVec>(u, e);
  store_codes<kVec>(cr, n, lane, q);
  store_exponents<kVec>(er, n, lane, e);
  q = encode8<T, kVec>(g, e);
  store_codes<kVec>(cr + I, n, lane, q);
  store_exponents<kVec>(er + nb, n, lane, e);
}

// From the kept values u, g and d = dL/dact: du = d g s, dg = d u s (1 + g (1 - s)), act = u g s, with s = sigmoid(g).
template <typename T, bool kVec>
__global__ void __launch_bounds__(kThreads) swiglu_backward8_kernel(const uint8_t* __restrict__ codes,
                                                                    const uint8_t* __restrict__ exps,
                                                                    const T* __restrict__ grad, int64_t stride, int R,
                                                                    int I, T* __restrict__ dh, T* __restrict__ act) {
  const int lane = threadIdx.x & 31;
  const int slices = (I + kSlice - 1) / kSlice, nb = (I + kBlk - 1) / kBlk;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int64_t r = unit / slices;
  if (r >= R) return;
  const int c = static_cast<int>(unit % slices) * kSlice, n = I - c;
  float u[8], g[8], d[8], a[8];
  const uint8_t* cr = codes + r * 2 * I + c;
  const uint8_t* er = exps + r * 2 * nb + c / kBlk;
  to_floats(load_raw8<T, kVec>(grad + r * stride + c, n, lane), d);
  decode8<kVec>(load_codes<kVec>(cr, n, lane), er, n, lane, u);
  decode8<kVec>(load_codes<kVec>(cr + I, n, lane), er + nb, n, lane, g);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float s = sigmoid(g[j]);
    const float gs = g[j] * s;
    a[j] = u[j] * gs;
    const float dg = d[j] * (u[j] * s * (1.0f + g[j] * (1.0f - s)));
    u[j] = d[j] * gs;
    g[j] = dg;
  }
  store_raw8<T, kVec>(dh + r * 2 * I + c, n, lane, from_floats<T>(u));
  store_raw8<T, kVec>(dh + r * 2 * I + I + c, n, lane, from_floats<T>(g));
  if (act) store_raw8<T, kVec>(act + r * I + c, n, lane, from_floats<T>(a));
}

bool valid_rows(int64_t R, int64_t W, int32_t dtype) {
  return R >= 0 && R <= KF_SORT_MAX_ROWS && W >= 1 && W <= KF_SORT_MAX_WIDTH && valid_dtype(dtype);
}

// Blocks of a grid of one warp per (row, slice); 0 when they are more than a grid holds.
unsigned grid_of(int64_t R, int64_t W) {
  const int64_t b = (R * ((W + kSlice - 1) / kSlice) + kWarps - 1) / kWarps;
  return b <= 0x7fffffff ? static_cast<unsigned>(b) : 0u;
}

inline bool aligned(const void* p, unsigned a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

template <typename F>
int launch(int32_t dtype, bool vec, F&& f) {
  int sms = 0;
  const int rc = device_ready(&sms);
  if (rc != KF_OK) return rc;
  return dispatch_rows(dtype, vec, [&](auto t, auto v) {
           f(t, v);
           return cudaGetLastError();
         }) == cudaSuccess
             ? KF_OK
             : KF_ERR_CUDA;
}

template <typename P>
using ElemOf = std::remove_const_t<std::remove_pointer_t<P>>;

}  // namespace
}  // namespace kf

using namespace kf;

extern "C" {

int kf_pack8(const void* x, int32_t dtype, int64_t x_stride, int32_t num_rows, int32_t width, void* codes,
             void* exponents, void* stream) {
  if (!valid_rows(num_rows, width, dtype) || x_stride < 0) return KF_ERR_INVALID_ARGUMENT;
  if (num_rows == 0) return KF_OK;
  const unsigned grid = grid_of(num_rows, width);
  if (!x || !codes || !exponents || !grid) return KF_ERR_INVALID_ARGUMENT;
  const bool vec = vec_rows(x, x_stride, width, dtype) && aligned(codes, 8);
  return launch(dtype, vec, [&](auto t, auto v) {
    using E = ElemOf<decltype(t)>;
    pack8_kernel<E, decltype(v)::value><<<grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const E*>(x), x_stride, num_rows, width, static_cast<uint8_t*>(codes),
        static_cast<uint8_t*>(exponents));
  });
}

int kf_restore8(const void* codes, const void* exponents, int32_t dtype, int32_t num_rows, int32_t width,
                const int32_t* row_pair, int32_t top_k, int32_t out_rows, void* output, void* stream) {
  if (!valid_rows(num_rows, width, dtype) || !valid_rows(out_rows, width, dtype)) return KF_ERR_INVALID_ARGUMENT;
  if (row_pair ? (top_k < 1 || top_k > KF_SORT_MAX_TOP_K) : out_rows != num_rows) return KF_ERR_INVALID_ARGUMENT;
  if (out_rows == 0) return KF_OK;
  const unsigned grid = grid_of(out_rows, width);
  if (!output || !grid || (num_rows > 0 && (!codes || !exponents))) return KF_ERR_INVALID_ARGUMENT;
  const bool vec = vec_rows(output, width, width, dtype) && aligned(codes, 8);
  return launch(dtype, vec, [&](auto t, auto v) {
    using E = ElemOf<decltype(t)>;
    restore8_kernel<E, decltype(v)::value><<<grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(exponents), num_rows, width, row_pair, top_k,
        out_rows, static_cast<E*>(output));
  });
}

int kf_swiglu_pack8(const void* h, int32_t dtype, int64_t h_stride, int32_t num_rows, int32_t inter, void* act,
                    void* codes, void* exponents, void* stream) {
  if (!valid_rows(num_rows, inter, dtype) || h_stride < 0) return KF_ERR_INVALID_ARGUMENT;
  if (num_rows == 0) return KF_OK;
  const unsigned grid = grid_of(num_rows, inter);
  if (!h || !act || !codes || !exponents || !grid) return KF_ERR_INVALID_ARGUMENT;
  const bool vec = vec_rows(h, h_stride, inter, dtype) && vec_rows(act, inter, inter, dtype) && aligned(codes, 8);
  return launch(dtype, vec, [&](auto t, auto v) {
    using E = ElemOf<decltype(t)>;
    swiglu_pack8_kernel<E, decltype(v)::value><<<grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const E*>(h), h_stride, num_rows, inter, static_cast<E*>(act), static_cast<uint8_t*>(codes),
        static_cast<uint8_t*>(exponents));
  });
}

int kf_swiglu_backward8(const void* codes, const void* exponents, const void* grad_act, int32_t dtype,
                        int64_t grad_stride, int32_t num_rows, int32_t inter, void* grad_h, void* act, void* stream) {
  if (!valid_rows(num_rows, inter, dtype) || grad_stride < 0) return KF_ERR_INVALID_ARGUMENT;
  if (num_rows == 0) return KF_OK;
  const unsigned grid = grid_of(num_rows, inter);
  if (!codes || !exponents || !grad_act || !grad_h || !grid) return KF_ERR_INVALID_ARGUMENT;
  const bool vec = vec_rows(grad_act, grad_stride, inter, dtype) && vec_rows(grad_h, inter, inter, dtype) &&
                   (!act || vec_rows(act, inter, inter, dtype)) && aligned(codes, 8);
  return launch(dtype, vec, [&](auto t, auto v) {
    using E = ElemOf<decltype(t)>;
    swiglu_backward8_kernel<E, decltype(v)::value><<<grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(exponents), static_cast<const E*>(grad_act),
        grad_stride, num_rows, inter, static_cast<E*>(grad_h), static_cast<E*>(act));
  });
}

}  // extern "C"
