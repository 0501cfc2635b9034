// Rows of bf16, fp16 or fp32 elements, read and written eight columns per lane.
//
// A warp covers a slice of 256 columns.  In the vector form (kVec) lane l holds
// columns 8l .. 8l+7 in 16-byte accesses, which needs 16-byte aligned rows and a
// width that is a multiple of 8; otherwise lane l holds columns l + 32 j, one
// element per access, so that a warp's accesses still fall in whole sectors.
// Arithmetic is fp32 whatever the element type.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "kf_moe.h"

namespace kf {

constexpr int kSlice = 256;  // columns per warp and step

inline size_t elem_bytes(int dtype) { return dtype == KF_DTYPE_F32 ? 4 : 2; }
inline bool valid_dtype(int dtype) { return dtype == KF_DTYPE_BF16 || dtype == KF_DTYPE_F16 || dtype == KF_DTYPE_F32; }

// Whether rows at `p`, `stride` elements apart and `width` wide, allow 16-byte accesses.
inline bool vec_rows(const void* p, int64_t stride, int64_t width, int dtype) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (static_cast<uint64_t>(stride) * elem_bytes(dtype)) % 16 == 0 &&
         width % 8 == 0;
}

__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }

__device__ __forceinline__ float2 unpack2(uint32_t w, const __nv_bfloat16*) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
}
__device__ __forceinline__ float2 unpack2(uint32_t w, const __half*) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, const __nv_bfloat16*) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, const __half*) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Column of element j of this lane inside a slice.
template <bool kVec>
__device__ __forceinline__ int slice_col(int lane, int j) {
  return kVec ? lane * 8 + j : lane + 32 * j;
}

// The raw bits of a lane's eight elements (bf16/fp16: 16 bytes in x[0..3]; fp32: 32 bytes).
template <typename T>
struct Raw8 {
  uint32_t x[sizeof(T) * 2];
};

// Eight elements of one row's slice.  `n` columns of the slice exist; the others read as zero.
template <typename T, bool kVec>
__device__ __forceinline__ Raw8<T> load_raw8(const T* __restrict__ slice, int n, int lane) {
  Raw8<T> r;
  if (kVec) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (lane * 8 < n) v = __ldg(reinterpret_cast<const uint4*>(slice + lane * 8) + i);
      r.x[4 * i] = v.x;
      r.x[4 * i + 1] = v.y;
      r.x[4 * i + 2] = v.z;
      r.x[4 * i + 3] = v.w;
    }
  } else if (sizeof(T) == 4) {
    const uint32_t* p = reinterpret_cast<const uint32_t*>(slice);
#pragma unroll
    for (int j = 0; j < 8; ++j) r.x[j % (sizeof(T) * 2)] = lane + 32 * j < n ? __ldg(p + lane + 32 * j) : 0u;
  } else {
    const unsigned short* p = reinterpret_cast<const unsigned short*>(slice);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t lo = lane + 64 * j < n ? __ldg(p + lane + 64 * j) : 0u;
      const uint32_t hi = lane + 64 * j + 32 < n ? __ldg(p + lane + 64 * j + 32) : 0u;
      r.x[j] = lo | (hi << 16);
    }
  }
  return r;
}

template <typename T, bool kVec>
__device__ __forceinline__ void store_raw8(T* __restrict__ slice, int n, int lane, const Raw8<T>& r) {
  if (kVec) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
      if (lane * 8 < n)
        reinterpret_cast<uint4*>(slice + lane * 8)[i] =
            make_uint4(r.x[4 * i], r.x[4 * i + 1], r.x[4 * i + 2], r.x[4 * i + 3]);
  } else if (sizeof(T) == 4) {
    uint32_t* p = reinterpret_cast<uint32_t*>(slice);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (lane + 32 * j < n) p[lane + 32 * j] = r.x[j % (sizeof(T) * 2)];
  } else {
    unsigned short* p = reinterpret_cast<unsigned short*>(slice);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (lane + 64 * j < n) p[lane + 64 * j] = static_cast<unsigned short>(r.x[j] & 0xffffu);
      if (lane + 64 * j + 32 < n) p[lane + 64 * j + 32] = static_cast<unsigned short>(r.x[j] >> 16);
    }
  }
}

__device__ __forceinline__ void to_floats(const Raw8<float>& r, float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(r.x[j]);
}
template <typename T>
__device__ __forceinline__ void to_floats(const Raw8<T>& r, float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = unpack2(r.x[j], static_cast<const T*>(nullptr));
    v[2 * j] = f.x;
    v[2 * j + 1] = f.y;
  }
}

// One rounding to the element type, to nearest even.
template <typename T>
__device__ __forceinline__ Raw8<T> from_floats(const float (&v)[8]) {
  Raw8<T> r;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 8; ++j) r.x[j] = __float_as_uint(v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) r.x[j] = pack2(v[2 * j], v[2 * j + 1], static_cast<const T*>(nullptr));
  }
  return r;
}

// Calls f(T*{}, bool_constant) for a dtype and access form.
template <bool B>
struct BoolTag {
  static constexpr bool value = B;
};
template <typename F>
inline cudaError_t dispatch_rows(int dtype, bool vec, F&& f) {
  if (dtype == KF_DTYPE_BF16) {
    const __nv_bfloat16* t = nullptr;
    return vec ? f(t, BoolTag<true>{}) : f(t, BoolTag<false>{});
  }
  if (dtype == KF_DTYPE_F16) {
    const __half* t = nullptr;
    return vec ? f(t, BoolTag<true>{}) : f(t, BoolTag<false>{});
  }
  const float* t = nullptr;
  return vec ? f(t, BoolTag<true>{}) : f(t, BoolTag<false>{});
}

}  // namespace kf
