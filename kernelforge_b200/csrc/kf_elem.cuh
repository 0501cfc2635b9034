// Rows of bf16, fp16 or fp32 elements, read and written eight columns per lane.
//
// A warp covers a slice of 256 columns.  In the vector form (kVec), which needs
// 16-byte aligned rows and a width that is a multiple of 8, a lane's accesses are 16
// bytes: lane l holds columns 8l .. 8l+7 of 16-bit types, and 4l .. 4l+3 and
// 128 + 4l .. 128 + 4l+3 of fp32, so that each access of a warp is one run of 512
// bytes.  Otherwise accesses are 4 bytes: lane l holds columns l + 32 j of fp32, and
// the pairs 2l + 64 j, 2l + 64 j + 1 of 16-bit types, which a row that starts between
// two 4-byte words takes from its neighbours' words by shuffles.  Nothing outside
// the row is read or written.  Arithmetic is fp32 whatever the element type.
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

// Column of a lane's 16-byte access i (of 1 for 16-bit types, 2 for fp32) inside a slice.
template <typename T>
__device__ __forceinline__ int vec_col(int lane, int i) {
  return i * 128 + lane * (16 / static_cast<int>(sizeof(T)));
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
      if (vec_col<T>(lane, i) < n) v = __ldg(reinterpret_cast<const uint4*>(slice + vec_col<T>(lane, i)));
      r.x[4 * i] = v.x;
      r.x[4 * i + 1] = v.y;
      r.x[4 * i + 2] = v.z;
      r.x[4 * i + 3] = v.w;
    }
  } else if constexpr (sizeof(T) == 4) {
    const uint32_t* p = reinterpret_cast<const uint32_t*>(slice);
    if (n >= kSlice) {   // without conditions the loads go out together
#pragma unroll
      for (int j = 0; j < 8; ++j) r.x[j] = __ldg(p + lane + 32 * j);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) r.x[j] = lane + 32 * j < n ? __ldg(p + lane + 32 * j) : 0u;
    }
  } else {
    const unsigned short* p = reinterpret_cast<const unsigned short*>(slice);
    const bool even = (reinterpret_cast<uintptr_t>(slice) & 3u) == 0;
    if (n >= kSlice && even) {
#pragma unroll
      for (int j = 0; j < 4; ++j) r.x[j] = __ldg(reinterpret_cast<const uint32_t*>(p) + lane + 32 * j);
    } else if (n >= kSlice) {
      // word q holds elements 2q - 1 and 2q; of words 0 and 128 only one element is the slice's
      uint32_t w[4], last = 0u;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int q = lane + 32 * j;
        w[j] = q == 0 ? static_cast<uint32_t>(__ldg(p)) << 16 : __ldg(reinterpret_cast<const uint32_t*>(p - 1) + q);
      }
      if (lane == 31) last = __ldg(p + kSlice - 1);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t up = __shfl_sync(0xffffffffu, w[j], (lane + 1) & 31);                 // word q + 1 of lanes 0..30
        const uint32_t wrap = j < 3 ? __shfl_sync(0xffffffffu, w[j < 3 ? j + 1 : 3], 0) : last;   // and of lane 31
        r.x[j] = __funnelshift_r(w[j], lane == 31 ? wrap : up, 16);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = 2 * lane + 64 * j;
        const uint32_t lo = c < n ? __ldg(p + c) : 0u, hi = c + 1 < n ? __ldg(p + c + 1) : 0u;
        r.x[j] = lo | (hi << 16);
      }
    }
  }
  return r;
}

template <typename T, bool kVec>
__device__ __forceinline__ void store_raw8(T* __restrict__ slice, int n, int lane, const Raw8<T>& r) {
  if (kVec) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
      if (vec_col<T>(lane, i) < n)
        *reinterpret_cast<uint4*>(slice + vec_col<T>(lane, i)) =
            make_uint4(r.x[4 * i], r.x[4 * i + 1], r.x[4 * i + 2], r.x[4 * i + 3]);
  } else if constexpr (sizeof(T) == 4) {
    uint32_t* p = reinterpret_cast<uint32_t*>(slice);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (lane + 32 * j < n) p[lane + 32 * j] = r.x[j];
  } else {
    unsigned short* p = reinterpret_cast<unsigned short*>(slice);
    const bool even = (reinterpret_cast<uintptr_t>(slice) & 3u) == 0;
    if (n >= kSlice && even) {
#pragma unroll
      for (int j = 0; j < 4; ++j) reinterpret_cast<uint32_t*>(p)[lane + 32 * j] = r.x[j];
    } else if (n >= kSlice) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t down = __shfl_sync(0xffffffffu, r.x[j], (lane + 31) & 31);                 // pair q - 1 of lanes 1..31
        const uint32_t wrap = __shfl_sync(0xffffffffu, r.x[j > 0 ? j - 1 : 0], 31);               // and of lane 0
        const uint32_t w = __funnelshift_r(lane == 0 ? wrap : down, r.x[j], 16);
        if (j == 0 && lane == 0)
          p[0] = static_cast<unsigned short>(r.x[0] & 0xffffu);
        else
          reinterpret_cast<uint32_t*>(p - 1)[lane + 32 * j] = w;
      }
      if (lane == 31) p[kSlice - 1] = static_cast<unsigned short>(r.x[3] >> 16);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = 2 * lane + 64 * j;
        if (c < n) p[c] = static_cast<unsigned short>(r.x[j] & 0xffffu);
        if (c + 1 < n) p[c + 1] = static_cast<unsigned short>(r.x[j] >> 16);
      }
    }
  }
}

// Column of element j of a lane in the form without 16-byte accesses.
template <typename T>
__device__ __forceinline__ int word_col(int lane, int j) {
  return sizeof(T) == 4 ? lane + 32 * j : 2 * lane + 64 * (j >> 1) + (j & 1);
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

// Zeroes the rows that row_pair gives no pair: this block's share of them, as block
// `part` of `parts`.  The shares are interleaved, because such rows come in runs (the
// ends of the segments, the rest of the buffer): a block looks at every parts-th row,
// a thread each, lists those without a pair in shared memory, and all its warps zero
// the listed rows together, a slice each.  The whole block calls it.
constexpr int kZeroList = 512;
template <typename T, bool kVec>
__device__ __forceinline__ void zero_rows(const int32_t* row_pair, int64_t pairs, int part, int parts, int R,
                                          int H, T* __restrict__ rows) {
  __shared__ int32_t list[kZeroList];
  __shared__ int listed;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarp = blockDim.x >> 5;
  const int slices = (H + kSlice - 1) / kSlice;
  const int per_pass = min(static_cast<int>(blockDim.x), kZeroList);
  for (int64_t first = part; first < R; first += static_cast<int64_t>(per_pass) * parts) {
    if (threadIdx.x == 0) listed = 0;
    __syncthreads();
    const int64_t r = first + static_cast<int64_t>(threadIdx.x) * parts;
    if (static_cast<int>(threadIdx.x) < per_pass && r < R) {
      const int p = row_pair[r];
      if (p < 0 || p >= pairs) list[atomicAdd(&listed, 1)] = static_cast<int32_t>(r);
    }
    __syncthreads();
    const int n = listed;
    const Raw8<T> z = {};
    int i = warp / slices, s = warp % slices;
    for (; i < n;) {
      store_raw8<T, kVec>(rows + static_cast<int64_t>(list[i]) * H + s * kSlice, H - s * kSlice, lane, z);
      s += nwarp;
      while (s >= slices) {
        s -= slices;
        ++i;
      }
    }
    __syncthreads();   // the list is rewritten next
  }
}
// Blocks for it at the front of a grid that does something else: two per SM, or one per 64 rows.
inline unsigned zero_blocks_for(int R) { return static_cast<unsigned>(R < 64 * 296 ? (R + 63) / 64 : 296); }

// Warps per token and tokens per block for `slices` slices of a row, `per` of them per warp.
constexpr int kScatterWarps = 16;
struct ScatterPlan {
  int warps, tokens;
};
inline ScatterPlan plan_scatter(int slices, int per) {
  const int need = (slices + per - 1) / per;
  const int steps = (need + kScatterWarps - 1) / kScatterWarps;
  const int warps = (need + steps - 1) / steps;
  return ScatterPlan{warps, warps > 8 ? 1 : 8 / warps};
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
