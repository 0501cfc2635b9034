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
#include <type_traits>

#include <cuda_fp8.h>

#include "kf_elem.cuh"
#include "kf_fp8.cuh"
#include "kf_internal.cuh"

namespace kf {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// Exponents are held as they are stored, e + 127 (1 .. 247).
template <typename T>
constexpr int kTopExponent = 127 + 120;   // 256 * 2^120 = 2^128 is beyond bf16 and fp32
template <>
constexpr int kTopExponent<__half> = 127 + 8;   // 256 * 2^8 = 65536 is beyond fp16

__device__ __forceinline__ float scale_of(int e) { return __uint_as_float(static_cast<uint32_t>(e) << 23); }   // 2^(e - 127)
__device__ __forceinline__ float inverse_scale(int e) { return scale_of(254 - e); }

// Smallest e >= 1 with amax <= 448 * 2^(e - 127) = 1.75 * 2^(e - 119), amax finite and not
// negative: its exponent field less 8, and one more where the mantissa is above 1.75,
// which adding 2^23 - 1 - 0.75 * 2^23 carries into the field.
__device__ __forceinline__ int block_exponent(uint32_t amax_bits) {
  return max(static_cast<int>((amax_bits + 0x1fffffu) >> 23) - 8, 1);
}

// Magnitudes as keys in the type's own bits: larger magnitude, larger key.  Above
// kRareKey a block needs more than the plain path: its scale is the type's last one
// (1.75 * 2^127, or 1.75 * 2^15 of fp16, and above), or a value is not finite.
// Two 16-bit keys share a word, and one instruction takes the larger of both, NaN
// (key 0x7fff) winning.
template <typename T>
constexpr uint32_t kRareKey = 0x7f600000u;
template <>
constexpr uint32_t kRareKey<__nv_bfloat16> = 0x7f60u;
template <>
constexpr uint32_t kRareKey<__half> = 0x7b00u;

__device__ __forceinline__ uint32_t key_bits(uint32_t key, const float*) { return key; }   // the magnitude's fp32 bits
__device__ __forceinline__ uint32_t key_bits(uint32_t key, const __nv_bfloat16*) { return key << 16; }
__device__ __forceinline__ uint32_t key_bits(uint32_t key, const __half*) {
  return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(key))));
}

__device__ __forceinline__ uint32_t max2_keys(uint32_t a, uint32_t b, const __nv_bfloat16*) {
  const __nv_bfloat162 m = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}
__device__ __forceinline__ uint32_t max2_keys(uint32_t a, uint32_t b, const __half*) {
  const __half2 m = __hmax2_nan(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}

// The larger magnitudes of words i and i + 1 of a lane's 16-bit elements.
template <typename T>
__device__ __forceinline__ uint32_t pair_keys(const Raw8<T>& r, int i) {
  return max2_keys(r.x[i] & 0x7fff7fffu, r.x[i + 1] & 0x7fff7fffu, static_cast<const T*>(nullptr));
}

// A slice of 256 columns = two blocks.  The vector form of 16-bit types has a block
// per half-warp, the other forms every lane in both (elements 0..3 and 4..7).
template <typename T, bool kVec>
constexpr bool kHalfWarp = kVec && sizeof(T) == 2;

// Largest keys of this lane's blocks (the same twice where a half-warp has one).
template <typename T, bool kVec>
__device__ __forceinline__ void block_keys(const Raw8<T>& r, uint32_t (&key)[2]) {
  const T* type = nullptr;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      key[h] = __reduce_max_sync(0xffffffffu, max(max(r.x[4 * h] & 0x7fffffffu, r.x[4 * h + 1] & 0x7fffffffu),
                                                  max(r.x[4 * h + 2] & 0x7fffffffu, r.x[4 * h + 3] & 0x7fffffffu)));
  } else if constexpr (kHalfWarp<T, kVec>) {
    uint32_t m = max2_keys(pair_keys(r, 0), pair_keys(r, 2), type);
#pragma unroll
    for (int off = 8; off >= 1; off >>= 1) m = max2_keys(m, __shfl_xor_sync(0xffffffffu, m, off), type);
    key[0] = key[1] = max(m & 0xffffu, m >> 16);
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t m = pair_keys(r, 2 * h);
      key[h] = __reduce_max_sync(0xffffffffu, max(m & 0xffffu, m >> 16));
    }
  }
}

// The same for two sets of values, whose 16-bit keys go through the shuffles in one word.
template <typename T, bool kVec>
__device__ __forceinline__ void block_keys2(const Raw8<T>& a, const Raw8<T>& b, uint32_t (&ka)[2], uint32_t (&kb)[2]) {
  if constexpr (kHalfWarp<T, kVec>) {
    const T* type = nullptr;
    const uint32_t ma = max2_keys(pair_keys(a, 0), pair_keys(a, 2), type);
    const uint32_t mb = max2_keys(pair_keys(b, 0), pair_keys(b, 2), type);
    uint32_t m = max2_keys(__byte_perm(ma, mb, 0x5410), __byte_perm(ma, mb, 0x7632), type);
#pragma unroll
    for (int off = 8; off >= 1; off >>= 1) m = max2_keys(m, __shfl_xor_sync(0xffffffffu, m, off), type);
    ka[0] = ka[1] = m & 0xffffu;
    kb[0] = kb[1] = m >> 16;
  } else {
    block_keys<T, kVec>(a, ka);
    block_keys<T, kVec>(b, kb);
  }
}

// Blocks above kRareKey: the scale from the finite values, codes up to 240 under the type's last scale, NaN codes
// for the others.
template <typename T, bool kVec>
__device__ __noinline__ void rare_blocks(float (&q)[8], int (&e)[2]) {
  uint32_t a[2] = {0u, 0u};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t b = __float_as_uint(q[j]) & 0x7fffffffu;
    if (b < 0x7f800000u) a[j >> 2] = max(a[j >> 2], b);
  }
  if (kHalfWarp<T, kVec>) {
    uint32_t m = max(a[0], a[1]);
#pragma unroll
    for (int off = 8; off >= 1; off >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, off));
    a[0] = a[1] = m;
  } else {
    a[0] = __reduce_max_sync(0xffffffffu, a[0]);
    a[1] = __reduce_max_sync(0xffffffffu, a[1]);
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) e[h] = block_exponent(a[h]);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float v = q[j];
    const float limit = e[j >> 2] == kTopExponent<T> ? 240.f : 448.f;
    q[j] = fminf(fmaxf(v * inverse_scale(e[j >> 2]), -limit), limit);
    if ((__float_as_uint(v) & 0x7fffffffu) >= 0x7f800000u) q[j] = __uint_as_float(0x7fffffffu);
  }
}

// Codes (byte j = element j) and exponents of this lane's eight elements, from their blocks' largest keys.
template <typename T, bool kVec>
__device__ __forceinline__ uint2 encode8(const float (&v)[8], const uint32_t (&key)[2], int (&e)[2]) {
  const T* type = nullptr;
  float q[8];
  if (__any_sync(0xffffffffu, max(key[0], key[1]) > kRareKey<T>)) {
#pragma unroll
    for (int j = 0; j < 8; ++j) q[j] = v[j];
    rare_blocks<T, kVec>(q, e);
  } else {
    e[0] = block_exponent(key_bits(key[0], type));
    e[1] = kHalfWarp<T, kVec> ? e[0] : block_exponent(key_bits(key[1], type));
    const float inv[2] = {inverse_scale(e[0]), inverse_scale(e[1])};
#pragma unroll
    for (int j = 0; j < 8; ++j) q[j] = v[j] * inv[j >> 2];
  }
  return make_uint2(pack_fp8x4(q[0], q[1], q[2], q[3]), pack_fp8x4(q[4], q[5], q[6], q[7]));
}

template <typename T, bool kVec>
__device__ __forceinline__ void store_codes(uint8_t* __restrict__ slice, int n, int lane, uint2 c) {
  if (kHalfWarp<T, kVec>) {
    if (lane * 8 < n) *reinterpret_cast<uint2*>(slice + lane * 8) = c;
  } else if (kVec) {
    if (lane * 4 < n) *reinterpret_cast<uint32_t*>(slice + lane * 4) = c.x;
    if (128 + lane * 4 < n) *reinterpret_cast<uint32_t*>(slice + 128 + lane * 4) = c.y;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (word_col<T>(lane, j) < n)
        slice[word_col<T>(lane, j)] = static_cast<uint8_t>((j < 4 ? c.x : c.y) >> (8 * (j & 3)));
  }
}

template <typename T, bool kVec>
__device__ __forceinline__ uint2 load_codes(const uint8_t* __restrict__ slice, int n, int lane) {
  uint2 c = make_uint2(0u, 0u);
  if (kHalfWarp<T, kVec>) {
    if (lane * 8 < n) c = __ldg(reinterpret_cast<const uint2*>(slice + lane * 8));
  } else if (kVec) {
    if (lane * 4 < n) c.x = __ldg(reinterpret_cast<const uint32_t*>(slice + lane * 4));
    if (128 + lane * 4 < n) c.y = __ldg(reinterpret_cast<const uint32_t*>(slice + 128 + lane * 4));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (word_col<T>(lane, j) < n)
        (j < 4 ? c.x : c.y) |= static_cast<uint32_t>(__ldg(slice + word_col<T>(lane, j))) << (8 * (j & 3));
  }
  return c;
}

// The slice's one or two exponent bytes.
template <typename T, bool kVec>
__device__ __forceinline__ void store_exponents(uint8_t* __restrict__ exps, int n, int lane, const int (&e)[2]) {
  if (kHalfWarp<T, kVec>) {
    if ((lane & 15) == 0 && (lane >> 4) * kBlk < n) exps[lane >> 4] = static_cast<uint8_t>(e[0]);
  } else {
    if (lane < 2 && lane * kBlk < n) exps[lane] = static_cast<uint8_t>(lane ? e[1] : e[0]);
  }
}

// 2^e of this lane's two blocks (of the one that it is in, twice, where a half-warp has a block).
template <typename T, bool kVec>
__device__ __forceinline__ void load_scales(const uint8_t* __restrict__ exps, int n, int lane, float (&s)[2]) {
  if (kHalfWarp<T, kVec>) {
    const int b = lane >> 4;
    s[0] = s[1] = b * kBlk < n ? scale_of(__ldg(exps + b)) : 0.f;
  } else {
    s[0] = 0 < n ? scale_of(__ldg(exps)) : 0.f;
    s[1] = kBlk < n ? scale_of(__ldg(exps + 1)) : 0.f;
  }
}

// The values of eight codes times their blocks' scales, exact in fp32.
__device__ __forceinline__ void decode8(uint2 c, const float (&s)[2], float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t w = (j < 2 ? c.x : c.y) >> (16 * (j & 1));
    const float2 f = fp8x2_to_float2(static_cast<__nv_fp8x2_storage_t>(w & 0xffffu));
    v[2 * j] = f.x * s[j >> 1];
    v[2 * j + 1] = f.y * s[j >> 1];
  }
}

// 1 / (1 + e^-x); 0 where 1 + e^-x is beyond 2^126.  For fp32 rows expf and a
// division of 2 ulp; for 16-bit rows, whose own rounding is 2^-9 or 2^-12, the
// hardware's 2^y of y = -x log2 e (a rounding of y costs |x| 2^-24 of the result) and
// reciprocal: 4 instructions instead of some 15, where the kernels are bound by
// issuing them.
template <typename T>
__device__ __forceinline__ float sigmoid(float x) {
  if constexpr (sizeof(T) == 4) {
    return __fdividef(1.0f, 1.0f + expf(-x));
  } else {
    float y, s;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * -1.4426950408889634f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.0f + y));
    return s;
  }
}

// Division of n < 2^31 by a constant of the launch, 1 <= d <= 4096, as a product: with
// 2^(s-1) < d <= 2^s and m = ceil(2^(31+s) / d) the error of n m / 2^(31+s) is below
// n / 2^(31+s) < 2^-s <= 1 / d, too little to reach the next integer.
struct Divisor {
  uint32_t m, shift;
};
inline Divisor divisor_of(uint32_t d) {
  uint32_t s = 0;
  while ((1u << s) < d) ++s;
  return s == 0 ? Divisor{0u, 0u}   // d = 1
                : Divisor{static_cast<uint32_t>(((uint64_t{1} << (31 + s)) + d - 1) / d), s - 1};
}
__device__ __forceinline__ uint32_t divide(uint32_t n, const Divisor& d) { return d.m ? __umulhi(n, d.m) >> d.shift : n; }

// One warp per (row, group of kGroup slices), consecutive warps on consecutive
// groups of a row: this warp's row and first slice.  `by`: the divisor for a row's groups.
struct Unit {
  int64_t row;
  int slice;
};
template <int kGroup>
__device__ __forceinline__ Unit unit_of(int slices, const Divisor& by) {
  const unsigned groups = (slices + kGroup - 1) / kGroup;
  const unsigned u = blockIdx.x * kWarps + (threadIdx.x >> 5);
  const unsigned row = divide(u, by);
  return Unit{row, static_cast<int>(u - row * groups) * kGroup};
}

// Slices per warp whose loads are in flight together: two, where that leaves at
// most an eighth of the warps half empty, else one.
inline bool pairs_of_slices(int slices) { return slices % 2 == 0 || slices >= 7; }

// 60 us = 5.8 TB/s for 16384 rows of 7168 bf16 columns, 43 us = 6.8 TB/s for 8192 of fp32; 16.5 us = 5.3 TB/s for 4096
// of bf16 among others and 19 us alone: memory and issue share it (of the issue slots 73 % while blocks run, 56 % over
// the launch), and such a launch's first and last blocks.  Off 16 bytes codes go a byte at a time: 28 us for 4096
// rows of 7167 bf16 columns, 27 us of fp32.
template <typename T, bool kVec, int kGroup>
__global__ void __launch_bounds__(kThreads) pack8_kernel(const T* __restrict__ x, int64_t stride, int R, int W,
                                                         const Divisor by, uint8_t* __restrict__ codes,
                                                         uint8_t* __restrict__ exps) {
  const int lane = threadIdx.x & 31;
  const int slices = (W + kSlice - 1) / kSlice, nb = (W + kBlk - 1) / kBlk;
  const Unit u = unit_of<kGroup>(slices, by);
  if (u.row >= R) return;
  const T* src = x + u.row * stride;
  Raw8<T> raw[kGroup];
#pragma unroll
  for (int j = 0; j < kGroup; ++j) {
    const int c = (u.slice + j) * kSlice;
    raw[j] = load_raw8<T, kVec>(src + c, W - c, lane);   // past the width: nothing is read
  }
#pragma unroll
  for (int j = 0; j < kGroup; ++j) {
    const int c = (u.slice + j) * kSlice, n = W - c;
    if (n <= 0) break;
    float v[8];
    uint32_t key[2];
    int e[2];
    block_keys<T, kVec>(raw[j], key);
    to_floats(raw[j], v);
    const uint2 q = encode8<T, kVec>(v, key, e);
    store_codes<T, kVec>(codes + u.row * W + c, n, lane, q);
    store_exponents<T, kVec>(exps + u.row * nb + c / kBlk, n, lane, e);
  }
}

template <typename T, bool kVec>
__device__ __forceinline__ Raw8<T> restored(uint2 codes, const float (&s)[2]) {
  float v[8];
  decode8(codes, s, v);
  return from_floats<T>(v);
}

// Rows as they were.  54 us = 6.6 TB/s for 16384 rows of 7168 bf16 columns, 46 us = 6.3 TB/s for 8192 of fp32; off 16
// bytes 28 us for 4096 rows of 7167 bf16 columns, 32 us of fp32.
template <typename T, bool kVec, int kGroup>
__global__ void __launch_bounds__(kThreads) restore8_kernel(const uint8_t* __restrict__ codes,
                                                            const uint8_t* __restrict__ exps, int R, int W,
                                                            const Divisor by, T* __restrict__ out) {
  const int lane = threadIdx.x & 31;
  const int slices = (W + kSlice - 1) / kSlice, nb = (W + kBlk - 1) / kBlk;
  const Unit u = unit_of<kGroup>(slices, by);
  if (u.row >= R) return;
  uint2 q[kGroup];
  float s[kGroup][2];
#pragma unroll
  for (int j = 0; j < kGroup; ++j) {
    const int c = (u.slice + j) * kSlice;
    q[j] = load_codes<T, kVec>(codes + u.row * W + c, W - c, lane);
    load_scales<T, kVec>(exps + u.row * nb + c / kBlk, W - c, lane, s[j]);
  }
#pragma unroll
  for (int j = 0; j < kGroup; ++j) {
    const int c = (u.slice + j) * kSlice;
    store_raw8<T, kVec>(out + u.row * W + c, W - c, lane, restored<T, kVec>(q[j], s[j]));
  }
}

// Rows in expert order: a block holds a token's row across its warps, two slices
// each, decodes it once and stores it K times (as scatter_rows_kernel, whose reason
// for one block per token holds here too).  The first blocks zero the rows of no pair.
// 93 us = 6.0 TB/s for 4096 tokens of 7168 bf16 columns into 36608 rows (fp32 175 us = 6.2 TB/s, 7167 bf16 columns
// 117 us); a warp per output row, which decodes a row K times, took 214 us.
template <typename T, bool kVec>
__global__ void __launch_bounds__(kScatterWarps * 32) restore8_sorted_kernel(
    const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exps, int T_, int W,
    const int32_t* __restrict__ pair_row, const int32_t* __restrict__ row_pair, int K, int R, int warps, int tokens,
    unsigned zero_blocks, T* __restrict__ out) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (blockIdx.x < zero_blocks) {
    zero_rows<T, kVec>(row_pair, static_cast<int64_t>(T_) * K, blockIdx.x, zero_blocks, R, W, out);
    return;
  }
  const int sub = warp / warps;
  const int64_t t = static_cast<int64_t>(blockIdx.x - zero_blocks) * tokens + sub;
  if (t >= T_) return;
  const int nb = (W + kBlk - 1) / kBlk;
  int mine = -1;
  if (lane < K) mine = pair_row[t * K + lane];
  for (int c0 = (warp - sub * warps) * kSlice; c0 < W; c0 += 2 * warps * kSlice) {
    uint2 q[2];
    float s[2][2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int c = c0 + j * warps * kSlice;
      q[j] = load_codes<T, kVec>(codes + t * W + c, W - c, lane);
      load_scales<T, kVec>(exps + t * nb + c / kBlk, W - c, lane, s[j]);
    }
    Raw8<T> v[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) v[j] = restored<T, kVec>(q[j], s[j]);
    for (int k = 0; k < K; ++k) {
      const int row = __shfl_sync(0xffffffffu, mine, k);
      if (row < 0 || row >= R) continue;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int c = c0 + j * warps * kSlice;
        store_raw8<T, kVec>(out + static_cast<int64_t>(row) * W + c, W - c, lane, v[j]);
      }
    }
  }
}

// h = [up | gate]: act = up * silu(gate), and h kept in 8 bits (each half's blocks begin at its own column 0).
// 90 us = 6.0 TB/s for 32768 rows of 2048 bf16 columns each (bound by issue and memory alike: 140 us with divisions
// and a check per element), 139 us = 6.8 TB/s of fp32; the activation alone 62 us = 6.5 TB/s.  Rows of 2047 bf16
// columns, whose codes go a byte at a time, 188 us.
template <typename T, bool kVec, int kGroup>
__global__ void __launch_bounds__(kThreads) swiglu_pack8_kernel(const T* __restrict__ h, int64_t stride, int R, int I,
                                                                const Divisor by, T* __restrict__ act,
                                                                uint8_t* __restrict__ codes,
                                                                uint8_t* __restrict__ exps) {
  const int lane = threadIdx.x & 31;
  const int slices = (I + kSlice - 1) / kSlice, nb = (I + kBlk - 1) / kBlk;
  const Unit unit = unit_of<kGroup>(slices, by);
  if (unit.row >= R) return;
  const int64_t r = unit.row;
  Raw8<T> ru[kGroup], rg[kGroup];
#pragma unroll
  for (int i = 0; i < kGroup; ++i) {
    const int c = (unit.slice + i) * kSlice, n = I - c;
    ru[i] = load_raw8<T, kVec>(h + r * stride + c, n, lane);
    rg[i] = load_raw8<T, kVec>(h + r * stride + I + c, n, lane);
  }
#pragma unroll
  for (int i = 0; i < kGroup; ++i) {
    const int c = (unit.slice + i) * kSlice, n = I - c;
    if (n <= 0) break;
    float u[8], g[8], a[8];
    to_floats(ru[i], u);
    to_floats(rg[i], g);
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] = u[j] * (g[j] * sigmoid<T>(g[j]));
    store_raw8<T, kVec>(act + r * I + c, n, lane, from_floats<T>(a));
    if (codes == nullptr) continue;   // the activation alone
    uint32_t ku[2], kg[2];
    block_keys2<T, kVec>(ru[i], rg[i], ku, kg);
    uint8_t* cr = codes + r * 2 * I + c;
    uint8_t* er = exps + r * 2 * nb + c / kBlk;
    int e[2];
    uint2 q = encode8<T, kVec>(u, ku, e);
    store_codes<T, kVec>(cr, n, lane, q);
    store_exponents<T, kVec>(er, n, lane, e);
    q = encode8<T, kVec>(g, kg, e);
    store_codes<T, kVec>(cr + I, n, lane, q);
    store_exponents<T, kVec>(er + nb, n, lane, e);
  }
}

// The fp32 bits of the largest magnitude of a lane's elements; NaN counts as the largest.
__device__ __forceinline__ uint32_t largest(const Raw8<float>& r) {
  uint32_t m = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, r.x[i] & 0x7fffffffu);
  return m;
}
__device__ __forceinline__ uint32_t largest(const Raw8<__nv_bfloat16>& r) {
  uint32_t m = 0u;
#pragma unroll
  for (int i = 0; i < 4; ++i) m = __vmaxu2(m, r.x[i] & 0x7fff7fffu);
  return max(m & 0xffffu, m >> 16) << 16;
}

// From u, g, s = sigmoid(g) and d = dL/dact: act, and the gradients in place of u and g.  dg = d u f with
// f = s + g s (1 - s), at most 1.1.  kFar: d u alone may be beyond fp32; f then goes into the larger of the two, so
// that nothing on the way is beyond fp32 or below its normal numbers unless the product is.  (With f always in one of
// them, u f would vanish for a small u and f, and exceed fp32 for a large u, where d makes up for it.)
template <bool kFar>
__device__ __forceinline__ void gate(float s, float d, float& u, float& g, float& act) {
  const float gs = g * s, f = fmaf(gs, 1.0f - s, s), t = d * u;
  act = u * gs;
  g = t * f;
  if (kFar && fabsf(t) == __uint_as_float(0x7f800000u)) g = fabsf(u) >= fabsf(d) ? u * f * d : d * f * u;
  u = d * gs;
}

// From the kept values u, g and d = dL/dact: du = d g s, dg = d u (s + g s (1 - s)), act = u g s, with s = sigmoid(g).
// One pass: 99 us = 6.8 TB/s for 32768 rows of 2048 bf16 columns, without act 84 us = 6.4 TB/s, bound by memory (the
// sigmoid in 15 instructions took 30 us more).  Telling the lanes whose d u may be beyond fp32 takes 5 us of the 84
// and none of the 99, a check per element 10.  fp32: 180 us = 6.7 TB/s.  2047 bf16 columns: 227 us.
template <typename T, bool kVec, int kGroup>
__global__ void __launch_bounds__(kThreads) swiglu_backward8_kernel(const uint8_t* __restrict__ codes,
                                                                    const uint8_t* __restrict__ exps,
                                                                    const T* __restrict__ grad, int64_t stride, int R,
                                                                    int I, const Divisor by, T* __restrict__ dh,
                                                                    T* __restrict__ act) {
  const int lane = threadIdx.x & 31;
  const int slices = (I + kSlice - 1) / kSlice, nb = (I + kBlk - 1) / kBlk;
  const Unit unit = unit_of<kGroup>(slices, by);
  if (unit.row >= R) return;
  const int64_t r = unit.row;
  Raw8<T> rd[kGroup];
  uint2 qu[kGroup], qg[kGroup];
  float su[kGroup][2], sg[kGroup][2];
#pragma unroll
  for (int i = 0; i < kGroup; ++i) {
    const int c = (unit.slice + i) * kSlice, n = I - c;
    const uint8_t* cr = codes + r * 2 * I + c;
    const uint8_t* er = exps + r * 2 * nb + c / kBlk;
    rd[i] = load_raw8<T, kVec>(grad + r * stride + c, n, lane);
    qu[i] = load_codes<T, kVec>(cr, n, lane);
    qg[i] = load_codes<T, kVec>(cr + I, n, lane);
    load_scales<T, kVec>(er, n, lane, su[i]);
    load_scales<T, kVec>(er + nb, n, lane, sg[i]);
  }
  bool far = false;   // whether some d u of this lane may be beyond fp32 (a NaN among d says so too); of fp16 none is
  if constexpr (!std::is_same_v<T, __half>) {
    uint32_t top = 0u;
    float scale = 0.f;
#pragma unroll
    for (int i = 0; i < kGroup; ++i) {
      top = max(top, largest(rd[i]));
      scale = fmaxf(scale, fmaxf(su[i][0], su[i][1]));
    }
    far = !(__uint_as_float(top) * (448.f * scale) < __uint_as_float(0x7f800000u));
  }
#pragma unroll
  for (int i = 0; i < kGroup; ++i) {
    const int c = (unit.slice + i) * kSlice, n = I - c;
    if (n <= 0) break;
    float u[8], g[8], d[8], a[8];
    to_floats(rd[i], d);
    decode8(qu[i], su[i], u);
    decode8(qg[i], sg[i], g);
    if (!far) {
#pragma unroll
      for (int j = 0; j < 8; ++j) gate<false>(sigmoid<T>(g[j]), d[j], u[j], g[j], a[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) gate<true>(sigmoid<T>(g[j]), d[j], u[j], g[j], a[j]);
    }
    store_raw8<T, kVec>(dh + r * 2 * I + c, n, lane, from_floats<T>(u));
    store_raw8<T, kVec>(dh + r * 2 * I + I + c, n, lane, from_floats<T>(g));
    if (act) store_raw8<T, kVec>(act + r * I + c, n, lane, from_floats<T>(a));
  }
}

bool valid_rows(int64_t R, int64_t W, int32_t dtype) {
  return R >= 0 && R <= KF_SORT_MAX_ROWS && W >= 1 && W <= KF_SORT_MAX_WIDTH && valid_dtype(dtype);
}

// Blocks of a grid of one warp per (row, group of slices); 0 when they are too many (rows of terabytes).
unsigned grid_of(int64_t R, int64_t W) {
  const int64_t slices = (W + kSlice - 1) / kSlice, group = pairs_of_slices(static_cast<int>(slices)) ? 2 : 1;
  const int64_t units = R * ((slices + group - 1) / group);
  return units <= 0x7fffffffll - kWarps ? static_cast<unsigned>((units + kWarps - 1) / kWarps) : 0u;
}

// `a`: a power of two; rows of a type begin at a multiple of its size
inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

template <int N>
struct IntTag {
  static constexpr int value = N;
};

// Calls f(type, access form, group, divisor for a row's groups) for rows of `width` columns.
template <typename F>
int launch(int32_t dtype, bool vec, int32_t width, F&& f) {
  int sms = 0;
  const int rc = device_ready(&sms);
  if (rc != KF_OK) return rc;
  return dispatch_rows(dtype, vec, [&](auto t, auto v) {
           const int slices = (width + kSlice - 1) / kSlice;
           if (pairs_of_slices(slices))
             f(t, v, IntTag<2>{}, divisor_of((slices + 1) / 2));
           else
             f(t, v, IntTag<1>{}, divisor_of(slices));
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
  if (!x || !codes || !exponents || !grid || !aligned(x, elem_bytes(dtype))) return KF_ERR_INVALID_ARGUMENT;
  const bool vec = vec_rows(x, x_stride, width, dtype) && aligned(codes, 8);
  return launch(dtype, vec, width, [&](auto t, auto v, auto g, const Divisor& by) {
    using E = ElemOf<decltype(t)>;
    pack8_kernel<E, decltype(v)::value, decltype(g)::value><<<grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const E*>(x), x_stride, num_rows, width, by, static_cast<uint8_t*>(codes),
        static_cast<uint8_t*>(exponents));
  });
}

int kf_restore8(const void* codes, const void* exponents, int32_t dtype, int32_t num_rows, int32_t width,
                const int32_t* pair_row, const int32_t* row_pair, int32_t top_k, int32_t out_rows, void* output,
                void* stream) {
  if (!valid_rows(num_rows, width, dtype) || !valid_rows(out_rows, width, dtype)) return KF_ERR_INVALID_ARGUMENT;
  if (num_rows > 0 && (!codes || !exponents)) return KF_ERR_INVALID_ARGUMENT;
  const bool sorted = top_k != 0;
  if (sorted ? (top_k < 1 || top_k > KF_SORT_MAX_TOP_K || !valid_tokens(num_rows) || (num_rows > 0 && !pair_row) ||
                (out_rows > 0 && !row_pair))
             : out_rows != num_rows)
    return KF_ERR_INVALID_ARGUMENT;
  if (out_rows == 0) return KF_OK;
  const unsigned grid = grid_of(num_rows, width);
  if (!output || (num_rows > 0 && !grid) || !aligned(output, elem_bytes(dtype))) return KF_ERR_INVALID_ARGUMENT;
  const bool vec = vec_rows(output, width, width, dtype) && aligned(codes, 8);
  return launch(dtype, vec, width, [&](auto t, auto v, auto g, const Divisor& by) {
    using E = ElemOf<decltype(t)>;
    const uint8_t* c = static_cast<const uint8_t*>(codes);
    const uint8_t* e = static_cast<const uint8_t*>(exponents);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (sorted) {
      const ScatterPlan p = plan_scatter((width + kSlice - 1) / kSlice, 2);
      const unsigned token_blocks = (num_rows + p.tokens - 1) / p.tokens, zero_blocks = zero_blocks_for(out_rows);
      restore8_sorted_kernel<E, decltype(v)::value><<<zero_blocks + token_blocks, p.warps * p.tokens * 32, 0, s>>>(
          c, e, num_rows, width, pair_row, row_pair, top_k, out_rows, p.warps, p.tokens, zero_blocks,
          static_cast<E*>(output));
    } else {
      restore8_kernel<E, decltype(v)::value, decltype(g)::value><<<grid, kThreads, 0, s>>>(c, e, num_rows, width, by,
                                                                                     static_cast<E*>(output));
    }
  });
}

int kf_swiglu_pack8(const void* h, int32_t dtype, int64_t h_stride, int32_t num_rows, int32_t inter, void* act,
                    void* codes, void* exponents, void* stream) {
  if (!valid_rows(num_rows, inter, dtype) || h_stride < 0) return KF_ERR_INVALID_ARGUMENT;
  if (num_rows == 0) return KF_OK;
  const unsigned grid = grid_of(num_rows, inter);
  if (!h || !act || !codes != !exponents || !grid) return KF_ERR_INVALID_ARGUMENT;
  if (!aligned(h, elem_bytes(dtype)) || !aligned(act, elem_bytes(dtype))) return KF_ERR_INVALID_ARGUMENT;
  const bool vec = vec_rows(h, h_stride, inter, dtype) && vec_rows(act, inter, inter, dtype) && aligned(codes, 8);
  return launch(dtype, vec, inter, [&](auto t, auto v, auto g, const Divisor& by) {
    using E = ElemOf<decltype(t)>;
    swiglu_pack8_kernel<E, decltype(v)::value, decltype(g)::value><<<grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const E*>(h), h_stride, num_rows, inter, by, static_cast<E*>(act), static_cast<uint8_t*>(codes),
        static_cast<uint8_t*>(exponents));
  });
}

int kf_swiglu_backward8(const void* codes, const void* exponents, const void* grad_act, int32_t dtype,
                        int64_t grad_stride, int32_t num_rows, int32_t inter, void* grad_h, void* act, void* stream) {
  if (!valid_rows(num_rows, inter, dtype) || grad_stride < 0) return KF_ERR_INVALID_ARGUMENT;
  if (num_rows == 0) return KF_OK;
  const unsigned grid = grid_of(num_rows, inter);
  if (!codes || !exponents || !grad_act || !grad_h || !grid) return KF_ERR_INVALID_ARGUMENT;
  if (!aligned(grad_act, elem_bytes(dtype)) || !aligned(grad_h, elem_bytes(dtype)) || !aligned(act, elem_bytes(dtype)))
    return KF_ERR_INVALID_ARGUMENT;
  const bool vec = vec_rows(grad_act, grad_stride, inter, dtype) && vec_rows(grad_h, inter, inter, dtype) &&
                   (!act || vec_rows(act, inter, inter, dtype)) && aligned(codes, 8);
  return launch(dtype, vec, inter, [&](auto t, auto v, auto g, const Divisor& by) {
    using E = ElemOf<decltype(t)>;
    swiglu_backward8_kernel<E, decltype(v)::value, decltype(g)::value><<<grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(exponents), static_cast<const E*>(grad_act),
        grad_stride, num_rows, inter, by, static_cast<E*>(grad_h), static_cast<E*>(act));
  });
}

}  // extern "C"
