// Tokens sorted by expert and back, for rows of bf16, fp16 or fp32.
//
//   order     a stable counting sort of the (token, choice) pairs by local expert:
//             a pair's row = its expert's segment start + the expert's pairs before it
//   scatter   rows[pair_row[t,k]] = x[t], zeros in the rows of no pair
//   combine   out[t] = sum_k w[t,k] rows[pair_row[t,k]], k ascending, fp32, one
//             rounding; without weights it is the gradient of the sort
//   backward  drows[r] = w[p] dout[t], dw[t,k] = <dout[t], rows[pair_row[t,k]]>
//
// A sort is one launch when it is small, else placing (after a histogram, for many
// pairs) and the scatter, chained by programmatic launches.  In the 16-byte forms all
// but the order (some 9 us at 32768 pairs, of them 3 us histogram) is bound by memory:
// every row is read or written once, in large calls at 5.5 to 6.8 TB/s where a plain
// copy reaches 6.55.  Rows off 16 bytes run at 2.3 to 4.9 TB/s in 16-bit types (the
// narrow ones slowest) and 5.5 to 6.6 in fp32.
//
// The reference sorts and combines inside its kernel() only, for its own FP8
// layer and without gradients (solution/triton/kernel.py:46-82, :1920-1925).
#include <algorithm>
#include <atomic>

#include "kf_elem.cuh"
#include "kf_internal.cuh"
#include "kf_ptx.cuh"

namespace kf {
namespace {

constexpr int kPlaceThreads = 1024;
constexpr int kPlaceWarps = kPlaceThreads / 32;
constexpr int kHistThreads = 1024;
constexpr int kMaxChunks = 64;   // histogram chunks of a large call: what each block of the placing kernel sums
// Calls of at most this many pairs need no histogram kernel: counting all ids in every
// block costs as much as the launch at 12000 pairs (a sort of 64-column rows 9.5 against
// 9.8 us), less below (7.2 against 8.2 us at 8800) and more above (12.3 against 10.3 us at 32768).
constexpr int kDirectPairs = 12288;

__device__ __forceinline__ int local_expert(int id, int offset, int E) {
  const unsigned le = static_cast<unsigned>(id) - static_cast<unsigned>(offset);
  return id >= 0 && le < static_cast<unsigned>(E) ? static_cast<int>(le) : -1;
}

// Tokens per histogram chunk, and chunks (0: the placing kernel counts the pairs itself).
struct OrderPlan {
  int chunk_tokens, nchunk;
};

inline OrderPlan plan_order(int T, int K) {
  if (static_cast<int64_t>(T) * K <= kDirectPairs) return OrderPlan{T, 0};
  const int least = (1024 + K - 1) / K, even = (T + kMaxChunks - 1) / kMaxChunks;
  const int ct = least > even ? least : even;
  return OrderPlan{ct, (T + ct - 1) / ct};
}

// hist[c][e] = pairs of local expert e among the tokens of chunk c.  2.7 us at 32768 or 131072 pairs.
__global__ void __launch_bounds__(kHistThreads) order_hist_kernel(const int32_t* __restrict__ ids, int n, int E,
                                                                  int offset, int chunk_pairs,
                                                                  int32_t* __restrict__ hist) {
  grid_dep_trigger();
  __shared__ int32_t h[kEG];
  if (threadIdx.x < kEG) h[threadIdx.x] = 0;
  __syncthreads();
  const int p0 = blockIdx.x * chunk_pairs, p1 = min(n, p0 + chunk_pairs);
  for (int p = p0 + threadIdx.x; p < p1; p += kHistThreads) {
    const int e = local_expert(ids[p], offset, E);
    if (e >= 0) atomicAdd(&h[e], 1);
  }
  __syncthreads();
  if (threadIdx.x < E) hist[static_cast<size_t>(blockIdx.x) * E + threadIdx.x] = h[threadIdx.x];
}

// Row q of those without a pair: zero_first[e] is the first such row of expert e's segment (entry kEG: of the
// buffer's rest), zero_upto[e] how many there are up to its end.
__device__ __forceinline__ int64_t zero_row(const int32_t* zero_first, const int32_t* zero_upto, int q) {
  int lo = 0, hi = kEG;   // the first entry whose zero_upto is above q
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (zero_upto[mid] > q) hi = mid; else lo = mid + 1;
  }
  return static_cast<int64_t>(zero_first[lo]) + q - (lo > 0 ? zero_upto[lo - 1] : 0);
}

struct PlaceArgs {
  const int32_t* ids;
  const int32_t* hist;   // [nchunk][E]
  int T, K, H, E, offset, align, R;
  int chunk_tokens, nchunk;
  int64_t stride;        // elements between rows of x
  int32_t *pair_row, *row_pair, *counts, *starts;
};

// Places the pairs: block b owns the tokens [b T / G, (b + 1) T / G).
//
// Counting.  Each block finds, for every expert, the pairs of the whole call and
// those before its own first token: from the histogram's rows and the ids between
// the last chunk border and its first token, or in smaller calls from all ids.  So
// no block waits for another, and the order needs one launch or two.
// Ranks.  A pair's row is its expert's next row, plus the pairs of its expert in
// the block's earlier warps, plus those in lower lanes of its own warp: stable and
// without atomics on the order.
// Bound by latencies (ids, histogram, some ten block barriers): 6.2 us at 32768 pairs
// and 6.7 us at 131072, waiting for the histogram included.
__global__ void __launch_bounds__(kPlaceThreads, 1) place_tokens_kernel(const PlaceArgs a) {
  grid_dep_trigger();
  __shared__ int32_t total[kEG], before[kEG];        // before becomes the next row of each expert
  __shared__ int32_t zero_first[kEG + 1];            // first row of expert e's padding; the last entry: the buffer's rest
  __shared__ int32_t zero_upto[kEG + 1];             // padding rows of experts <= e
  __shared__ uint16_t warp_count[kPlaceWarps][kEG];
  __shared__ int32_t warp_sum[2][kEG / 32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = gridDim.x;
  const int t0 = static_cast<int>(static_cast<int64_t>(a.T) * blockIdx.x / G);
  const int t1 = static_cast<int>(static_cast<int64_t>(a.T) * (blockIdx.x + 1) / G);

  if (tid < kEG) total[tid] = before[tid] = 0;
  __syncthreads();
  const int first_pair = t0 * a.K;
  if (a.nchunk == 0) {
    const int n = a.T * a.K;
    for (int p = tid; p < n; p += kPlaceThreads) {
      const int e = local_expert(a.ids[p], a.offset, a.E);
      if (e >= 0) {
        atomicAdd(&total[e], 1);
        if (p < first_pair) atomicAdd(&before[e], 1);
      }
    }
  } else {
    const int c0 = t0 / a.chunk_tokens;
    for (int p = c0 * a.chunk_tokens * a.K + tid; p < first_pair; p += kPlaceThreads) {
      const int e = local_expert(a.ids[p], a.offset, a.E);
      if (e >= 0) atomicAdd(&before[e], 1);
    }
    grid_dep_wait();   // the histogram is complete
    const int e = tid & (kEG - 1);
    if (e < a.E) {
      int all = 0, bef = 0;
#pragma unroll 8
      for (int c = tid / kEG; c < a.nchunk; c += kPlaceThreads / kEG) {
        const int v = a.hist[static_cast<size_t>(c) * a.E + e];
        all += v;
        if (c < c0) bef += v;
      }
      atomicAdd(&total[e], all);
      atomicAdd(&before[e], bef);
    }
  }
  __syncthreads();

  // segments: inclusive scan of the padded counts over the experts, and of the padding inside the buffer
  int count = 0, padded = 0, incl = 0;
  if (tid < kEG) {
    count = total[tid];
    padded = (count + a.align - 1) / a.align * a.align;
    incl = padded;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += v;
    }
    if (lane == 31) warp_sum[0][warp] = incl;
  }
  __syncthreads();
  int pads = 0, pads_incl = 0;
  if (tid < kEG) {
    for (int w = 0; w < warp; ++w) incl += warp_sum[0][w];
    const int start = incl - padded;
    before[tid] += start;
    const int live_end = min(start + count, a.R), end = min(incl, a.R);
    pads = end - live_end;
    zero_first[tid] = live_end;
    if (blockIdx.x == 0 && tid < a.E) {
      a.counts[tid] = count;
      a.starts[tid] = min(start, a.R);
      if (tid == a.E - 1) a.starts[a.E] = end;
    }
    if (tid == kEG - 1) zero_first[kEG] = end;   // experts past E have no rows: the last one ends them all
    pads_incl = pads;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, pads_incl, off);
      if (lane >= off) pads_incl += v;
    }
    if (lane == 31) warp_sum[1][warp] = pads_incl;
  }
  __syncthreads();
  if (tid < kEG) {
    for (int w = 0; w < warp; ++w) pads_incl += warp_sum[1][w];
    zero_upto[tid] = pads_incl;
    if (tid == kEG - 1) zero_upto[kEG] = pads_incl + a.R - zero_first[kEG];
  }

  const int round_tokens = kPlaceThreads / a.K;
  for (int r0 = t0; r0 < t1; r0 += round_tokens) {
    const int ntok = min(round_tokens, t1 - r0), npair = ntok * a.K;
    const int nwarp = (npair + 31) / 32;
    for (int i = tid; i < nwarp * (kEG / 2); i += kPlaceThreads) reinterpret_cast<uint32_t*>(warp_count)[i] = 0u;
    __syncthreads();   // also: zero_upto and before
    const int p = r0 * a.K + tid;
    int e = -1, rank = 0;
    if (warp < nwarp) {
      e = tid < npair ? local_expert(a.ids[p], a.offset, a.E) : -1;
      const unsigned same = __match_any_sync(0xffffffffu, e);
      rank = __popc(same & ((1u << lane) - 1u));
      if (e >= 0 && rank == 0) warp_count[warp][e] = static_cast<uint16_t>(__popc(same));
    }
    __syncthreads();
    if (tid < kEG) {   // counts become the pairs in earlier warps; `before` moves on after the rows are read
      int run = 0;
      for (int w = 0; w < nwarp; ++w) {
        const int v = warp_count[w][tid];
        warp_count[w][tid] = static_cast<uint16_t>(run);
        run += v;
      }
      total[tid] = run;   // this round's pairs
    }
    __syncthreads();
    if (tid < npair) {
      int row = -1;
      if (e >= 0) {
        row = before[e] + warp_count[warp][e] + rank;
        if (row >= a.R) row = -1;
      }
      a.pair_row[p] = row;
      if (row >= 0) a.row_pair[row] = p;
    }
    __syncthreads();
    if (tid < kEG) before[tid] += total[tid];

  }

  __syncthreads();   // zero_upto (a block without tokens)
  const int zeros = zero_upto[kEG];
  for (int q = blockIdx.x * kPlaceThreads + tid; q < zeros; q += G * kPlaceThreads)
    a.row_pair[zero_row(zero_first, zero_upto, q)] = -1;
}

// Small calls (at most kSmallPairs pairs, few rows) in one launch.  Every block
// ranks all pairs -- a call's worth of ids is a few loads per thread -- and then
// copies its share of the (token, slice) units and zeroes its share of the rows
// without a pair; a warp's first unit is on its way from memory meanwhile.  With K = 8
// and bf16, against placing and scatter: 3.1 us against 6.4 us for one token of 7168
// columns, 3.4 against 7.0 for 16, 7.6 against 10.8 for 128, and 4.7 against 5.8 for
// 128 tokens of 64 columns.
constexpr int kSmallThreads = 256;
constexpr int kSmallPairs = 1024;

template <typename T, bool kVec>
__global__ void __launch_bounds__(kSmallThreads) sort_small_kernel(const PlaceArgs a, const T* __restrict__ x,
                                                                   T* __restrict__ rows) {
  constexpr int kWarps = kSmallThreads / 32, kRounds = kSmallPairs / kSmallThreads;
  __shared__ uint16_t warp_count[kSmallPairs / 32][kEG];
  __shared__ int32_t first[kEG], zero_first[kEG + 1], zero_upto[kEG + 1];
  __shared__ int32_t srow[kSmallPairs];
  __shared__ int2 warp_sum[kWarps];
  __shared__ int zeros;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n = a.T * a.K, nwarp = (n + 31) / 32;
  const int slices = (a.H + kSlice - 1) / kSlice, units = a.T * slices;
  const int gw = blockIdx.x * kWarps + warp, nw = gridDim.x * kWarps;

  Raw8<T> v = {};
  if (gw < units) {
    const int t = gw / slices, c = (gw - t * slices) * kSlice;
    v = load_raw8<T, kVec>(x + static_cast<int64_t>(t) * a.stride + c, a.H - c, lane);
  }
  int e[kRounds], rank[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int p = r * kSmallThreads + tid;
    e[r] = p < n ? local_expert(a.ids[p], a.offset, a.E) : -1;
  }
  for (int i = tid; i < nwarp * (kEG / 2); i += kSmallThreads) reinterpret_cast<uint32_t*>(warp_count)[i] = 0u;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    if (r * kSmallThreads >= n) break;
    const unsigned same = __match_any_sync(0xffffffffu, e[r]);
    rank[r] = __popc(same & ((1u << lane) - 1u));
    if (e[r] >= 0 && rank[r] == 0) warp_count[r * kWarps + warp][e[r]] = static_cast<uint16_t>(__popc(same));
  }
  __syncthreads();
  // thread e owns expert e: its pairs in earlier warps, its segment, and the rows without a pair up to its end
  static_assert(kSmallThreads == kEG, "a thread per expert");
  int count = 0;
  for (int w = 0; w < nwarp; ++w) {
    const int c = warp_count[w][tid];
    warp_count[w][tid] = static_cast<uint16_t>(count);
    count += c;
  }
  const int padded = (count + a.align - 1) / a.align * a.align;
  int2 incl = make_int2(padded, count);
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int px = __shfl_up_sync(0xffffffffu, incl.x, off), py = __shfl_up_sync(0xffffffffu, incl.y, off);
    if (lane >= off) {
      incl.x += px;
      incl.y += py;
    }
  }
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  for (int w = 0; w < warp; ++w) {
    incl.x += warp_sum[w].x;
    incl.y += warp_sum[w].y;
  }
  const int start = incl.x - padded, end = min(incl.x, a.R);
  const int live = start < a.R ? min(count, a.R - start) : 0;      // rows of this expert inside the buffer
  first[tid] = start;
  zero_first[tid] = min(start, a.R) + live;
  // the experts before this one lie inside the buffer if this one starts in it; those past the end have no rows to zero
  const int upto = start < a.R ? end - (incl.y - count + live) : 0x7fffffff;
  zero_upto[tid] = upto;
  if (tid == kEG - 1) {
    zero_first[kEG] = end;
    zero_upto[kEG] = 0x7fffffff;
    if (incl.x < a.R) zeros = a.R - incl.y;                        // everything fits, and the buffer's rest is empty
  }
  if (start < a.R && incl.x >= a.R) zeros = upto;                  // the expert at the buffer's end
  if (tid == 0 && a.R == 0) zeros = 0;
  if (blockIdx.x == 0 && tid < a.E) {
    a.counts[tid] = count;
    a.starts[tid] = min(start, a.R);
    if (tid == a.E - 1) a.starts[a.E] = end;
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int p = r * kSmallThreads + tid;
    if (p < n) {
      int row = -1;
      if (e[r] >= 0) {
        row = first[e[r]] + warp_count[r * kWarps + warp][e[r]] + rank[r];
        if (row >= a.R) row = -1;
      }
      srow[p] = row;
      if (blockIdx.x == 0) {
        a.pair_row[p] = row;
        if (row >= 0) a.row_pair[row] = p;
      }
    }
  }
  __syncthreads();
  for (int u = gw; u < units; u += nw) {
    const int t = u / slices, c = (u - t * slices) * kSlice;
    if (u != gw) v = load_raw8<T, kVec>(x + static_cast<int64_t>(t) * a.stride + c, a.H - c, lane);
    for (int k = 0; k < a.K; ++k) {
      const int row = srow[t * a.K + k];
      if (row >= 0) store_raw8<T, kVec>(rows + static_cast<int64_t>(row) * a.H + c, a.H - c, lane, v);
    }
  }
  const Raw8<T> z = {};
  const int nz = zeros;
  int q = gw / slices, s = gw - q * slices;
  while (q < nz) {
    const int64_t row = zero_row(zero_first, zero_upto, q);
    store_raw8<T, kVec>(rows + row * a.H + s * kSlice, a.H - s * kSlice, lane, z);
    if (s == 0 && lane == 0) a.row_pair[row] = -1;
    s += nw;
    q += s / slices;
    s %= slices;
  }
}

// ---------------------------------------------------------------- scatter --

// A token's rows and weights, lane k holding pair k's (row -1 and weight 0 without one).
struct PairLane {
  int row;
  float w;
};
// (No __restrict__: the order may come from the kernel before, which a block starts
// before it ends, so these loads must stay behind grid_dep_wait().)
__device__ __forceinline__ PairLane load_pair(const int32_t* pair_row, const float* weight, int64_t t, int K, int R,
                                              int lane) {
  PairLane p{-1, 0.f};
  if (lane < K) {
    p.row = pair_row[t * K + lane];
    if (p.row >= R) p.row = -1;
    if (p.row >= 0) p.w = weight ? weight[t * K + lane] : 1.f;
  }
  return p;
}

// rows[pair_row[t, k]] = x[t] (times weight[t, k] with kWeighted), zeros in the rows
// of no pair.  A block holds a token's row across its warps, two slices each, reads
// it once and stores it K times; one block per token and not a loop over tokens:
// blocks that start in token order keep each expert's segment filling in address
// order, which the memory wants (4096 tokens, K = 8, 14336-byte rows: 86 us
// against 99 us for blocks that stay and loop).  The first blocks zero the rows of no
// pair, which overlaps their stores with the other blocks' reads (last in the grid:
// 99 us against 88 us for 16384 tokens, 32 local experts and 24576 rows, a third empty).
template <typename T, bool kVec, bool kWeighted, int kPer>
__global__ void __launch_bounds__(kScatterWarps * 32) scatter_rows_kernel(
    const T* __restrict__ x, int64_t stride, const int32_t* pair_row, const int32_t* row_pair,
    const float* weight, int T_, int K, int H, int R, int warps, int tokens, unsigned zero_blocks,
    T* __restrict__ rows) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (blockIdx.x < zero_blocks) {
    grid_dep_wait();
    zero_rows<T, kVec>(row_pair, static_cast<int64_t>(T_) * K, blockIdx.x, zero_blocks, R, H, rows);
    return;
  }
  const int sub = warp / warps;
  const int64_t t = static_cast<int64_t>(blockIdx.x - zero_blocks) * tokens + sub;
  const bool live = t < T_;
  grid_dep_wait();
  PairLane mine{-1, 0.f};
  if (live) mine = load_pair(pair_row, weight, t, K, R, lane);
  if (!__any_sync(0xffffffffu, mine.row >= 0)) return;   // a token of other ranks' experts: its row is not read
  for (int c = (warp - sub * warps) * kSlice; c < H; c += kPer * warps * kSlice) {
    Raw8<T> v[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int ci = c + i * warps * kSlice;
      v[i] = load_raw8<T, kVec>(x + t * stride + ci, H - ci, lane);
    }
    for (int k = 0; k < K; ++k) {
      const int row = __shfl_sync(0xffffffffu, mine.row, k);
      if (row < 0) continue;
      const float w = __shfl_sync(0xffffffffu, mine.w, k);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int ci = c + i * warps * kSlice;
        T* dst = rows + static_cast<int64_t>(row) * H + ci;
        if constexpr (kWeighted) {
          float f[8];
          to_floats(v[i], f);
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] *= w;
          store_raw8<T, kVec>(dst, H - ci, lane, from_floats<T>(f));
        } else {
          store_raw8<T, kVec>(dst, H - ci, lane, v[i]);
        }
      }
    }
  }
}

template <typename T, bool kVec, bool kWeighted>
cudaError_t launch_scatter(const void* x, int64_t stride, const int32_t* pair_row, const int32_t* row_pair,
                           const float* weight, int T_, int K, int H, int R, void* rows, bool chained, cudaStream_t s) {
  constexpr int kPer = 2;   // four: 107 us against 105 us for the sort of 4096 tokens
  const ScatterPlan p = plan_scatter((H + kSlice - 1) / kSlice, kPer);
  const int nwarp = p.warps * p.tokens;
  const unsigned token_blocks = (static_cast<unsigned>(T_) + p.tokens - 1) / p.tokens;
  const unsigned zero_blocks = zero_blocks_for(R);
  const dim3 grid(token_blocks + zero_blocks), block(nwarp * 32);
  if (grid.x == 0) return cudaSuccess;
  auto* kernel = scatter_rows_kernel<T, kVec, kWeighted, kPer>;
  if (chained)
    return launch_chained(kernel, grid, block, 0, s, static_cast<const T*>(x), stride, pair_row, row_pair, weight, T_, K,
                          H, R, p.warps, p.tokens, zero_blocks, static_cast<T*>(rows));
  kernel<<<grid, block, 0, s>>>(static_cast<const T*>(x), stride, pair_row, row_pair, weight, T_, K, H, R, p.warps,
                                p.tokens, zero_blocks, static_cast<T*>(rows));
  return cudaGetLastError();
}

// ---------------------------------------------------------------- combine --

// ---- the pipelined forms, for 16-byte rows ----
//
// Both directions read every pair's row once (K times the output) and are bound by
// memory.  A warp's step is a slice of a token: its loads -- up to eight rows, and the
// output's gradient in the backward pass -- go by cp.async straight to shared memory,
// into the lane's own 16-byte slots, so they need no barrier and hold no registers.

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// A slot row is 512 bytes per 16-byte access of a warp (one for 16-bit types, two for fp32).
template <typename T>
constexpr int kHalves = static_cast<int>(sizeof(T)) / 2;

// Starts the copy of a slice (at column c of `row`, null for none) into a slot row; the rest of it becomes zeros.
template <typename T>
__device__ __forceinline__ void slot_copy(uint32_t slot, const T* row, const T* any, int c, int H, int lane) {
#pragma unroll
  for (int h = 0; h < kHalves<T>; ++h) {
    const int col = c + vec_col<T>(lane, h);
    const bool live = row != nullptr && col < H;
    cp_async16(slot + h * 512, live ? row + col : any, live);
  }
}

// This lane's eight elements of a slot row.
template <typename T>
__device__ __forceinline__ Raw8<T> slot_load(const uint4* slot) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < kHalves<T>; ++i) {
    const uint4 q = slot[i * 32];
    r.x[4 * i] = q.x;
    r.x[4 * i + 1] = q.y;
    r.x[4 * i + 2] = q.z;
    r.x[4 * i + 3] = q.w;
  }
  return r;
}

struct CombineArgs {
  const void* rows;
  const void* dout;        // backward
  const int32_t* pair_row;
  const int32_t* row_pair; // backward with drows
  const float* weight;
  void* out;               // forward: output; backward: drows or null
  float* dweight;
  int64_t stride;
  int T, K, H, R;
};

// Forward.  A block of up to 14 warps (7 for fp32) stays and loops over tokens, on each
// SM as many blocks as make about that many warps of eight rows (one block at 7168
// columns); each warp sums one step while the next one's rows arrive, and the pairs of
// the token after that are on their way.  Measured (K = 8, bf16; 4096 tokens of 7168
// columns and 16384 of 2048): 81 and 90 us = 6.5 and 6.7 TB/s, against 94 and 106 us with
// the rows loaded to registers; fp32, 4096 tokens of 7168 columns: 155 us = 6.8 TB/s.
constexpr int kForwardStages = 2;
template <typename T>
constexpr int kForwardWarps = sizeof(T) == 4 ? 7 : 14;

// kRows rows per step, kBatches steps per slice (K <= kRows * kBatches).
template <typename T, int kRows, int kBatches>
__global__ void __launch_bounds__(kForwardWarps<T> * 32) combine_pipe_kernel(const CombineArgs a) {
  constexpr int kStages = kForwardStages;
  constexpr int kStep = kRows * kHalves<T>;                  // 512-byte slots of a step
  extern __shared__ __align__(16) uint4 pipe_smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = blockDim.x >> 5;
  const uint4* mine = pipe_smem + static_cast<size_t>(warp) * kStages * kStep * 32 + lane;
  const uint32_t mine_s = smem_u32(mine);
  const T* rows = static_cast<const T*>(a.rows);
  const int slices = (a.H + kSlice - 1) / kSlice;

  // the stream of steps to issue, kStages - 1 ahead of the ones summed: token, slice, batch;
  // and the pairs of its token, of the token before it (being summed while the stream
  // is one step into the next) and of the token after it (on their way: looked at only
  // when the stream gets there, as a warp waits at a load's first use)
  int it = blockIdx.x, is = warp, ib = 0;
  auto after = [&](int t) { return t + gridDim.x < static_cast<unsigned>(a.T) ? static_cast<int>(t + gridDim.x) : a.T; };
  auto fetch = [&](int t) {
    PairLane p{-1, 1.f};
    if (t < a.T && lane < a.K) {
      p.row = a.pair_row[static_cast<int64_t>(t) * a.K + lane];
      if (a.weight) p.w = a.weight[static_cast<int64_t>(t) * a.K + lane];
    }
    return p;
  };
  auto checked = [&](PairLane p) { return p.row >= 0 && p.row < a.R ? p : PairLane{-1, 0.f}; };
  PairLane before{-1, 0.f}, now = fetch(it), next = fetch(after(it));
  now = checked(now);
  auto issue = [&](int stage) {
    if (it < a.T) {
      const uint32_t dst = mine_s + stage * kStep * 512;
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        const int row = __shfl_sync(0xffffffffu, now.row, ib * kRows + j);
        slot_copy<T>(dst + j * kHalves<T> * 512, row >= 0 ? rows + static_cast<int64_t>(row) * a.stride : nullptr, rows,
                     is * kSlice, a.H, lane);
      }
      if (++ib == kBatches) {
        ib = 0;
        is += W;
        if (is >= slices) {
          is = warp;
          it = after(it);
          before = now;
          now = checked(next);
          next = fetch(after(it));
        }
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) issue(i);

  int stage = 0;
  for (int t = blockIdx.x; t < a.T; t += gridDim.x) {
    const PairLane pair = it == t ? now : before;
    for (int sl = warp; sl < slices; sl += W) {
      const int c = sl * kSlice;
      float acc[8] = {};
#pragma unroll
      for (int b = 0; b < kBatches; ++b) {
        issue(stage == 0 ? kStages - 1 : stage - 1);
        cp_async_wait<kStages - 1>();   // the oldest step's copies, all of this lane's own
        const uint4* slot = mine + stage * kStep * 32;
#pragma unroll
        for (int j = 0; j < kRows; ++j) {
          const float w = __shfl_sync(0xffffffffu, pair.w, b * kRows + j);
          float f[8];
          to_floats(slot_load<T>(slot + j * kHalves<T> * 32), f);
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[i] = fmaf(w, f[i], acc[i]);
        }
        stage = stage + 1 == kStages ? 0 : stage + 1;
      }
      store_raw8<T, true>(static_cast<T*>(a.out) + static_cast<int64_t>(t) * a.H + c, a.H - c, lane, from_floats<T>(acc));
    }
  }
  cp_async_wait<0>();
}

// Backward.  One block of up to seven warps per token, in token order, and not blocks
// that stay: what it stores, K rows for one, then fills the experts' segments in
// address order (as in scatter_rows_kernel).  The blocks of an SM overlap each other;
// a warp with several steps issues the next before it sums one.  The first blocks
// zero the rows without a pair.  Measured (K = 8, bf16; 4096 tokens of 7168 columns,
// 16384 of 2048): 162 to 169 and 180 us = 6.2 to 6.5 and 6.4 TB/s, against 171 and 205
// us for blocks that stay and 202 and 239 us with the rows loaded to registers; 14 warps
// and one stage: 174 and 193 us.  fp32, 4096 tokens of 7168 columns: 329 us = 6.4 TB/s.
constexpr int kBackwardStages = 2;
constexpr int kBackwardWarps = 7;

template <typename T, int kRows, int kBatches>
__global__ void __launch_bounds__(kBackwardWarps * 32)
    combine_backward_pipe_kernel(const CombineArgs a, int stages, unsigned zero_blocks) {
  constexpr int kStages = kBackwardStages;
  constexpr int kStep = (kRows + 1) * kHalves<T>;            // the last slot row: the output's gradient
  extern __shared__ __align__(16) uint4 pipe_smem[];
  __shared__ float part[kBackwardWarps][kRows * kBatches];
  T* drows = static_cast<T*>(a.out);
  if (blockIdx.x < zero_blocks) {
    zero_rows<T, true>(a.row_pair, static_cast<int64_t>(a.T) * a.K, blockIdx.x, zero_blocks, a.R, a.H, drows);
    return;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = blockDim.x >> 5;
  const uint4* mine = pipe_smem + static_cast<size_t>(warp) * stages * kStep * 32 + lane;   // stages in use
  const uint32_t mine_s = smem_u32(mine);
  const T* rows = static_cast<const T*>(a.rows);
  const int64_t t = blockIdx.x - zero_blocks;
  const T* dout = static_cast<const T*>(a.dout) + t * a.H;
  const int slices = (a.H + kSlice - 1) / kSlice;
  const PairLane pair = load_pair(a.pair_row, a.weight, t, a.K, a.R, lane);
  const int out_row = drows ? pair.row : -1;   // where this lane's pair is stored

  int is = warp, ib = 0;
  auto issue = [&](int stage) {
    if (is < slices) {
      const uint32_t dst = mine_s + stage * kStep * 512;
      slot_copy<T>(dst + kRows * kHalves<T> * 512, dout, dout, is * kSlice, a.H, lane);
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        const int row = __shfl_sync(0xffffffffu, pair.row, ib * kRows + j);
        slot_copy<T>(dst + j * kHalves<T> * 512, row >= 0 ? rows + static_cast<int64_t>(row) * a.stride : nullptr, dout,
                     is * kSlice, a.H, lane);
      }
      if (++ib == kBatches) {
        ib = 0;
        is += W;
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) issue(i);

  int stage = 0;
  float dot[kBatches][kRows] = {};
  for (int sl = warp; sl < slices; sl += W) {
    const int c = sl * kSlice, n = a.H - c;
#pragma unroll
    for (int b = 0; b < kBatches; ++b) {
      issue(stage == 0 ? kStages - 1 : stage - 1);
      cp_async_wait<kStages - 1>();
      const uint4* slot = mine + stage * kStep * 32;
      float g[8];
      to_floats(slot_load<T>(slot + kRows * kHalves<T> * 32), g);
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        const int row = __shfl_sync(0xffffffffu, out_row, b * kRows + j);
        const float w = __shfl_sync(0xffffffffu, pair.w, b * kRows + j);
        float f[8];
        to_floats(slot_load<T>(slot + j * kHalves<T> * 32), f);
#pragma unroll
        for (int i = 0; i < 8; ++i) dot[b][j] = fmaf(g[i], f[i], dot[b][j]);
        if (row >= 0) {
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = w * g[i];
          store_raw8<T, true>(drows + static_cast<int64_t>(row) * a.H + c, n, lane, from_floats<T>(f));
        }
      }
      stage = stage + 1 == kStages ? 0 : stage + 1;
    }
  }
#pragma unroll
  for (int b = 0; b < kBatches; ++b)
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      float d = dot[b][j];
#pragma unroll
      for (int off = 16; off >= 1; off >>= 1) d += __shfl_xor_sync(0xffffffffu, d, off);
      if (lane == 0) part[warp][b * kRows + j] = d;
    }
  cp_async_wait<0>();
  __syncthreads();
  if (static_cast<int>(threadIdx.x) < a.K) {
    float sum = 0.f;
    if (pair.row >= 0)   // lane k of warp 0 holds pair k
      for (int w = 0; w < W; ++w) sum += part[w][threadIdx.x];
    a.dweight[t * a.K + threadIdx.x] = sum;
  }
}

// Lets `kernel` use `bytes` of dynamic shared memory on the current device; `allowed` remembers the devices
// (a second thread that gets here first does the same again).
template <typename K>
cudaError_t allow_smem(K* kernel, int bytes, std::atomic<uint64_t>& allowed) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = uint64_t{1} << (dev & 63);
  if (dev < 64 && (allowed.load(std::memory_order_acquire) & bit)) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) allowed.fetch_or(bit, std::memory_order_release);
  return e;
}

// The warps, at most `most`, that share a row's slices evenly.
inline int warps_for(int H, int most) {
  const int slices = (H + kSlice - 1) / kSlice, steps = (slices + most - 1) / most;
  return (slices + steps - 1) / steps;
}

template <typename T, int kRows, int kBatches>
cudaError_t launch_pipe(const CombineArgs& a, int sms, cudaStream_t s) {
  constexpr int kWarps = kForwardWarps<T>, kWarpBytes = kForwardStages * kRows * kHalves<T> * 512;
  static std::atomic<uint64_t> allowed{0};
  auto* kernel = combine_pipe_kernel<T, kRows, kBatches>;
  const cudaError_t e = allow_smem(kernel, kWarpBytes * kWarps, allowed);
  if (e != cudaSuccess) return e;
  // blocks for about kWarps warps of eight rows on each SM
  const int warps = warps_for(a.H, kWarps), target = kWarps * 8 / kRows;
  const int grid = std::min(a.T, sms * std::max(1, (target + warps / 2) / warps));
  kernel<<<grid, warps * 32, kWarpBytes * warps, s>>>(a);
  return cudaGetLastError();
}

template <typename T, int kRows, int kBatches>
cudaError_t launch_backward_pipe(const CombineArgs& a, cudaStream_t s) {
  constexpr int kStageBytes = (kRows + 1) * kHalves<T> * 512;
  static std::atomic<uint64_t> allowed{0};
  auto* kernel = combine_backward_pipe_kernel<T, kRows, kBatches>;
  const cudaError_t e = allow_smem(kernel, kStageBytes * kBackwardStages * kBackwardWarps, allowed);
  if (e != cudaSuccess) return e;
  // a warp with a single step uses one stage: more blocks fit an SM
  const int warps = warps_for(a.H, kBackwardWarps), slices = (a.H + kSlice - 1) / kSlice;
  const int stages = slices * kBatches <= warps ? 1 : kBackwardStages;
  const unsigned zero_blocks = a.out ? zero_blocks_for(a.R) : 0u;
  kernel<<<zero_blocks + a.T, warps * 32, kStageBytes * stages * warps, s>>>(a, stages, zero_blocks);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_pipe(const CombineArgs& a, int sms, cudaStream_t s) {
  if (a.K <= 2) return launch_pipe<T, 2, 1>(a, sms, s);
  if (a.K <= 4) return launch_pipe<T, 4, 1>(a, sms, s);
  if (a.K <= 8) return launch_pipe<T, 8, 1>(a, sms, s);
  return launch_pipe<T, 8, 2>(a, sms, s);
}

template <typename T>
cudaError_t launch_backward_pipe(const CombineArgs& a, cudaStream_t s) {
  if (a.K <= 2) return launch_backward_pipe<T, 2, 1>(a, s);
  if (a.K <= 4) return launch_backward_pipe<T, 4, 1>(a, s);
  if (a.K <= 8) return launch_backward_pipe<T, 8, 1>(a, s);
  return launch_backward_pipe<T, 8, 2>(a, s);
}

// ---- the plain form, for rows of any alignment ----

inline unsigned blocks(int64_t items, int per) { return static_cast<unsigned>((items + per - 1) / per); }

constexpr int kRowWarps = 8;
template <typename T>
constexpr int kBatch = sizeof(T) == 4 ? 4 : 8;   // rows whose loads are in flight together

// One warp per (token, slice of 256 columns), consecutive warps on consecutive slices.
// 33 us = 2.3 TB/s for 4096 tokens of 1031 columns, K = 8, bf16 (rows between two words:
// bound by the shuffles; 25 us from the L2), 23 us for 1030 columns; 7167 columns 172 us
// = 3.1 TB/s; fp32 rows of 7164 columns 161 us = 6.6 TB/s.
template <typename T>
__global__ void __launch_bounds__(kRowWarps * 32) combine_kernel(const CombineArgs a) {
  const T* rows = static_cast<const T*>(a.rows);
  const int lane = threadIdx.x & 31;
  const unsigned slices = (a.H + kSlice - 1) / kSlice;
  const unsigned u = blockIdx.x * kRowWarps + (threadIdx.x >> 5);
  const int64_t t = u / slices;
  if (t >= a.T) return;
  const int c = static_cast<int>(u % slices) * kSlice, n = a.H - c;
  const PairLane mine = load_pair(a.pair_row, a.weight, t, a.K, a.R, lane);
  float acc[8] = {};
  for (int k0 = 0; k0 < a.K; k0 += kBatch<T>) {
    Raw8<T> v[kBatch<T>];
#pragma unroll
    for (int j = 0; j < kBatch<T>; ++j) {
      const int row = __shfl_sync(0xffffffffu, mine.row, k0 + j);   // lanes past K hold no row
      v[j] = load_raw8<T, false>(rows + static_cast<int64_t>(row < 0 ? 0 : row) * a.stride + c, row < 0 ? 0 : n, lane);
    }
#pragma unroll
    for (int j = 0; j < kBatch<T>; ++j) {
      const float w = __shfl_sync(0xffffffffu, mine.w, k0 + j);
      float f[8];
      to_floats(v[j], f);
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] = fmaf(w, f[i], acc[i]);
    }
  }
  store_raw8<T, false>(static_cast<T*>(a.out) + t * a.H + c, n, lane, from_floats<T>(acc));
}

// `warps` warps per token share its slices, `tokens` tokens per block.  The first
// blocks zero the rows without a pair.  61 us = 2.5 TB/s for 1031 columns, 43 us for
// 1030 columns, 295 us = 3.6 TB/s for 7167, fp32 352 us = 6.0 TB/s for 7164; with one
// element per access 1031 columns took 165 us.
template <typename T>
__global__ void __launch_bounds__(kRowWarps * 32) combine_backward_kernel(const CombineArgs a, int warps, int tokens,
                                                                          unsigned zero_blocks) {
  const T* rows = static_cast<const T*>(a.rows);
  const T* dout = static_cast<const T*>(a.dout);
  T* drows = static_cast<T*>(a.out);
  if (blockIdx.x < zero_blocks) {
    zero_rows<T, false>(a.row_pair, static_cast<int64_t>(a.T) * a.K, blockIdx.x, zero_blocks, a.R, a.H, drows);
    return;
  }
  __shared__ float part[kRowWarps][KF_SORT_MAX_TOP_K];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = warp / warps, w0 = warp - sub * warps;
  const int64_t t = static_cast<int64_t>(blockIdx.x - zero_blocks) * tokens + sub;
  const bool live = t < a.T;
  PairLane mine{-1, 0.f};
  if (live) mine = load_pair(a.pair_row, a.weight, t, a.K, a.R, lane);
  for (int k0 = 0; k0 < a.K; k0 += kBatch<T>) {
    float dot[kBatch<T>] = {};
    for (int c = w0 * kSlice; live && c < a.H; c += warps * kSlice) {
      const int n = a.H - c;
      Raw8<T> v[kBatch<T>];
      const Raw8<T> graw = load_raw8<T, false>(dout + t * a.H + c, n, lane);
#pragma unroll
      for (int j = 0; j < kBatch<T>; ++j) {
        const int row = __shfl_sync(0xffffffffu, mine.row, k0 + j);
        v[j] = load_raw8<T, false>(rows + static_cast<int64_t>(row < 0 ? 0 : row) * a.stride + c, row < 0 ? 0 : n, lane);
      }
      float g[8];
      to_floats(graw, g);
#pragma unroll
      for (int j = 0; j < kBatch<T>; ++j) {
        const int row = __shfl_sync(0xffffffffu, mine.row, k0 + j);
        const float w = __shfl_sync(0xffffffffu, mine.w, k0 + j);
        float f[8];
        to_floats(v[j], f);
#pragma unroll
        for (int i = 0; i < 8; ++i) dot[j] = fmaf(g[i], f[i], dot[j]);
        if (drows && row >= 0) {
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = w * g[i];
          store_raw8<T, false>(drows + static_cast<int64_t>(row) * a.H + c, n, lane, from_floats<T>(f));
        }
      }
    }
#pragma unroll
    for (int j = 0; j < kBatch<T>; ++j) {
#pragma unroll
      for (int off = 16; off >= 1; off >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], off);
      if (lane == 0 && k0 + j < a.K) part[warp][k0 + j] = dot[j];
    }
  }
  __syncthreads();
  if (live && w0 == 0 && lane < a.K) {
    float s = 0.f;
    if (mine.row >= 0)
      for (int w = 0; w < warps; ++w) s += part[warp + w][lane];
    a.dweight[t * a.K + lane] = s;
  }
}

template <typename T>
cudaError_t launch_combine(const CombineArgs& a, cudaStream_t s) {
  const int64_t units = static_cast<int64_t>(a.T) * ((a.H + kSlice - 1) / kSlice);
  combine_kernel<T><<<blocks(units, kRowWarps), kRowWarps * 32, 0, s>>>(a);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_combine_backward(const CombineArgs& a, cudaStream_t s) {
  // as many warps as share the slices evenly, kRowWarps at most
  const int slices = (a.H + kSlice - 1) / kSlice, steps = (slices + kRowWarps - 1) / kRowWarps;
  const int warps = (slices + steps - 1) / steps, tokens = kRowWarps / warps;
  const unsigned zero_blocks = a.out ? zero_blocks_for(a.R) : 0u;
  combine_backward_kernel<T>
      <<<zero_blocks + blocks(a.T, tokens), warps * tokens * 32, 0, s>>>(a, warps, tokens, zero_blocks);
  return cudaGetLastError();
}

bool valid_shape(int32_t T, int32_t K, int64_t H, int32_t dtype) {
  return valid_tokens(T) && K >= 1 && K <= KF_SORT_MAX_TOP_K && H >= 1 && H <= KF_SORT_MAX_WIDTH && valid_dtype(dtype);
}

// Rows of a type begin at a multiple of its size (a null pointer does).
bool elem_aligned(const void* p, int32_t dtype) { return reinterpret_cast<uintptr_t>(p) % elem_bytes(dtype) == 0; }

// Small calls (kSmallPairs) whose rows are at most this many bytes in all are sorted in
// one launch: above it the bandwidth of the scatter is worth the launch.
constexpr int64_t kSmallBytes = 16 << 20;

template <typename P>
using ElemOf = std::remove_const_t<std::remove_pointer_t<P>>;

inline int code(cudaError_t e) { return e == cudaSuccess ? KF_OK : KF_ERR_CUDA; }

}  // namespace
}  // namespace kf

using namespace kf;

extern "C" {

size_t kf_sort_workspace_bytes(int32_t num_tokens, int32_t top_k, int32_t num_experts) {
  if (!valid_tokens(num_tokens) || top_k < 1 || top_k > KF_SORT_MAX_TOP_K || num_experts < 1 || num_experts > kEG)
    return 0;
  const OrderPlan plan = plan_order(num_tokens, top_k);
  return static_cast<size_t>(plan.nchunk) * num_experts * sizeof(int32_t);
}

int kf_sort_tokens(const void* x, int32_t dtype, int64_t x_stride, const int32_t* topk_idx, int32_t num_tokens,
                   int32_t top_k, int32_t width, int32_t num_experts, int32_t expert_offset, int32_t row_align,
                   int32_t num_rows, void* rows, int32_t* pair_row, int32_t* row_pair, int32_t* counts,
                   int32_t* starts, void* workspace, size_t workspace_bytes, void* stream) {
  if (!valid_shape(num_tokens, top_k, width, dtype) || x_stride < 0) return KF_ERR_INVALID_ARGUMENT;
  if (num_experts < 1 || num_experts > kEG || expert_offset < 0 || expert_offset > kEG - num_experts)
    return KF_ERR_INVALID_ARGUMENT;
  if (row_align < 1 || row_align > KF_SORT_MAX_ALIGN || num_rows < 0 || num_rows > KF_SORT_MAX_ROWS ||
      num_rows % row_align)
    return KF_ERR_INVALID_ARGUMENT;
  if (!counts || !starts || (num_tokens > 0 && (!x || !topk_idx || !pair_row)) || (num_rows > 0 && (!rows || !row_pair)))
    return KF_ERR_INVALID_ARGUMENT;
  if (!elem_aligned(x, dtype) || !elem_aligned(rows, dtype)) return KF_ERR_INVALID_ARGUMENT;
  const size_t need = kf_sort_workspace_bytes(num_tokens, top_k, num_experts);
  if (need && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 3u))) return KF_ERR_INVALID_ARGUMENT;
  if (workspace_bytes < need) return KF_ERR_WORKSPACE_TOO_SMALL;
  int sms = 0;
  const int rc = device_ready(&sms);
  if (rc != KF_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const OrderPlan plan = plan_order(num_tokens, top_k);
  PlaceArgs a;
  a.ids = topk_idx;
  a.hist = static_cast<const int32_t*>(workspace);
  a.T = num_tokens;
  a.K = top_k;
  a.H = width;
  a.E = num_experts;
  a.offset = expert_offset;
  a.align = row_align;
  a.R = num_rows;
  a.chunk_tokens = plan.chunk_tokens;
  a.nchunk = plan.nchunk;
  a.stride = x_stride;
  a.pair_row = pair_row;
  a.row_pair = row_pair;
  a.counts = counts;
  a.starts = starts;
  if (plan.nchunk) {
    order_hist_kernel<<<plan.nchunk, kHistThreads, 0, s>>>(topk_idx, num_tokens * top_k, num_experts, expert_offset,
                                                           plan.chunk_tokens * top_k, static_cast<int32_t*>(workspace));
    if (cudaGetLastError() != cudaSuccess) return KF_ERR_CUDA;
  }
  const int slices = (width + kSlice - 1) / kSlice;
  const bool vec = vec_rows(x, x_stride, width, dtype) && vec_rows(rows, width, width, dtype);
  const bool small = num_tokens * top_k <= kSmallPairs &&
                     static_cast<int64_t>(num_rows) * width * static_cast<int64_t>(elem_bytes(dtype)) <= kSmallBytes;
  return code(dispatch_rows(dtype, vec, [&](auto t, auto v) {
    using E = ElemOf<decltype(t)>;
    constexpr bool kVec = decltype(v)::value;
    if (small) {
      // a unit per warp, and up to eight of zeroing; two blocks per SM at most
      const int64_t units = std::max<int64_t>(static_cast<int64_t>(num_tokens) * slices,
                                              static_cast<int64_t>(num_rows) * slices / 8);
      const int grid = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(2 * sms, (units + 7) / 8)));
      sort_small_kernel<E, kVec><<<grid, kSmallThreads, 0, s>>>(a, static_cast<const E*>(x), static_cast<E*>(rows));
      return cudaGetLastError();
    }
    cudaError_t e;
    const int grid = std::min(sms, std::max(1, num_tokens));
    if (plan.nchunk) {
      e = launch_chained(place_tokens_kernel, dim3(grid), dim3(kPlaceThreads), 0, s, a);
    } else {
      place_tokens_kernel<<<grid, kPlaceThreads, 0, s>>>(a);
      e = cudaGetLastError();
    }
    if (e != cudaSuccess) return e;
    return launch_scatter<E, kVec, false>(x, x_stride, pair_row, row_pair, nullptr, num_tokens, top_k, width, num_rows,
                                          rows, true, s);
  }));
}

int kf_combine_tokens(const void* rows, int32_t dtype, int64_t rows_stride, int32_t num_rows, const int32_t* pair_row,
                      const float* topk_weight, int32_t num_tokens, int32_t top_k, int32_t width, void* output,
                      void* stream) {
  if (!valid_shape(num_tokens, top_k, width, dtype) || num_rows < 0 || num_rows > KF_SORT_MAX_ROWS || rows_stride < 0)
    return KF_ERR_INVALID_ARGUMENT;
  if (num_tokens == 0) return KF_OK;
  if (!pair_row || !output || (num_rows > 0 && !rows)) return KF_ERR_INVALID_ARGUMENT;
  if (!elem_aligned(rows, dtype) || !elem_aligned(output, dtype)) return KF_ERR_INVALID_ARGUMENT;
  const int64_t units = static_cast<int64_t>(num_tokens) * ((width + kSlice - 1) / kSlice);
  if (units > 0xffffffffll - kRowWarps) return KF_ERR_INVALID_ARGUMENT;   // rows of terabytes
  int sms = 0;
  const int rc = device_ready(&sms);
  if (rc != KF_OK) return rc;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (num_rows == 0)   // no pair has a row
    return code(cudaMemsetAsync(output, 0, static_cast<size_t>(num_tokens) * width * elem_bytes(dtype), s));
  const bool vec = vec_rows(rows, rows_stride, width, dtype) && vec_rows(output, width, width, dtype);
  const CombineArgs a{rows,   nullptr, pair_row,    nullptr,    topk_weight, output,
                      nullptr, rows_stride, num_tokens, top_k, width,       num_rows};
  return code(dispatch_rows(dtype, vec, [&](auto t, auto v) {
    using E = ElemOf<decltype(t)>;
    constexpr bool kVec = decltype(v)::value;
    if constexpr (kVec)
      return launch_pipe<E>(a, sms, s);
    else
      return launch_combine<E>(a, s);
  }));
}

int kf_combine_backward(const void* grad_output, const void* rows, int32_t dtype, int64_t rows_stride, int32_t num_rows,
                        const int32_t* pair_row, const int32_t* row_pair, const float* topk_weight, int32_t num_tokens,
                        int32_t top_k, int32_t width, void* grad_rows, float* grad_weight, void* stream) {
  if (!valid_shape(num_tokens, top_k, width, dtype) || num_rows < 0 || num_rows > KF_SORT_MAX_ROWS || rows_stride < 0)
    return KF_ERR_INVALID_ARGUMENT;
  if (num_tokens > 0 && (!grad_output || !pair_row)) return KF_ERR_INVALID_ARGUMENT;
  if (grad_weight && num_rows > 0 && !rows) return KF_ERR_INVALID_ARGUMENT;
  if (grad_rows && num_rows > 0 && !row_pair) return KF_ERR_INVALID_ARGUMENT;
  if (!elem_aligned(grad_output, dtype) || !elem_aligned(rows, dtype) || !elem_aligned(grad_rows, dtype))
    return KF_ERR_INVALID_ARGUMENT;
  if (num_rows == 0) grad_rows = nullptr;
  if (num_tokens == 0) grad_weight = nullptr;
  if (!grad_weight && !grad_rows) return KF_OK;
  int sms = 0;
  const int rc = device_ready(&sms);
  if (rc != KF_OK) return rc;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (num_rows == 0)
    return code(cudaMemsetAsync(grad_weight, 0, static_cast<size_t>(num_tokens) * top_k * sizeof(float), s));
  const bool vec = vec_rows(grad_output, width, width, dtype) && (!grad_weight || vec_rows(rows, rows_stride, width, dtype)) &&
                   (!grad_rows || vec_rows(grad_rows, width, width, dtype));
  return code(dispatch_rows(dtype, vec, [&](auto t, auto v) {
    using E = ElemOf<decltype(t)>;
    constexpr bool kVec = decltype(v)::value;
    if (!grad_weight)   // the rows are not read: scatter the weighted gradient
      return launch_scatter<E, kVec, true>(grad_output, width, pair_row, row_pair, topk_weight, num_tokens, top_k, width,
                                           num_rows, grad_rows, false, s);
    const CombineArgs a{rows,        grad_output, pair_row,   row_pair, topk_weight, grad_rows,
                        grad_weight, rows_stride, num_tokens, top_k,    width,       num_rows};
    if constexpr (kVec)
      return launch_backward_pipe<E>(a, s);
    else
      return launch_combine_backward<E>(a, s);
  }));
}

}  // extern "C"
