// Gradient of the routing weights with respect to the routing logits.
//
// With s_k = sigmoid(logit of the k-th chosen expert), S = sum_k s_k + 1e-20 and
// w_k = f s_k / S (the routing of route_kernel; reference
// solution/triton/kernel.py:1861-1867), and g = dL/dw:
//
//   dL/dlogit_k = f (s_k / S) (1 - s_k) (g_k - sum_j g_j s_j / S)
//
// and zero for every other expert: the choice itself has no gradient, and the
// bias enters the choice only.  The sigmoids are taken again from the logits.
//
// Four tokens per warp, eight lanes each: lane 8 i + k holds choice k of token i.
// The warp first zeroes its four rows of 256 gradients, 512 bytes per store, and
// after a warp barrier each lane stores its choice's gradient into its row.
// (Every lane of a warp per token comparing its own eight columns with the eight
// ids was bound by issuing those compares: 6.8 us against 5.0 us at 16384 tokens.)
#include "kf_internal.cuh"

namespace kf {
namespace {

constexpr int kThreads = 256;
constexpr int kTokens = 4;   // per warp

__global__ void __launch_bounds__(kThreads) route_backward_kernel(const float* __restrict__ logits,
                                                                  const int32_t* __restrict__ topk_idx,
                                                                  const float* __restrict__ grad_w, int T, float rsf,
                                                                  float* __restrict__ grad_logits) {
  const int lane = threadIdx.x & 31;
  const int64_t t0 = (static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5)) * kTokens;
  const int64_t t = t0 + (lane >> 3);
  if (t0 >= T) return;
  const bool live = t < T;
  int e = live ? topk_idx[t * kTopK + (lane & 7)] : -1;
  float g = live ? grad_w[t * kTopK + (lane & 7)] : 0.f;
  if (e < 0 || e >= kEG) {   // no choice
    e = -1;
    g = 0.f;
  }
  const float x = e >= 0 ? logits[t * kEG + e] : 0.f;
  const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < kTokens; ++i) {
    if (t0 + i < T) {
      float4* row = reinterpret_cast<float4*>(grad_logits + (t0 + i) * kEG);
      row[lane] = zero;
      row[32 + lane] = zero;
    }
  }
  const float s = e >= 0 ? 1.0f / (1.0f + expf(-x)) : 0.f;
  const float c = 1.0f / (1.0f + expf(x));   // 1 - s without the cancellation
  float sum = s;
#pragma unroll
  for (int off = 4; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  const float p = s / (sum + 1e-20f);
  float mean = g * p;
#pragma unroll
  for (int off = 4; off >= 1; off >>= 1) mean += __shfl_xor_sync(0xffffffffu, mean, off);
  float d = rsf * p * c * (g - mean);
  // an id that a token repeats (outside the routing's contract) gets the sum of its gradients, from its first lane
  const unsigned mine = 0xffu << (lane & 24);
  const unsigned same = __match_any_sync(0xffffffffu, e) & mine;
  bool store = e >= 0;
  if (__any_sync(0xffffffffu, store && (same & (same - 1)))) {
    float all = 0.f;
#pragma unroll
    for (int k = 0; k < kTopK; ++k) {
      const float dk = __shfl_sync(0xffffffffu, d, (lane & 24) + k);
      if ((same >> ((lane & 24) + k)) & 1u) all += dk;
    }
    d = all;
    store = store && lane == __ffs(same) - 1;
  }
  __syncwarp();   // the zeroes come first
  if (store) grad_logits[t * kEG + e] = d;
}

}  // namespace
}  // namespace kf

using namespace kf;

extern "C" int kf_moe_route_backward(const float* routing_logits, const int32_t* topk_idx, const float* grad_weight,
                                     int32_t num_tokens, float routed_scaling_factor, float* grad_logits,
                                     void* stream) {
  if (!valid_tokens(num_tokens)) return KF_ERR_INVALID_ARGUMENT;
  if (num_tokens == 0) return KF_OK;
  if (!routing_logits || !topk_idx || !grad_weight || !grad_logits) return KF_ERR_INVALID_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(grad_logits) & 15u) return KF_ERR_INVALID_ARGUMENT;
  int sms = 0;
  const int rc = device_ready(&sms);
  if (rc != KF_OK) return rc;
  constexpr int tokens = kThreads / 32 * kTokens;
  route_backward_kernel<<<(num_tokens + tokens - 1) / tokens, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
      routing_logits, topk_idx, grad_weight, num_tokens, routed_scaling_factor, grad_logits);
  return cudaGetLastError() == cudaSuccess ? KF_OK : KF_ERR_CUDA;
}
