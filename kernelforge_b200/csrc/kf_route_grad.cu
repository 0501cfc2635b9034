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
// One warp per token.  Lanes 0..7 hold the chosen experts; the row of 256
// gradients is written in full, lane l columns 4 l .. and 128 + 4 l .. .
#include "kf_internal.cuh"

namespace kf {
namespace {

constexpr int kThreads = 256;

__global__ void __launch_bounds__(kThreads) route_backward_kernel(const float* __restrict__ logits,
                                                                  const int32_t* __restrict__ topk_idx,
                                                                  const float* __restrict__ grad_w, int T, float rsf,
                                                                  float* __restrict__ grad_logits) {
  const int lane = threadIdx.x & 31;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  if (t >= T) return;
  int e = -1;
  float s = 0.f, c = 0.f, g = 0.f;
  if (lane < kTopK) {
    e = topk_idx[t * kTopK + lane];
    if (e >= 0 && e < kEG) {
      g = grad_w[t * kTopK + lane];
      const float x = logits[t * kEG + e];
      s = 1.0f / (1.0f + expf(-x));
      c = 1.0f / (1.0f + expf(x));   // 1 - s without the cancellation
    } else {
      e = -1;
    }
  }
  float sum = s;
#pragma unroll
  for (int off = 4; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  const float p = s / (sum + 1e-20f);
  float mean = g * p;
#pragma unroll
  for (int off = 4; off >= 1; off >>= 1) mean += __shfl_xor_sync(0xffffffffu, mean, off);
  const float d = rsf * p * c * (g - mean);
  float v[8] = {};
#pragma unroll
  for (int k = 0; k < kTopK; ++k) {
    const int ek = __shfl_sync(0xffffffffu, e, k);
    const float dk = __shfl_sync(0xffffffffu, d, k);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (ek == (j >> 2) * 128 + lane * 4 + (j & 3)) v[j] += dk;
  }
  float4* dst = reinterpret_cast<float4*>(grad_logits + t * kEG);
  dst[lane] = make_float4(v[0], v[1], v[2], v[3]);
  dst[32 + lane] = make_float4(v[4], v[5], v[6], v[7]);
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
  constexpr int warps = kThreads / 32;
  route_backward_kernel<<<(num_tokens + warps - 1) / warps, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
      routing_logits, topk_idx, grad_weight, num_tokens, routed_scaling_factor, grad_logits);
  return cudaGetLastError() == cudaSuccess ? KF_OK : KF_ERR_CUDA;
}
