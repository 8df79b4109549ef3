// Rows of logits to rows of probabilities (lcr_token_probs): with t the row's
// temperature, p = exp((x - max) / t) / sum, or one at the largest logit
// (lowest id on ties) for t <= 0.
#pragma once

#include "common.cuh"

namespace lcrb {

struct TokenProbsArgs {
  float* probs;
  long long probs_stride;
  const float* logits;
  long long logits_stride;
  int rows, vocab;
  const float* temperature;
  const int32_t* row_sequence;
};

constexpr int kProbsThreads = 1024;

__device__ __forceinline__ float probs_temperature(const TokenProbsArgs& a, int r) {
  if (a.temperature == nullptr) return 1.0f;
  return a.temperature[a.row_sequence != nullptr ? a.row_sequence[r] : r];
}

// One CTA per row, three passes (maximum, sum, write).
__global__ void __launch_bounds__(kProbsThreads) token_probs_kernel(const TokenProbsArgs a) {
  __shared__ float red[32];
  __shared__ int first;
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float* x = a.logits + r * a.logits_stride;
  float* p = a.probs + r * a.probs_stride;
  const float t = probs_temperature(a, r);
  float m = -INFINITY;
  for (int i = tid; i < a.vocab; i += kProbsThreads) m = fmaxf(m, x[i]);
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  if (lane == 0) red[warp] = m;
  if (tid == 0) first = a.vocab;
  __syncthreads();
  m = red[lane];
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  __syncthreads();
  if (!(t > 0.f)) {
    for (int i = tid; i < a.vocab; i += kProbsThreads) {
      if (x[i] == m) {
        atomicMin(&first, i);
        break;
      }
    }
    __syncthreads();
    const int best = m == -INFINITY ? -1 : first;
    for (int i = tid; i < a.vocab; i += kProbsThreads) p[i] = i == best ? 1.0f : 0.0f;
    return;
  }
  const float k = kLog2e / t;
  float sum = 0.f;
  for (int i = tid; i < a.vocab; i += kProbsThreads) sum += m == -INFINITY ? 0.f : exp2f((x[i] - m) * k);
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  if (lane == 0) red[warp] = sum;
  __syncthreads();
  sum = red[lane];
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  const float inv = m == -INFINITY ? 0.f : 1.0f / sum;
  for (int i = tid; i < a.vocab; i += kProbsThreads) p[i] = m == -INFINITY ? 0.f : exp2f((x[i] - m) * k) * inv;
}

}  // namespace lcrb
