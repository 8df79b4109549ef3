// Rows of logits to rows of probabilities (lcr_token_probs): with t the row's
// temperature, p = exp((x - max) / t) / sum, or one at the largest logit
// (lowest id on ties) for t <= 0.
//
// HBM bound (8 bytes an id). A cluster of CTAs takes a row, each a contiguous
// slice that its threads keep in registers, so a row is read once and written
// once: the weights are formed against the CTA's own maximum, the CTAs exchange
// (maximum, sum) through distributed shared memory, and one factor brings them
// to the row's.
#pragma once

#include <cooperative_groups.h>

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
  int slice;  // ids per CTA, a multiple of 4
};

constexpr int kProbsThreads = 512;
constexpr int kProbsKeep = 8;                                      // groups of 4 ids a thread keeps
constexpr int kProbsSlice = kProbsThreads * kProbsKeep * 4;        // ids a CTA can keep
constexpr int kProbsMaxCtas = 8;

__device__ __forceinline__ float probs_temperature(const TokenProbsArgs& a, int r) {
  if (a.temperature == nullptr) return 1.0f;
  return a.temperature[a.row_sequence != nullptr ? a.row_sequence[r] : r];
}

// The order of (logit, lowest id first) as an integer.
__device__ __forceinline__ unsigned long long probs_key(float x, int i) {
  const uint32_t b = __float_as_uint(x), k = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return (static_cast<unsigned long long>(k) << 32) | (0xffffffffu - static_cast<uint32_t>(i));
}

// Grid: a cluster for each row. VEC: rows are 16-byte aligned.
// A slice beyond kProbsSlice ids (vocabularies beyond 8 x 16384) is gone over
// again in memory.
template <bool VEC>
__global__ void __launch_bounds__(kProbsThreads, 2) token_probs_kernel(const TokenProbsArgs a) {
  const auto cluster = cooperative_groups::this_cluster();
  const int ctas = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  __shared__ float red[2][kProbsThreads / 32];
  __shared__ float2 ms[kProbsMaxCtas];
  __shared__ unsigned long long best_s[kProbsMaxCtas], best_w[kProbsThreads / 32];
  cluster.barrier_arrive();  // this CTA runs: the others may write to its shared memory
  const int r = blockIdx.x / ctas, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float* x = a.logits + r * a.logits_stride;
  float* p = a.probs + r * a.probs_stride;
  const int i0 = rank * a.slice, i1 = min(a.vocab, i0 + a.slice);
  const float t = probs_temperature(a, r);
  auto load = [&](int i, float (&v)[4]) {
    if (VEC && i + 4 <= i1) {
      const float4 q = *reinterpret_cast<const float4*>(x + i);
      v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = i + e < i1 ? x[i + e] : -INFINITY;
    }
  };
  auto store = [&](int i, const float (&v)[4]) {
    if (VEC && i + 4 <= i1) {
      *reinterpret_cast<float4*>(p + i) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (i + e < i1) p[i + e] = v[e];
      }
    }
  };
  constexpr int STEP = kProbsThreads * 4;
  const int more = i0 + kProbsKeep * STEP + 4 * tid;  // this thread's ids past those it keeps

  if (!(t > 0.f)) {
    unsigned long long best = 0ull;
    for (int i = i0 + 4 * tid; i < i1; i += STEP) {
      float v[4];
      load(i, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (v[e] > -INFINITY) best = max(best, probs_key(v[e], i + e));
      }
    }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, off));
    if (lane == 0) best_w[warp] = best;
    __syncthreads();
    cluster.barrier_wait();
    if (tid < ctas) {
      for (int q = 0; q < kProbsThreads / 32; ++q) best = max(best, best_w[q]);
      cluster.map_shared_rank(best_s, tid)[rank] = best;
    }
    cluster.sync();
    best = 0ull;
    for (int q = 0; q < ctas; ++q) best = max(best, best_s[q]);
    const int at = best == 0ull ? -1 : static_cast<int>(0xffffffffu - static_cast<uint32_t>(best));
    for (int i = i0 + 4 * tid; i < i1; i += STEP) {
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = i + e == at ? 1.0f : 0.0f;
      store(i, v);
    }
    return;
  }

  float v[kProbsKeep][4];
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < kProbsKeep; ++k) load(i0 + k * STEP + 4 * tid, v[k]);
#pragma unroll
  for (int k = 0; k < kProbsKeep; ++k) m = fmaxf(m, fmaxf(fmaxf(v[k][0], v[k][1]), fmaxf(v[k][2], v[k][3])));
  for (int i = more; i < i1; i += STEP) {
    float q[4];
    load(i, q);
    m = fmaxf(m, fmaxf(fmaxf(q[0], q[1]), fmaxf(q[2], q[3])));
  }
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  if (lane == 0) red[0][warp] = m;
  __syncthreads();
  m = red[0][lane % (kProbsThreads / 32)];
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  const float k2 = kLog2e / t;
  const float base = m == -INFINITY ? 0.f : m;  // a slice of nothing but -inf weighs nothing
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < kProbsKeep; ++k) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[k][e] = exp2f((v[k][e] - base) * k2);
    sum += (v[k][0] + v[k][1]) + (v[k][2] + v[k][3]);
  }
  for (int i = more; i < i1; i += STEP) {
    float q[4];
    load(i, q);
#pragma unroll
    for (int e = 0; e < 4; ++e) sum += exp2f((q[e] - base) * k2);
  }
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  if (lane == 0) red[1][warp] = sum;
  __syncthreads();
  cluster.barrier_wait();
  if (tid < ctas) {
    sum = 0.f;
    for (int q = 0; q < kProbsThreads / 32; ++q) sum += red[1][q];
    cluster.map_shared_rank(ms, tid)[rank] = make_float2(m, sum);
  }
  cluster.sync();
  float top = -INFINITY, all = 0.f;
  for (int q = 0; q < ctas; ++q) top = fmaxf(top, ms[q].x);
  for (int q = 0; q < ctas; ++q) all += ms[q].x == -INFINITY ? 0.f : ms[q].y * exp2f((ms[q].x - top) * k2);
  const float f = m == -INFINITY ? 0.f : exp2f((m - top) * k2) / all;
#pragma unroll
  for (int k = 0; k < kProbsKeep; ++k) {
    const int i = i0 + k * STEP + 4 * tid;
    if (i < i1) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[k][e] *= f;
      store(i, v[k]);
    }
  }
  for (int i = more; i < i1; i += STEP) {
    float q[4];
    load(i, q);
#pragma unroll
    for (int e = 0; e < 4; ++e) q[e] = exp2f((q[e] - base) * k2) * f;
    store(i, q);
  }
}

}  // namespace lcrb
