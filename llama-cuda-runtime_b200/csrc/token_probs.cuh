// Rows of logits to rows of probabilities (lcr_token_probs): with t the row's
// temperature, p = exp((x - max) / t) / sum, or one at the largest logit
// (lowest id on ties) for t <= 0.
//
// HBM bound: 8 bytes an id. A cluster of CTAs takes a row, each a contiguous
// slice kept in shared memory, so that a row is read once and written once.
// Every thread works on the ids it brought itself: a warp forms its weights
// against its own maximum, the warps of the cluster exchange (maximum, sum)
// through distributed shared memory behind one cluster barrier, and one factor
// brings a warp's weights to the row's. Three CTAs of 64 KB on an SM keep
// loads, exponentials and stores of different rows going at a time.
//
// 320 rows of 128256 ids: 73 us, 4.5 TB/s, 0.69 of a copy's rate (what is
// lost goes to the barrier's wait and to the cluster's start). Measured beside
// it: the slice in registers, two CTAs on an SM, 89 us; clusters of 5, 6 and 7
// with larger slices 81, 77 and 76; 256 threads a CTA 82. Five rows: 5.9 us,
// latency.
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
  int temperatures;
  const int32_t* row_sequence;
  int slice;  // ids per CTA, a multiple of 4
};

constexpr int kProbsThreads = 512;
constexpr int kProbsWarps = kProbsThreads / 32;
constexpr int kProbsKeep = 8;                                // groups of 4 ids a thread keeps
constexpr int kProbsSlice = kProbsThreads * kProbsKeep * 4;  // ids a CTA can keep
constexpr int kProbsMaxCtas = 8;

// False: the row is nobody's.
__device__ __forceinline__ bool probs_temperature(const TokenProbsArgs& a, int r, float& t) {
  t = 1.0f;
  if (a.temperature == nullptr) return true;
  const int b = a.row_sequence != nullptr ? a.row_sequence[r] : r;
  t = 0.f;
  if (b < 0 || b >= a.temperatures) return false;
  t = a.temperature[b];
  return true;
}

// The order of (logit, lowest id first) as an integer. x + 0.0f: -0.0 equals 0.0.
__device__ __forceinline__ unsigned long long probs_key(float x, int i) {
  const uint32_t b = __float_as_uint(__fadd_rn(x, 0.0f)), k = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return (static_cast<unsigned long long>(k) << 32) | (0xffffffffu - static_cast<uint32_t>(i));
}

// Grid: a cluster for each row. VEC: rows are 16-byte aligned.
// A slice beyond kProbsSlice ids (vocabularies beyond 8 x 16384) is gone over
// again in memory.
template <bool VEC>
__global__ void __launch_bounds__(kProbsThreads, 3) token_probs_kernel(const TokenProbsArgs a) {
  const auto cluster = cooperative_groups::this_cluster();
  const int ctas = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  __shared__ float2 ms[kProbsMaxCtas * kProbsWarps];
  __shared__ unsigned long long best_s[kProbsMaxCtas], best_w[kProbsWarps];
  cluster.barrier_arrive();  // this CTA runs: the others may write to its shared memory
  const int r = blockIdx.x / ctas, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float* x = a.logits + r * a.logits_stride;
  float* p = a.probs + r * a.probs_stride;
  const int i0 = rank * a.slice, i1 = min(a.vocab, i0 + a.slice);
  float t;
  const bool owned = probs_temperature(a, r, t);
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
    for (int i = i0 + 4 * tid; i < (owned ? i1 : 0); i += STEP) {
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
      for (int q = 0; q < kProbsWarps; ++q) best = max(best, best_w[q]);
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

  // The slice's first kProbsSlice ids stay in shared memory.
  extern __shared__ float4 kept[];
  float4* mine = kept + tid;
#pragma unroll
  for (int k = 0; k < kProbsKeep; ++k) {
    const int i = i0 + k * STEP + 4 * tid;
    if (VEC && i + 4 <= i1) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(mine + k * kProbsThreads)), "l"(x + i) : "memory");
    } else if (i < i1) {
      float q[4];
      load(i, q);
      mine[k * kProbsThreads] = make_float4(q[0], q[1], q[2], q[3]);
    }
  }
  asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
  const int keep = min(i1 - i0, kProbsSlice) - 4 * tid, groups = keep > 0 ? (keep + STEP - 1) / STEP : 0;
  float m = -INFINITY;
#pragma unroll 2
  for (int k = 0; k < groups; ++k) {
    const float4 q = mine[k * kProbsThreads];
    m = fmaxf(m, fmaxf(fmaxf(q.x, q.y), fmaxf(q.z, q.w)));
  }
  for (int i = more; i < i1; i += STEP) {
    float q[4];
    load(i, q);
    m = fmaxf(m, fmaxf(fmaxf(q[0], q[1]), fmaxf(q[2], q[3])));
  }
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  const float k2 = fminf(fmaxf(kLog2e / t, 2e-38f), 1e30f);  // 0 * inf, at the ends of t's range, is no weight
  const float base = m == -INFINITY ? 0.f : m;  // a slice of nothing but -inf weighs nothing
  float sum = 0.f;
#pragma unroll 2
  for (int k = 0; k < groups; ++k) {
    float4 q = mine[k * kProbsThreads];
    q = make_float4(exp2f((q.x - base) * k2), exp2f((q.y - base) * k2), exp2f((q.z - base) * k2), exp2f((q.w - base) * k2));
    mine[k * kProbsThreads] = q;
    sum += (q.x + q.y) + (q.z + q.w);
  }
  for (int i = more; i < i1; i += STEP) {
    float q[4];
    load(i, q);
#pragma unroll
    for (int e = 0; e < 4; ++e) sum += exp2f((q[e] - base) * k2);
  }
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  cluster.barrier_wait();
  if (lane < ctas) cluster.map_shared_rank(ms, lane)[rank * kProbsWarps + warp] = make_float2(m, sum);
  cluster.sync();
  float top = -INFINITY, all = 0.f;
  for (int q = lane; q < ctas * kProbsWarps; q += 32) top = fmaxf(top, ms[q].x);
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
  for (int q = lane; q < ctas * kProbsWarps; q += 32) all += ms[q].y * (ms[q].x == -INFINITY ? 0.f : exp2f((ms[q].x - top) * k2));
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) all += __shfl_xor_sync(0xffffffffu, all, off);
  // (A NaN logit has made its warp's sum NaN, and with it the row.)
  const float f = m == -INFINITY ? 0.f * all : exp2f((m - top) * k2) / all;
#pragma unroll 2
  for (int k = 0; k < groups; ++k) {
    const float4 q = mine[k * kProbsThreads];
    const float w[4] = {q.x * f, q.y * f, q.z * f, q.w * f};
    store(i0 + k * STEP + 4 * tid, w);
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
