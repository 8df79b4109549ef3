// Verification of drafted tokens (lcr_verify_drafts) in whole numbers:
// probabilities in units of 2^-38 and uniforms in units of 2^-24, so sums are
// exact in 64 bits and no result depends on the order in which they are
// formed. Draft j (of k) is kept while U_j Q_j(d_j) < P_j(d_j) 2^24; the next
// token is the lowest x with R(0) + .. + R(x) > floor(U sum(R) / 2^24), R =
// max(P_j - Q_j, 0) at the first refusal j and P_k after k kept drafts.
// Only the row that is drawn from (and its Q row) is read whole.
#pragma once

#include <cooperative_groups.h>

#include "common.cuh"

namespace lcrb {

struct VerifyArgs {
  int32_t* tokens;
  int32_t* accepted;
  const float* target;
  long long target_stride;
  const int32_t* target_starts;
  const int32_t* drafts;
  const int32_t* counts;
  const float* draft_probs;  // [sequences][max_drafts][vocab], or null: certain drafts
  const float* uniforms;
  int sequences, max_drafts, vocab;
};

constexpr int kVerifyThreads = 512;
constexpr int kVerifyCtas = 8;       // a cluster for each request
constexpr int kVerifyChunks = 1024;  // of a CTA's slice, at most
constexpr int kVerifyElsewhere = -2; // verify_write: another CTA writes the drawn token
constexpr long long kVerifyOne = 1ll << 38;

// p in units of 2^-38. The scaling by a power of two is exact, so this is one
// rounding (to nearest even), the same wherever it is done.
__device__ __forceinline__ long long verify_fixed(float p) {
  return __float2ll_rn(fminf(fmaxf(p, 0.f), 1.f) * 274877906944.0f);  // fmaxf drops a NaN
}

__device__ __forceinline__ unsigned long long verify_uniform(float u) {
  return static_cast<unsigned long long>(fminf(fmaxf(u, 0.f) * 16777216.0f, 16777215.0f));
}

// floor(U T / 2^24) for any 64-bit T.
__device__ __forceinline__ unsigned long long verify_target(unsigned long long u, unsigned long long t) {
  return (__umul64hi(u, t) << 40) | ((u * t) >> 24);
}

struct VerifyRow {
  const float* p;
  const float* q;  // null: no Q
  int drafted;     // the refused draft where Q is certain, else -1
};

// R of id i from its P and Q.
__device__ __forceinline__ long long verify_residual(const VerifyRow& r, int i, float p, float q) {
  long long v = verify_fixed(p);
  if (r.q != nullptr) v -= verify_fixed(q);
  if (i == r.drafted) v -= kVerifyOne;
  return v > 0 ? v : 0;
}

// P and Q of ids i .. i + 3, zeros from `end` on.
__device__ __forceinline__ void verify_load(const VerifyRow& r, bool vec, int i, int end, float (&p)[4], float (&q)[4]) {
  if (vec && i + 4 <= end) {
    const float4 x = *reinterpret_cast<const float4*>(r.p + i);
    const float4 y = r.q != nullptr ? *reinterpret_cast<const float4*>(r.q + i) : make_float4(0.f, 0.f, 0.f, 0.f);
    p[0] = x.x; p[1] = x.y; p[2] = x.z; p[3] = x.w;
    q[0] = y.x; q[1] = y.y; q[2] = y.z; q[3] = y.w;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      p[e] = i + e < end ? r.p[i + e] : 0.f;
      q[e] = i + e < end && r.q != nullptr ? r.q[i + e] : 0.f;
    }
  }
}

// Inclusive prefix sum over a warp.
__device__ __forceinline__ long long verify_scan(long long v, int lane) {
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v += x;
  }
  return v;
}

// Where the drafts of request b end: the number kept, and the row drawn from.
// Every thread of the CTA calls it; `kept_s` is shared.
__device__ __forceinline__ int verify_kept(const VerifyArgs& a, int b, int first, int k, int* kept_s) {
  if (threadIdx.x == 0) *kept_s = k;
  __syncthreads();
  for (int j = threadIdx.x; j < k; j += blockDim.x) {
    const size_t row = static_cast<size_t>(b) * a.max_drafts + j;
    const int d = a.drafts[row];
    bool ok = false;
    if (d >= 0 && d < a.vocab) {
      const unsigned long long u = verify_uniform(a.uniforms[static_cast<size_t>(b) * (a.max_drafts + 1) + j]);
      const long long p = verify_fixed(a.target[(first + j) * a.target_stride + d]);
      const long long q = a.draft_probs != nullptr ? verify_fixed(a.draft_probs[row * a.vocab + d]) : kVerifyOne;
      ok = u * static_cast<unsigned long long>(q) < static_cast<unsigned long long>(p) << 24;
    }
    if (!ok) atomicMin(kept_s, j);
  }
  __syncthreads();
  return *kept_s;
}

__device__ __forceinline__ void verify_write(const VerifyArgs& a, int b, int kept, int token) {
  int32_t* out = a.tokens + static_cast<size_t>(b) * (a.max_drafts + 1);
  for (int j = threadIdx.x; j <= a.max_drafts; j += blockDim.x) {
    if (j != kept) out[j] = j < kept ? a.drafts[static_cast<size_t>(b) * a.max_drafts + j] : -1;
    else if (token != kVerifyElsewhere) out[j] = token;
  }
  if (threadIdx.x == 0) a.accepted[b] = max(0, kept);
}

// Where the drawn token is in the row, by chunks of the vocabulary in order:
// one cluster of eight CTAs takes a request, each CTA a contiguous slice in up
// to kVerifyChunks chunks, a warp a chunk at a time, so that the row (two rows
// after a refusal) is read once. The CTAs exchange their slices' sums through
// distributed shared memory; the one whose slice holds the target finds the
// chunk and reads only that again. HBM bound for many requests; for one, a
// chain of latencies (the draft, its two probabilities, the row, the exchange).
__global__ void __cluster_dims__(kVerifyCtas, 1, 1) __launch_bounds__(kVerifyThreads) verify_drafts_kernel(const VerifyArgs a) {
  __shared__ int kept_s;
  __shared__ long long sums[kVerifyChunks];
  __shared__ long long slice_s[2][kVerifyCtas];  // by pass
  __shared__ long long part[kVerifyThreads / 32];
  const auto cluster = cooperative_groups::this_cluster();
  cluster.barrier_arrive();  // this CTA runs: the others may write to its shared memory
  const int rank = static_cast<int>(cluster.block_rank());
  const int b = blockIdx.x / kVerifyCtas, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r0 = a.target_starts[b], r1 = a.target_starts[b + 1];
  if (r1 <= r0) {  // the same for the whole cluster
    if (rank == 0) verify_write(a, b, -1, -1);
    cluster.barrier_wait();
    return;
  }
  const int k = max(0, min(min(a.counts[b], a.max_drafts), r1 - r0 - 1));
  const int first = r1 - 1 - k;
  const int kept = verify_kept(a, b, first, k, &kept_s);
  VerifyRow row;
  row.p = a.target + (first + kept) * a.target_stride;
  row.q = nullptr;
  row.drafted = -1;
  if (kept < k) {
    const size_t at = static_cast<size_t>(b) * a.max_drafts + kept;
    if (a.draft_probs != nullptr) row.q = a.draft_probs + at * a.vocab;
    else row.drafted = a.drafts[at];
  }
  const unsigned long long u = verify_uniform(a.uniforms[static_cast<size_t>(b) * (a.max_drafts + 1) + a.max_drafts]);
  const int slice = (a.vocab + kVerifyCtas * 128 - 1) / (kVerifyCtas * 128) * 128;
  const int i0 = min(a.vocab, rank * slice), i1 = min(a.vocab, i0 + slice);
  // Chunks of a multiple of 128 ids: lane l has ids 4 l .. 4 l + 3 of each 128.
  const int chunk = (slice + kVerifyChunks * 128 - 1) / (kVerifyChunks * 128) * 128;
  const int chunks = (i1 - i0 + chunk - 1) / chunk;
  int token = -1;
  cluster.barrier_wait();
  for (int pass = 0; pass < 2; ++pass) {  // the second from P alone, where R is 0 everywhere
    const bool vec = ((reinterpret_cast<uintptr_t>(row.p) | reinterpret_cast<uintptr_t>(row.q)) & 15u) == 0;
    long long mine = 0;
    constexpr int WARPS = kVerifyThreads / 32;
    for (int c0 = warp; c0 < chunks; c0 += 4 * WARPS) {  // four chunks at a time, for their loads' sake
      long long v[4] = {0, 0, 0, 0};
      for (int o = 4 * lane; o < chunk; o += 128) {
        float p[4][4], q[4][4];
#pragma unroll
        for (int s = 0; s < 4; ++s) verify_load(row, vec, i0 + (c0 + s * WARPS) * chunk + o, i1, p[s], q[s]);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[s] += verify_residual(row, i0 + (c0 + s * WARPS) * chunk + o + e, p[s][e], q[s][e]);
        }
      }
#pragma unroll
      for (int s = 0; s < 4; ++s) {
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) v[s] += __shfl_xor_sync(0xffffffffu, v[s], off);
        if (c0 + s * WARPS < chunks) {
          if (lane == 0) sums[c0 + s * WARPS] = v[s];
          mine += v[s];
        }
      }
    }
    if (lane == 0) part[warp] = mine;
    __syncthreads();
    if (tid < kVerifyCtas) {
      long long all = 0;
      for (int w = 0; w < WARPS; ++w) all += part[w];
      cluster.map_shared_rank(slice_s[pass], tid)[rank] = all;
    }
    cluster.sync();
    long long before = 0, total = 0;
    for (int c = 0; c < kVerifyCtas; ++c) {
      if (c < rank) before += slice_s[pass][c];
      total += slice_s[pass][c];
    }
    if (total > 0) {
      const long long t = static_cast<long long>(verify_target(u, static_cast<unsigned long long>(total)));
      if (warp == 0 && before <= t && t < before + slice_s[pass][rank]) {
        // The chunk, 32 at a time; then the id in it, 128 at a time.
        int c = 0;
        for (;; c += 32) {
          const long long s = c + lane < chunks ? sums[c + lane] : 0;
          const long long incl = verify_scan(s, lane);
          const unsigned over = __ballot_sync(0xffffffffu, before + incl > t);
          if (over != 0u) {
            const int l = __ffs(over) - 1;
            before += __shfl_sync(0xffffffffu, incl - s, l);
            c += l;
            break;
          }
          before += __shfl_sync(0xffffffffu, incl, 31);
        }
        for (int i = i0 + c * chunk;; i += 128) {
          float p[4], q[4];
          long long s[4];
          verify_load(row, vec, i + 4 * lane, i1, p, q);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[e] = verify_residual(row, i + 4 * lane + e, p[e], q[e]);
          const long long sum = (s[0] + s[1]) + (s[2] + s[3]);
          const long long incl = verify_scan(sum, lane);
          const unsigned over = __ballot_sync(0xffffffffu, before + incl > t);
          if (over != 0u) {
            const int l = __ffs(over) - 1;
            if (lane == l) {
              before += incl - sum;
#pragma unroll
              for (int e = 3; e >= 0; --e) {  // the lowest id whose running sum passes t
                long long run = before;
                for (int d = 0; d <= e; ++d) run += s[d];
                if (run > t) token = i + 4 * lane + e;
              }
              a.tokens[static_cast<size_t>(b) * (a.max_drafts + 1) + kept] = token;
            }
            break;
          }
          before += __shfl_sync(0xffffffffu, incl, 31);
        }
      }
      if (rank == 0) verify_write(a, b, kept, kVerifyElsewhere);
      return;
    }
    row.q = nullptr;
    row.drafted = -1;
  }
  if (rank == 0) verify_write(a, b, kept, -1);
}

}  // namespace lcrb
