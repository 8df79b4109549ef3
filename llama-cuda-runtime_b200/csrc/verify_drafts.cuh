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
  int target_rows;
  const int32_t* target_starts;
  const int32_t* drafts;
  const int32_t* counts;
  const float* draft_probs;  // [sequences][max_drafts][vocab], or null: certain drafts
  const float* uniforms;
  int sequences, max_drafts, vocab;
};

constexpr int kVerifyThreads = 512;
constexpr int kVerifyMaxCtas = 8;    // of a request's cluster
constexpr int kVerifyChunks = 512;   // of a CTA's slice, at most
constexpr int kVerifyElsewhere = -2; // verify_write: another CTA writes the drawn token
constexpr long long kVerifyOne = 1ll << 38;

// p in units of 2^-38, as h 2^22 + l: h = p 2^16 and l = the exact rest, both
// rounded to whole numbers by adding 1.5 2^23, whose bits then carry them (less
// kVerifyBias). h 2^22 is even, so ties fall as in one rounding to nearest even.
// (A conversion to 64 bits has a fraction of the rate of these.)
constexpr int kVerifyBias = 0x4B400000;
struct VerifyFixed {
  int h, l;  // biased
};
__device__ __forceinline__ VerifyFixed verify_split(float p) {
  p = __saturatef(p);  // NaN becomes 0
  const float t = __fmaf_rn(p, 65536.0f, 12582912.0f), h = __fsub_rn(t, 12582912.0f);
  const float u = __fmaf_rn(__fmaf_rn(p, 65536.0f, -h), 4194304.0f, 12582912.0f);
  return {__float_as_int(t), __float_as_int(u)};
}
__device__ __forceinline__ long long verify_fixed(float p) {
  const VerifyFixed f = verify_split(p);
  return static_cast<long long>(f.h - kVerifyBias) * 4194304ll + (f.l - kVerifyBias);
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

// Adds R of id i to (h, l). |l| of a difference is at most 2^22, so its sign
// is h's, or l's where h is 0.
__device__ __forceinline__ void verify_add(const VerifyRow& r, int i, float p, float q, int& h, int& l) {
  const VerifyFixed x = verify_split(p);
  if (r.q == nullptr) {
    if (i == r.drafted) return;  // P - 1 is not above 0
    h += x.h - kVerifyBias;
    l += x.l - kVerifyBias;
  } else {
    const VerifyFixed y = verify_split(q);
    const int dh = x.h - y.h, dl = x.l - y.l;
    if (dh > 0 || (dh == 0 && dl > 0)) {
      h += dh;
      l += dl;
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
// one cluster of up to eight CTAs takes a request, each a contiguous slice in up
// to kVerifyChunks chunks, a warp a chunk at a time, so that the row (two rows
// after a refusal) is read once. The CTAs exchange their slices' sums through
// distributed shared memory; the one whose slice holds the target finds the
// chunk and reads only that again.
//
// A chain of latencies (the draft, its two probabilities, the row, the exchange,
// the chunk) around the row's reading: one request of four drafts over 128256
// ids 8.6 us; 64 of them, 49 MB, 19.8 us, 2.5 TB/s (with conversions to 64 bits
// in place of verify_split, 41; with each half chunk loaded ahead, 21). With
// certain drafts 7.4 and 15.3 us.
__global__ void __launch_bounds__(kVerifyThreads, 2) verify_drafts_kernel(const VerifyArgs a) {
  __shared__ int kept_s;
  __shared__ long long sums[kVerifyChunks];
  __shared__ long long slice_s[2][kVerifyMaxCtas];  // by pass
  __shared__ long long part[kVerifyThreads / 32];
  const auto cluster = cooperative_groups::this_cluster();
  cluster.barrier_arrive();  // this CTA runs: the others may write to its shared memory
  const int ctas = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int b = blockIdx.x / ctas, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r0 = a.target_starts[b], r1 = a.target_starts[b + 1];
  if (r1 <= r0 || r0 < 0 || r1 > a.target_rows) {  // the same for the whole cluster
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
  const int slice = (a.vocab + ctas * 128 - 1) / (ctas * 128) * 128;
  const int i0 = min(a.vocab, rank * slice), i1 = min(a.vocab, i0 + slice);
  // Chunks of 512 ids (a 64-bit sum over the lanes costs ten shuffles) or more:
  // lane l has ids 4 l .. 4 l + 3 of each 128.
  const int chunk = max(512, (slice + kVerifyChunks * 128 - 1) / (kVerifyChunks * 128) * 128);
  const int chunks = (i1 - i0 + chunk - 1) / chunk;
  int token = -1;
  cluster.barrier_wait();
  for (int pass = 0; pass < 2; ++pass) {  // the second from P alone, where R is 0 everywhere
    const bool vec = ((reinterpret_cast<uintptr_t>(row.p) | reinterpret_cast<uintptr_t>(row.q)) & 15u) == 0;
    long long mine = 0;
    constexpr int WARPS = kVerifyThreads / 32;
    for (int c = warp; c < chunks; c += WARPS) {
      long long v = 0;
      for (int o = 0; o < chunk; o += 512) {
        const int i = i0 + c * chunk + o + 4 * lane;
        float p[4][4], q[4][4];
#pragma unroll
        for (int s = 0; s < 4; ++s) verify_load(row, vec, i + 128 * s, o + 128 * s < chunk ? i1 : 0, p[s], q[s]);
        int h = 0, l = 0;  // of 16 ids: far from 2^31
#pragma unroll
        for (int s = 0; s < 4; ++s) {
#pragma unroll
          for (int e = 0; e < 4; ++e) verify_add(row, i + 128 * s + e, p[s][e], q[s][e], h, l);
        }
        v += static_cast<long long>(h) * 4194304ll + l;
      }
#pragma unroll
      for (int off = 16; off >= 1; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
      if (lane == 0) sums[c] = v;
      mine += v;
    }
    if (lane == 0) part[warp] = mine;
    __syncthreads();
    if (tid < ctas) {
      long long all = 0;
      for (int w = 0; w < WARPS; ++w) all += part[w];
      cluster.map_shared_rank(slice_s[pass], tid)[rank] = all;
    }
    cluster.sync();
    long long before = 0, total = 0;
    for (int c = 0; c < ctas; ++c) {
      if (c < rank) before += slice_s[pass][c];
      total += slice_s[pass][c];
    }
    if (total > 0) {
      const long long t = static_cast<long long>(verify_target(u, static_cast<unsigned long long>(total)));
      if (warp == 0 && before <= t && t < before + slice_s[pass][rank]) {
        // The chunk, 32 at a time; then the id in it, 128 at a time.
        int c = 0;
        for (; c < chunks; c += 32) {
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
        for (int i = i0 + c * chunk; i < i1; i += 128) {
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
