// Verification of drafted tokens (lcr_verify_drafts) in whole numbers:
// probabilities in units of 2^-38 and uniforms in units of 2^-24, so sums are
// exact in 64 bits and no result depends on the order in which they are
// formed. Draft j (of k) is kept while U_j Q_j(d_j) < P_j(d_j) 2^24; the next
// token is the lowest x with R(0) + .. + R(x) > floor(U sum(R) / 2^24), R =
// max(P_j - Q_j, 0) at the first refusal j and P_k after k kept drafts.
// Only the row that is drawn from (and its Q row) is read whole.
#pragma once

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

constexpr int kVerifyThreads = 1024;
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

__device__ __forceinline__ long long verify_residual(const VerifyRow& r, int i) {
  long long v = verify_fixed(r.p[i]);
  if (r.q != nullptr) v -= verify_fixed(r.q[i]);
  if (i == r.drafted) v -= kVerifyOne;
  return v > 0 ? v : 0;
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
    out[j] = j < kept ? a.drafts[static_cast<size_t>(b) * a.max_drafts + j] : j == kept ? token : -1;
  }
  if (threadIdx.x == 0) a.accepted[b] = max(0, kept);
}

// One CTA per request; thread t owns a contiguous range of the vocabulary.
__global__ void __launch_bounds__(kVerifyThreads) verify_drafts_kernel(const VerifyArgs a) {
  __shared__ int kept_s, token_s;
  __shared__ long long part[kVerifyThreads / 32];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r0 = a.target_starts[b], r1 = a.target_starts[b + 1];
  if (r1 <= r0) {
    verify_write(a, b, -1, -1);
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
  const int per = (a.vocab + kVerifyThreads - 1) / kVerifyThreads;
  const int i0 = min(a.vocab, tid * per), i1 = min(a.vocab, i0 + per);
  if (tid == 0) token_s = -1;
  for (int pass = 0; pass < 2; ++pass) {  // the second from P alone, where R is 0 everywhere
    long long mine = 0;
    for (int i = i0; i < i1; ++i) mine += verify_residual(row, i);
    long long incl = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += x;
    }
    if (lane == 31) part[warp] = incl;
    __syncthreads();
    long long before = incl - mine, total = 0;
    for (int w = 0; w < kVerifyThreads / 32; ++w) {
      if (w < warp) before += part[w];
      total += part[w];
    }
    if (total > 0) {
      const long long t = static_cast<long long>(verify_target(u, static_cast<unsigned long long>(total)));
      if (before <= t && t < before + mine) {
        for (int i = i0; i < i1; ++i) {
          before += verify_residual(row, i);
          if (before > t) {
            token_s = i;
            break;
          }
        }
      }
      break;
    }
    row.q = nullptr;
    row.drafted = -1;
    __syncthreads();
  }
  __syncthreads();
  verify_write(a, b, kept, token_s);
}

}  // namespace lcrb
