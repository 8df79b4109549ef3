// Block tables, slot map and row map of a ragged step (lcr_plan_step).
//
// With h_b pages held (0 after a turn-over, which pushes them on the free
// stack), c_b cached and n_b new positions, request b wants
// ceil((c_b + n_b) / page_size) pages and needs the difference. Three prefix
// sums over the requests (rows, pages needed, pages given back) place
// everything: the k-th page handed out is the stack's entry F - 1 - k, F the
// stack's height after the push, and request b is granted its pages iff its
// inclusive prefix of needs is at most F.
#pragma once

#include "common.cuh"

namespace lcrb {

constexpr int kPlanThreads = 1024;

struct StepPlanArgs {
  int32_t* tables;
  int max_pages;
  const int32_t* held;
  int32_t* held_out;
  int32_t* free_pages;
  const int32_t* free_count;
  int32_t* free_count_out;
  int pool_pages;
  const int32_t* cached;
  const int32_t* new_tokens;
  const int32_t* finished;
  int sequences, page_size, max_rows;
  int32_t* row_starts;
  int32_t* kv_lengths;
  int32_t* positions;
  int32_t* slots;
  int32_t* row_sequence;
};

// One request's part of the plan, from its inputs.
struct PlanNeed {
  int cached, rows, held, back, need;
  bool fits;
};

__device__ __forceinline__ PlanNeed plan_need(const StepPlanArgs& a, int b) {
  PlanNeed r;
  r.cached = max(0, a.cached[b]);
  r.rows = max(0, a.new_tokens[b]);
  const int held = min(max(0, a.held[b]), a.max_pages);
  const bool done = a.finished != nullptr && a.finished[b] != 0;
  r.back = done ? held : 0;
  r.held = done ? 0 : held;
  const long long want = (static_cast<long long>(r.cached) + r.rows + a.page_size - 1) / a.page_size;
  r.fits = want <= a.max_pages;
  r.need = r.fits ? max(0, static_cast<int>(want) - r.held) : 0;
  return r;
}

// First index b in [0, n) with ends[b] > k (ends non-decreasing, k < ends[n - 1]).
__device__ __forceinline__ int plan_owner(const int32_t* ends, int n, int k) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (ends[mid] > k) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// Sums of row counts saturate at max_rows (rows past it are cut off).
__device__ __forceinline__ int plan_add_rows(int x, int y, int most) {
  const uint32_t s = static_cast<uint32_t>(x) + static_cast<uint32_t>(y);
  return s < static_cast<uint32_t>(most) ? static_cast<int>(s) : most;
}

// One CTA: scan, push, hand out, rows, with a block barrier between.
__global__ void __launch_bounds__(kPlanThreads) step_plan_kernel(const StepPlanArgs a) {
  extern __shared__ int32_t plan_smem[];
  int32_t* row_end = plan_smem;            // inclusive prefixes per request
  int32_t* need_end = row_end + a.sequences;
  int32_t* back_end = need_end + a.sequences;
  int32_t* base = back_end + a.sequences;  // pages held before this step's
  __shared__ int part[3][kPlanThreads / 32];
  __shared__ int used_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int B = a.sequences;

  // Thread t scans a contiguous share of the requests.
  const int per = (B + kPlanThreads - 1) / kPlanThreads;
  const int b0 = min(B, tid * per), b1 = min(B, b0 + per);
  int rows = 0, need = 0, back = 0;
  for (int b = b0; b < b1; ++b) {
    const PlanNeed r = plan_need(a, b);
    rows = plan_add_rows(rows, min(r.rows, a.max_rows), a.max_rows);
    need += r.need;
    back += r.back;
    row_end[b] = rows;
    need_end[b] = need;
    back_end[b] = back;
    base[b] = r.held;
  }
  int irows = rows, ineed = need, iback = back;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, irows, off), y = __shfl_up_sync(0xffffffffu, ineed, off),
              z = __shfl_up_sync(0xffffffffu, iback, off);
    if (lane >= off) {
      irows = plan_add_rows(irows, x, a.max_rows);
      ineed += y;
      iback += z;
    }
  }
  if (lane == 31) {
    part[0][warp] = irows;
    part[1][warp] = ineed;
    part[2][warp] = iback;
  }
  if (tid == 0) used_s = 0;
  __syncthreads();
  int prow = 0, pneed = 0, pback = 0;  // exclusive prefixes of this thread
  for (int w = 0; w < warp; ++w) {
    prow = plan_add_rows(prow, part[0][w], a.max_rows);
    pneed += part[1][w];
    pback += part[2][w];
  }
  {
    const int x = __shfl_up_sync(0xffffffffu, irows, 1), y = __shfl_up_sync(0xffffffffu, ineed, 1),
              z = __shfl_up_sync(0xffffffffu, iback, 1);
    if (lane > 0) {
      prow = plan_add_rows(prow, x, a.max_rows);
      pneed += y;
      pback += z;
    }
  }
  int total_back = 0;
  for (int w = 0; w < kPlanThreads / 32; ++w) total_back += part[2][w];
  const int free0 = min(max(0, *a.free_count), a.pool_pages);
  const int height = min(free0 + total_back, a.pool_pages);
  int used = 0;
  for (int b = b0; b < b1; ++b) {
    row_end[b] = plan_add_rows(prow, row_end[b], a.max_rows);
    need_end[b] += pneed;
    back_end[b] += pback;
    if (need_end[b] <= height) used = max(used, need_end[b]);
  }
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) used = max(used, __shfl_xor_sync(0xffffffffu, used, off));
  if (lane == 0 && used > 0) atomicMax(&used_s, used);
  __syncthreads();
  used = used_s;
  const int pushed = height - free0;

  // Pages given back, on top of the free ones.
  for (int k = tid; k < pushed; k += kPlanThreads) {
    const int b = plan_owner(back_end, B, k);
    const int first = b > 0 ? back_end[b - 1] : 0;
    a.free_pages[free0 + k] = a.tables[static_cast<size_t>(b) * a.max_pages + (k - first)];
  }
  __syncthreads();
  // Pages handed out, from the top.
  for (int k = tid; k < used; k += kPlanThreads) {
    const int b = plan_owner(need_end, B, k);
    const int first = b > 0 ? need_end[b - 1] : 0;
    a.tables[static_cast<size_t>(b) * a.max_pages + base[b] + (k - first)] = a.free_pages[height - 1 - k];
  }
  __syncthreads();
  // Per request (held may be held_out, free_count free_count_out: every
  // thread has read them).
  for (int b = b0; b < b1; ++b) {
    const int c = max(0, a.cached[b]), n = max(0, a.new_tokens[b]);
    const long long want = (static_cast<long long>(c) + n + a.page_size - 1) / a.page_size;
    const int nb = need_end[b] - (b > 0 ? need_end[b - 1] : 0);
    const bool granted = want <= a.max_pages && (nb == 0 || need_end[b] <= height);
    a.row_starts[b] = b > 0 ? row_end[b - 1] : 0;
    a.held_out[b] = base[b] + (granted ? nb : 0);
    a.kv_lengths[b] = granted ? c + n : 0;
  }
  if (tid == 0) {
    a.row_starts[B] = row_end[B - 1];
    *a.free_count_out = height - used;
  }
  const int total = row_end[B - 1];
  for (int r = tid; r < total; r += kPlanThreads) {
    const int b = plan_owner(row_end, B, r);
    const int i = r - (b > 0 ? row_end[b - 1] : 0);
    const int c = max(0, a.cached[b]), n = max(0, a.new_tokens[b]);
    const long long want = (static_cast<long long>(c) + n + a.page_size - 1) / a.page_size;
    const int nb = need_end[b] - (b > 0 ? need_end[b - 1] : 0);
    const bool granted = want <= a.max_pages && (nb == 0 || need_end[b] <= height);
    const int pos = c + i;
    int slot = -1;
    if (granted) {
      const int page = a.tables[static_cast<size_t>(b) * a.max_pages + pos / a.page_size];
      if (page >= 0 && page < a.pool_pages) slot = page * a.page_size + pos % a.page_size;
    }
    a.positions[r] = pos;
    a.slots[r] = slot;
    a.row_sequence[r] = b;
  }
}

}  // namespace lcrb
