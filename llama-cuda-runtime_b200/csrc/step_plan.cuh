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

#include <cooperative_groups.h>

#include "common.cuh"

namespace lcrb {

constexpr int kPlanThreads = 1024;
constexpr int kPlanCtas = 8;  // one cluster

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
  int sequences;
  uint32_t page_size;
  unsigned page_mul, page_shift;  // position / page_size = umulhi(position, page_mul) >> page_shift (page_size > 1)
  int max_rows;
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
  const uint32_t all = static_cast<uint32_t>(r.cached) + static_cast<uint32_t>(r.rows), q = all / a.page_size;
  const uint32_t want = q + (all != q * a.page_size);
  r.fits = want <= static_cast<uint32_t>(a.max_pages);
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

// One cluster of eight CTAs. Every CTA scans all requests (a few loads and
// shuffles; cheaper than passing the prefixes on), then they share the pages
// and the rows; cluster barriers stand between pushing pages, handing them out
// and reading the tables back, so held and free_count may be updated in place.
// A step of a few rows is bound by latency -- launch, the lengths' load, two
// block barriers, a cluster barrier, the table's load -- and a large one by the
// rows' stores, four rows a thread. 64 requests with up to five rows each: 5.6
// us; 512 requests, 64 of them with chunks of up to 2048 rows: 15.3 us (one CTA
// that did it all: 16.5 and 171 us, both timed with the call).
__global__ void __cluster_dims__(kPlanCtas, 1, 1) __launch_bounds__(kPlanThreads) step_plan_kernel(const StepPlanArgs a) {
  extern __shared__ int32_t plan_smem[];
  int32_t* row_end = plan_smem;            // inclusive prefixes per request
  int32_t* need_end = row_end + a.sequences;
  int32_t* back_end = need_end + a.sequences;
  int32_t* base = back_end + a.sequences;  // pages held before this step's; ~pages: the request does not fit its table
  int32_t* cached = base + a.sequences;
  __shared__ int part[3][kPlanThreads / 32];
  __shared__ int used_s;
  const auto cluster = cooperative_groups::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int me = static_cast<int>(cluster.block_rank()) * kPlanThreads + tid;
  constexpr int kAll = kPlanCtas * kPlanThreads;
  const int B = a.sequences;
  const int free0 = min(max(0, *a.free_count), a.pool_pages);

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
    base[b] = r.fits ? r.held : ~r.held;
    cached[b] = r.cached;
  }
  auto scan = [&](int& x, int& y, int& z) {  // inclusive, over a warp
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, x, off), v = __shfl_up_sync(0xffffffffu, y, off),
                t = __shfl_up_sync(0xffffffffu, z, off);
      if (lane >= off) {
        x = plan_add_rows(x, u, a.max_rows);
        y += v;
        z += t;
      }
    }
  };
  int irows = rows, ineed = need, iback = back;
  scan(irows, ineed, iback);
  if (lane == 31) {
    part[0][warp] = irows;
    part[1][warp] = ineed;
    part[2][warp] = iback;
  }
  if (tid == 0) used_s = 0;
  __syncthreads();
  // The warps' totals, scanned by every warp; then this thread's exclusive
  // prefixes.
  int wrows = part[0][lane], wneed = part[1][lane], wback = part[2][lane];
  scan(wrows, wneed, wback);
  const int total_back = __shfl_sync(0xffffffffu, wback, 31);
  int prow = __shfl_sync(0xffffffffu, wrows, max(0, warp - 1)), pneed = __shfl_sync(0xffffffffu, wneed, max(0, warp - 1)),
      pback = __shfl_sync(0xffffffffu, wback, max(0, warp - 1));
  if (warp == 0) prow = pneed = pback = 0;
  {
    const int x = __shfl_up_sync(0xffffffffu, irows, 1), y = __shfl_up_sync(0xffffffffu, ineed, 1),
              z = __shfl_up_sync(0xffffffffu, iback, 1);
    if (lane > 0) {
      prow = plan_add_rows(prow, x, a.max_rows);
      pneed += y;
      pback += z;
    }
  }
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
  if (pushed > 0) {
    for (int k = me; k < pushed; k += kAll) {
      const int b = plan_owner(back_end, B, k);
      const int first = b > 0 ? back_end[b - 1] : 0;
      a.free_pages[free0 + k] = a.tables[static_cast<size_t>(b) * a.max_pages + (k - first)];
    }
    cluster.sync();
  }
  // Pages handed out, from the top.
  for (int k = me; k < used; k += kAll) {
    const int b = plan_owner(need_end, B, k);
    const int first = b > 0 ? need_end[b - 1] : 0;
    a.tables[static_cast<size_t>(b) * a.max_pages + base[b] + (k - first)] = __ldcg(a.free_pages + height - 1 - k);
  }
  cluster.sync();
  auto granted = [&](int b) {
    return base[b] >= 0 && (need_end[b] <= height || need_end[b] == (b > 0 ? need_end[b - 1] : 0));
  };
  // Per request, by one CTA (held may be held_out, free_count free_count_out:
  // every thread of the cluster has read them).
  if (cluster.block_rank() == 0) {
    for (int b = b0; b < b1; ++b) {
      const bool got = granted(b);
      a.row_starts[b] = b > 0 ? row_end[b - 1] : 0;
      a.held_out[b] = base[b] < 0 ? ~base[b] : base[b] + (got ? need_end[b] - (b > 0 ? need_end[b - 1] : 0) : 0);
      a.kv_lengths[b] = got ? cached[b] + max(0, a.new_tokens[b]) : 0;
    }
    if (tid == 0) {
      a.row_starts[B] = row_end[B - 1];
      *a.free_count_out = height - used;
    }
  }
  // Four neighbouring rows a thread: one search, and 16-byte stores.
  const int total = row_end[B - 1];
  const bool wide = ((reinterpret_cast<uintptr_t>(a.positions) | reinterpret_cast<uintptr_t>(a.slots) |
                      reinterpret_cast<uintptr_t>(a.row_sequence)) & 15u) == 0;
  for (int r0 = 4 * me; r0 < total; r0 += 4 * kAll) {
    int b = plan_owner(row_end, B, r0);
    int begin = b > 0 ? row_end[b - 1] : 0, end = row_end[b];
    int c = cached[b];
    bool got = granted(b);
    int pos[4], slot[4], seq[4], at[4];  // at: the page's place in the tables, -1: none
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = r0 + e;
      at[e] = -1;
      if (r < total) {
        if (r >= end) {
          do {
            begin = end;
            end = row_end[++b];
          } while (r >= end);
          c = cached[b];
          got = granted(b);
        }
        pos[e] = c + (r - begin);
        seq[e] = b;
        const int q = a.page_size == 1 ? pos[e] : static_cast<int>(__umulhi(pos[e], a.page_mul) >> a.page_shift);
        slot[e] = pos[e] - q * a.page_size;
        if (got) at[e] = b * a.max_pages + q;
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (at[e] >= 0) at[e] = __ldcg(a.tables + at[e]);  // four loads at once
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) slot[e] = at[e] >= 0 && at[e] < a.pool_pages ? at[e] * static_cast<int>(a.page_size) + slot[e] : -1;
    if (wide && r0 + 4 <= total) {
      *reinterpret_cast<int4*>(a.positions + r0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
      *reinterpret_cast<int4*>(a.slots + r0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
      *reinterpret_cast<int4*>(a.row_sequence + r0) = make_int4(seq[0], seq[1], seq[2], seq[3]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (r0 + e < total) {
          a.positions[r0 + e] = pos[e];
          a.slots[r0 + e] = slot[e];
          a.row_sequence[r0 + e] = seq[e];
        }
      }
    }
  }
  // The rows left over, for steps of a fixed number of rows: nobody's.
  for (int r = total + me; r < a.max_rows; r += kAll) {
    a.positions[r] = 0;
    a.slots[r] = -1;
    a.row_sequence[r] = -1;
  }
}

}  // namespace lcrb
