// Attention of every request's new rows over its paged cache
// (lcr_chunk_attention) on the 5th-generation tensor cores: row i of the n
// rows of request b is at position p = kv_length - n + i and sees keys 0 .. p.
//
// Tiles. A tile is one KV head of one request and up to 128 of its (row, query
// head) pairs: QB = 128 / G' rows (G' = the group rounded up to a power of
// two) by the G heads of the group, pair r = row * G + head, so that a few
// rows of a decoding request fill the lowest lanes. Keys come in blocks of 64:
//
//   S = Q K^T          m128 n64 k16, both from shared memory (K-major, 128-byte
//                      swizzle), into one of two TMEM buffers
//   softmax            one thread per pair (TMEM lane): maximum and sum in the
//                      log2 domain, held in fp32; P rounded to bf16 -- the
//                      tensor cores' operand; its share of the result's error
//                      is that of the output's own rounding -- and stored over
//                      S in TMEM
//   O += P V           m128 n64 k16, P from TMEM, V in place as an MN-major
//                      operand (its rows are keys), O in TMEM
//
// The running maximum moves only when a block's exceeds it by more than 8 (a
// factor of 256): P and the sum use the same stale maximum, so O / l is
// unchanged, and rescaling O (a round trip through registers) is rare.
//
// Work. Lengths are known only on the device, and tiles cost from one block to
// thousands, so the blocks of all tiles (in order of request, KV head, rows)
// are laid end to end and every CTA (two per SM) takes an equal contiguous
// range of them: each CTA sums the requests' block counts (a closed form) and
// finds its range without a second launch. A tile that spans several ranges
// leaves one partial (m, l, O) for each in the workspace; the CTA that stores
// its partial last (a counter per split tile) joins them in range order, so
// the result does not depend on which one that is.
//
// Loads. Pages may have any size and any strides, so K and V rows are fetched
// 16 bytes at a time (cp.async) by two warps, each lane holding the cache row
// of one key, into a ring of 64-key half-blocks in the swizzled layout; keys
// past the tile's last position are filled with zeros and their pages never
// looked up, so what lies there cannot reach the sums. The ring runs ahead
// across tiles.
//
// Warps: 0-3 softmax (warp w owns TMEM lanes 32 w .. + 31) and epilogue, 4
// TMEM allocation and MMA issue (one lane), 5-6 loads. Every wait is bounded.
#pragma once

#include "attn_prefill_tc.cuh"
#include "common.cuh"
#include "gemm_tc.cuh"

namespace lcrb {

constexpr int kCaThreads = 224;
constexpr int kCaBlock = 64;      // keys per block
constexpr int kCaRows = 128;      // (row, head) pairs per tile
constexpr int kCaMinRange = 4;    // blocks a CTA takes at least (where there are as many)
constexpr int kCaMinPart = 2;     // blocks a part of a split tile has at least
constexpr int kCaFmaGroups = 2;   // of 8 groups of exponentials, on the FMA pipe

struct ChunkAttnArgs {
  bf16* out;
  long long out_stride;
  const bf16* q;
  long long q_stride;
  const bf16* keys;
  const bf16* values;
  const int32_t* tables;  // [sequences][max_pages]
  int max_pages, pool_pages, page_size;
  long long page_stride, head_stride;
  const int32_t* row_starts;
  const int32_t* kv_lengths;
  int sequences, rows, kv_heads, group;
  int qb;               // rows per tile, a power of two
  float scale_log2;
  uint32_t* status;
  unsigned* counters;   // [grid], zero between calls
  float* partials;      // [2 * grid] parts of ca_part_floats(D)
};

constexpr size_t ca_part_floats(int d) { return static_cast<size_t>(kCaRows) * (d + 2); }

template <int D>
struct CaGeom {
  static constexpr int PANELS = D / 64;                 // 128-byte wide panels
  static constexpr int Q_BYTES = PANELS * kCaRows * 128;
  static constexpr int SLOT = PANELS * kCaBlock * 128;  // K or V of one block
  static constexpr int SLOTS = D == 64 ? 10 : 5;        // two CTAs share an SM's shared memory
  static constexpr int LAG = D == 64 ? 6 : 3;           // loads in flight before the oldest is waited for
  static constexpr int BARS = 2 * SLOTS + 10;
  static constexpr size_t SMEM = Q_BYTES + SLOTS * SLOT + BARS * 8 + 64;
  static constexpr uint32_t O_COL = 128;                // TMEM: S0 0-63, S1 64-127, O from 128
  static_assert(LAG < SLOTS, "a load is signalled before its slot's next use");
};

// Blocks of a request's tiles 0 .. t - 1 for one KV head (t < its tiles),
// each tile reaching to key s + (t + 1) * qb: the sum of ceil((s + i qb) / 64)
// for i = 1 .. t.
__device__ __forceinline__ long long ca_blocks_before(int s, int t, int qb) {
  const long long a = static_cast<long long>(s) + kCaBlock - 1;
  if (qb >= kCaBlock) {
    const long long r = qb / kCaBlock;
    return t * (a / kCaBlock) + r * t * (t + 1ll) / 2;
  }
  const long long r = kCaBlock / qb;
  auto below = [r](long long m) {  // sum of i / r for i < m
    const long long k = m / r;
    return r * k * (k - 1) / 2 + k * (m - r * k);
  };
  const long long a1 = a / qb;
  return below(a1 + t + 1) - below(a1 + 1);
}

// One request as the kernel sees it: malformed lengths are cut to what the
// arrays hold.
struct CaSeq {
  int row0, n;   // rows
  int kv;        // cached positions
  int s;         // max(0, kv - n): where the block count starts
  int tiles;
  long long blocks;  // of one KV head
};

__device__ __forceinline__ CaSeq ca_seq(const ChunkAttnArgs& a, int b) {
  CaSeq q;
  q.row0 = min(max(0, a.row_starts[b]), a.rows);
  q.n = min(max(0, a.row_starts[b + 1]), a.rows) - q.row0;
  if (q.n < 0) q.n = 0;
  const long long cap = static_cast<long long>(a.max_pages) * a.page_size;
  q.kv = static_cast<int>(min(static_cast<long long>(max(0, a.kv_lengths[b])), cap));
  q.s = max(0, q.kv - q.n);
  q.tiles = (q.n + a.qb - 1) / a.qb;
  q.blocks = q.tiles == 0 ? 0
                          : ca_blocks_before(q.s, q.tiles - 1, a.qb) +
                                (static_cast<long long>(q.s) + q.n + kCaBlock - 1) / kCaBlock;
  return q;
}

__device__ __forceinline__ int ca_tile_len(const CaSeq& q, int t, int qb) {
  const long long end = static_cast<long long>(q.s) + min(static_cast<long long>(q.n), (t + 1ll) * qb);
  return static_cast<int>((end + kCaBlock - 1) / kCaBlock);
}

// A CTA's walk over its range of blocks, segment by segment (a segment = its
// share of one tile). Every warp walks for itself.
struct CaWalk {
  int b, h, t;
  CaSeq q;
  int len;        // blocks of the tile
  int off;        // first block of this segment
  long long left; // blocks of the range from here on

  __device__ __forceinline__ void open(const ChunkAttnArgs& a, int b0, long long at, long long count) {
    b = b0;
    q = ca_seq(a, b);
    h = static_cast<int>(at / q.blocks);
    const long long rem = at - h * q.blocks;
    int lo = 0, hi = q.tiles - 1;  // the last tile that begins at or before rem
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (ca_blocks_before(q.s, mid, a.qb) <= rem) lo = mid;
      else hi = mid - 1;
    }
    t = lo;
    len = ca_tile_len(q, t, a.qb);
    off = static_cast<int>(rem - ca_blocks_before(q.s, t, a.qb));
    left = count;
  }
  __device__ __forceinline__ int count() const { return static_cast<int>(min(static_cast<long long>(len - off), left)); }
  // Past this segment; false at the end of the range.
  __device__ __forceinline__ bool next(const ChunkAttnArgs& a) {
    left -= count();
    if (left <= 0) return false;
    off = 0;
    if (++t == q.tiles) {
      t = 0;
      if (++h == a.kv_heads) {
        h = 0;
        do {
          q = ca_seq(a, ++b);
        } while (q.n == 0);
      }
    }
    len = ca_tile_len(q, t, a.qb);
    return true;
  }
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
  const int bytes = live ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Two bf16 in one conversion (the single conversions run on the
// transcendental pipe, at an eighth of the rate).
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// Pairs of fp32 operations in one instruction.
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// exp2_fma on a pair (2^x for x <= 8). x below -125, a masked key's -inf too,
// counts as -125: a row that sees any key has a sum of at least 2^-8, beside
// which 2^-125 is nothing, and ca_inverse tells a row that sees none by its
// sum.
__device__ __forceinline__ uint64_t exp2_fma2(float x, float y) {
  const uint64_t v = pair(fmaxf(x, -125.0f), fmaxf(y, -125.0f));
  const uint64_t t = add2(v, pair(12582912.0f, 12582912.0f));
  const uint64_t n = add2(t, pair(-12582912.0f, -12582912.0f));
  const uint64_t f = fma2(n, pair(-1.0f, -1.0f), v);
  uint64_t p = pair(0.009569993242621422f, 0.009569993242621422f);
  p = fma2(p, f, pair(0.055917542427778244f, 0.055917542427778244f));
  p = fma2(p, f, pair(0.240247443318367f, 0.240247443318367f));
  p = fma2(p, f, pair(0.6931218504905701f, 0.6931218504905701f));
  p = fma2(p, f, pair(0.9999992847442627f, 0.9999992847442627f));
  const float2 pf = unpair(p), tf = unpair(t);
  return pair(__int_as_float(__float_as_int(pf.x) + (__float_as_int(tf.x) << 23)),
              __int_as_float(__float_as_int(pf.y) + (__float_as_int(tf.y) << 23)));
}

// D (+)= A B with A in TMEM.
__device__ __forceinline__ void tc_mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t b_desc, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tc_st32(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
      "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
      "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}

// 1 / l, 0 for a row that saw no key (whose l is at most 2^-125 for each
// masked key), NaN for NaN.
__device__ __forceinline__ float ca_inverse(float l) { return l > 1e-20f ? 1.0f / l : (l == l ? 0.f : l); }

// Pair r of a split tile: the parts of ranges c0 .. c1 in that order.
template <int D>
__device__ __forceinline__ void ca_join(const ChunkAttnArgs& a, long long c0, long long c1, int r, bf16* dst) {
  for (int x0 = 0; x0 < D; x0 += 64) {
    float m = kNegBig, l = 0.f;
    float acc[64];
#pragma unroll
    for (int x = 0; x < 64; ++x) acc[x] = 0.f;
    for (long long k = c0; k <= c1; ++k) {
      const float* part = a.partials + static_cast<size_t>(2 * k + (k == c0 ? 1 : 0)) * ca_part_floats(D);
      const float pm = __ldcg(part + r), pl = __ldcg(part + kCaRows + r);
      const float nm = fmaxf(m, pm);
      const float wa = ex2_approx(m - nm), wb = ex2_approx(pm - nm);
      m = nm;
      l = l * wa + pl * wb;
      const float4* p4 = reinterpret_cast<const float4*>(part + 2 * kCaRows) + (x0 / 4) * kCaRows + r;
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const float4 v = __ldcg(p4 + x * kCaRows);
        acc[4 * x] = fmaf(v.x, wb, acc[4 * x] * wa);
        acc[4 * x + 1] = fmaf(v.y, wb, acc[4 * x + 1] * wa);
        acc[4 * x + 2] = fmaf(v.z, wb, acc[4 * x + 2] * wa);
        acc[4 * x + 3] = fmaf(v.w, wb, acc[4 * x + 3] * wa);
      }
    }
    const float inv = ca_inverse(l);
    uint4* d4 = reinterpret_cast<uint4*>(dst + x0);
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      d4[x] = make_uint4(pack2(acc[8 * x] * inv, acc[8 * x + 1] * inv),
                         pack2(acc[8 * x + 2] * inv, acc[8 * x + 3] * inv),
                         pack2(acc[8 * x + 4] * inv, acc[8 * x + 5] * inv),
                         pack2(acc[8 * x + 6] * inv, acc[8 * x + 7] * inv));
    }
  }
}

template <int D>
__global__ void __launch_bounds__(kCaThreads, 2) chunk_attn_kernel(const ChunkAttnArgs a) {
  using G = CaGeom<D>;
  constexpr int SLOTS = G::SLOTS;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* qs = smem;
  uint8_t* ring = smem + G::Q_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + SLOTS * G::SLOT);
  uint64_t* empty = full + SLOTS;
  uint64_t* q_full = empty + SLOTS;
  uint64_t* s_full = q_full + 1;  // [2]
  uint64_t* p_full = s_full + 2;  // [2]
  uint64_t* pv_done = p_full + 2;
  uint64_t* drain = pv_done + 1;
  uint64_t* stored = drain + 1;   // this CTA's part is in the workspace
  uint64_t* counted = stored + 1; // and counted: *last_s
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(full + G::BARS);
  int* last_s = reinterpret_cast<int*>(tmem_slot + 1);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // --- This CTA's range of blocks --------------------------------------------
  // Scratch of the scan, in the ring before its first use.
  struct Ends {
    long long part[kCaThreads / 32];
    long long at[2];    // the range's ends as offsets into their requests' blocks
    long long edge[2];  // and snapped, over all blocks
    int b[2];
  };
  Ends* e = reinterpret_cast<Ends*>(ring);
  const int per_thread = (a.sequences + kCaThreads - 1) / kCaThreads;
  const int b0 = min(a.sequences, tid * per_thread), b1 = min(a.sequences, b0 + per_thread);
  long long mine = 0;
  for (int b = b0; b < b1; ++b) mine += ca_seq(a, b).blocks * a.kv_heads;
  long long incl = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += x;
  }
  if (lane == 31) e->part[warp] = incl;
  __syncthreads();
  long long before = incl - mine, total = 0;
  for (int w = 0; w < kCaThreads / 32; ++w) {
    if (w < warp) before += e->part[w];
    total += e->part[w];
  }
  if (total == 0) return;
  // As many ranges as CTAs, fewer where each would be short.
  const long long ranges = min(static_cast<long long>(gridDim.x), max(1ll, total / kCaMinRange));
  const long long per = (total + ranges - 1) / ranges;
  const int c = blockIdx.x;
  if (c * per >= total) return;
  // An end that would leave a sliver of a tile moves to the tile's edge; the
  // two ranges that meet there move alike.
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const long long x = min(total, (c + k) * per);
    if (x == total) {
      if (tid == 0) e->edge[k] = total;
    } else if (x >= before && x < before + mine) {
      long long at = x - before;
      int b = b0;
      CaSeq q = ca_seq(a, b);
      while (at >= q.blocks * a.kv_heads) {
        at -= q.blocks * a.kv_heads;
        q = ca_seq(a, ++b);
      }
      CaWalk w;
      w.open(a, b, at, 1);
      int shift = 0;
      if (w.off < kCaMinPart) shift = -w.off;
      else if (w.len - w.off < kCaMinPart) shift = w.len - w.off;
      e->edge[k] = x + shift;
      if (k == 0) {
        // The snapped end may be the first block of a later request.
        at += shift;
        while (at >= q.blocks * a.kv_heads && b + 1 < a.sequences) {
          at -= q.blocks * a.kv_heads;
          q = ca_seq(a, ++b);
        }
        e->b[0] = b;
        e->at[0] = at;
      }
    }
  }
  __syncthreads();
  const long long lo = e->edge[0], hi = e->edge[1];
  const int first_b = e->b[0];
  const long long first_at = e->at[0];
  if (lo >= hi) return;  // the next range took it all
  __syncthreads();       // the scratch becomes the ring

  if (tid == 0) {
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(&full[s], 2);
      mbar_init(&empty[s], 1);
    }
    mbar_init(q_full, 4);
    for (int k = 0; k < 2; ++k) {
      mbar_init(&s_full[k], 1);
      mbar_init(&p_full[k], 4);
    }
    mbar_init(pv_done, 1);
    mbar_init(drain, 1);
    mbar_init(stored, 4);
    mbar_init(counted, 1);
    mbar_fence_init();
  }
  if (warp == 4) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)),
                 "r"(256)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const bool aligned = (smem_addr(smem) & 1023u) == 0;
  if (!aligned && tid == 0) atomicOr(a.status, kStatusBadSmem | kStatusAbort);

  if (!aligned) {
    // Nothing is in flight.
  } else if (warp >= 5) {
    // --- Loads: this warp's 32 keys of every block --------------------------
    const int half = warp - 5;
    int issued = 0;  // half-blocks (K, V, K, V, ...) issued / signalled
    bool ok = true;
    CaWalk w;
    w.open(a, first_b, first_at, hi - lo);
    // Signals the half-block issued LAG calls ago.
    auto signal = [&](int i) {
      cp_async_wait<G::LAG>();
      fence_proxy_async_smem();
      __syncwarp();
      if (i >= 0 && lane == 0) mbar_arrive(&full[i % SLOTS]);
    };
    const uint32_t ring_addr = smem_addr(ring);
    do {
      const int cnt = w.count();
      // Keys the tile's last row sees, of those cached.
      const long long seen = static_cast<long long>(w.q.kv) - w.q.n + min(static_cast<long long>(w.q.n), (w.t + 1ll) * a.qb);
      const int key_end = static_cast<int>(max(0ll, seen));
      const int32_t* table = a.tables + static_cast<size_t>(w.b) * a.max_pages;
      auto locate = [&](int j) {  // cache row (in 16-byte units) of this lane's key of block j; ~0u: zeros
        const int key = j * kCaBlock + half * 32 + lane;
        if (key >= key_end) return 0xffffffffu;
        const int page = table[key / a.page_size];
        if (page < 0 || page >= a.pool_pages) {
          atomicOr(a.status, kStatusBadPage);
          return 0xffffffffu;
        }
        return static_cast<uint32_t>(
            (page * a.page_stride + w.h * a.head_stride + static_cast<long long>(key % a.page_size) * D) >> 3);
      };
      uint32_t ahead = locate(w.off);
      for (int j = w.off; j < w.off + cnt && ok; ++j) {
        const uint32_t row = ahead;
        if (j + 1 < w.off + cnt) ahead = locate(j + 1);
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const int slot = issued % SLOTS;
          if (issued >= SLOTS) ok = mbar_wait(&empty[slot], ((issued / SLOTS) - 1) & 1, a.status, kStatusTimeoutEmpty);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          const bf16* base = kv == 0 ? a.keys : a.values;
          const uint32_t dst = ring_addr + slot * G::SLOT;
          // Lane l copies piece l % 8 of the rows l / 8, l / 8 + 4, ...
          const int piece = lane & 7;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = (lane >> 3) + 4 * i;
            const uint32_t at = __shfl_sync(0xffffffffu, row, r);
            const bool live = at != 0xffffffffu;
            const int key = half * 32 + r;
            const uint4* src = reinterpret_cast<const uint4*>(base) + (live ? at : 0u) + piece;
#pragma unroll
            for (int p = 0; p < G::PANELS; ++p) {
              cp_async16(dst + p * (kCaBlock * 128) + key * 128 + ((piece ^ (key & 7)) << 4), src + p * 8, live);
            }
          }
          cp_async_commit();
          ++issued;
          signal(issued - 1 - G::LAG);
        }
      }
    } while (ok && w.next(a));
    for (int k = 0; ok && k < G::LAG; ++k) {
      cp_async_commit();
      signal(issued + k - G::LAG);
    }
    cp_async_wait<0>();
  } else if (warp == 4) {
    // --- MMA issue -----------------------------------------------------------
    if (lane == 0) {
      const uint32_t idesc_s = tc_idesc<64>();
      const uint32_t idesc_pv = tc_idesc<64>() | (1u << 16);  // V MN-major
      const uint64_t qdesc = tc_desc_sw128(smem_addr(qs));
      const uint32_t ring_addr = smem_addr(ring);
      CaWalk w;
      w.open(a, first_b, first_at, hi - lo);
      int g = 0;  // blocks so far: S buffer g % 2, half-blocks 2 g and 2 g + 1
      int tile = 0;
      bool ok = true;
      // Every phase of pv_done is waited for in turn before the next but one
      // can complete: a parity tells only neighbouring phases apart.
      int pv_seen = 0;
      auto see_pv = [&](int upto) {
        for (; pv_seen <= upto; ++pv_seen) {
          if (!mbar_wait(pv_done, pv_seen & 1, a.status, kStatusTimeoutFull)) return false;
        }
        return true;
      };
      auto do_s = [&](int g, bool first) {
        const int i = 2 * g, slot = i % SLOTS;
        if (!mbar_wait(&full[slot], (i / SLOTS) & 1, a.status, kStatusTimeoutFull)) return false;
        // The buffer's P (block g - 2) has been used; at a tile's start block
        // g - 1 is issued too.
        if (!see_pv(first ? g - 1 : g - 2)) return false;
        tc_fence_after();
        const uint64_t kdesc = tc_desc_sw128(ring_addr + slot * G::SLOT);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const int p = k / 4, kk = k % 4;
          tc_mma(tmem + (g & 1) * 64u, qdesc + p * (kCaRows * 128 / 16) + 2 * kk,
                 kdesc + p * (kCaBlock * 128 / 16) + 2 * kk, idesc_s, k > 0 ? 1u : 0u);
        }
        tc_commit(&empty[slot]);
        tc_commit(&s_full[g & 1]);
        return true;
      };
      auto do_pv = [&](int g, bool fresh) {
        const int i = 2 * g + 1, slot = i % SLOTS;
        if (!mbar_wait(&full[slot], (i / SLOTS) & 1, a.status, kStatusTimeoutFull)) return false;
        if (!mbar_wait(&p_full[g & 1], (g >> 1) & 1, a.status, kStatusTimeoutFull)) return false;
        if (!see_pv(g - 1)) return false;
        tc_fence_after();
        const uint32_t vbase = ring_addr + slot * G::SLOT;
#pragma unroll
        for (int k = 0; k < kCaBlock / 16; ++k) {
#pragma unroll
          for (int p = 0; p < G::PANELS; ++p) {
            tc_mma_ts(tmem + G::O_COL + p * 64u, tmem + (g & 1) * 64u + k * 8u,
                      ap_vdesc(vbase + p * (kCaBlock * 128) + k * 2048), idesc_pv, (!fresh || k > 0) ? 1u : 0u);
          }
        }
        tc_commit(&empty[slot]);
        tc_commit(pv_done);
        return true;
      };
      do {
        const int cnt = w.count();
        ok = mbar_wait(q_full, tile & 1, a.status, kStatusTimeoutFull);
        for (int j = 0; j < cnt && ok; ++j) {
          ok = do_s(g + j, j == 0);
          if (ok && j > 0) ok = do_pv(g + j - 1, j == 1);
        }
        if (ok) ok = do_pv(g + cnt - 1, cnt == 1);
        g += cnt;
        ++tile;
      } while (ok && w.next(a));
      if (!ok) atomicOr(a.status, kStatusAbort);
      tc_commit(drain);
      mbar_wait(drain, 0, nullptr, 0);  // the MMAs in flight land even after an abort
    }
  } else {
    // --- Softmax and epilogue: thread = pair r of the tile = TMEM lane --------
    const int r = tid;
    const int qi = r / a.group, hl = r % a.group;
    const uint32_t trow = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    CaWalk w;
    w.open(a, first_b, first_at, hi - lo);
    int g = 0;
    bool ok = true;
    int parts = 0;        // parts stored so far
    long long done = lo;  // blocks of all tiles before this segment
    do {
      const int cnt = w.count();
      const int row = w.t * a.qb + qi;  // of the request
      const bool live = qi < a.qb && row < w.q.n;
      const long long head = static_cast<long long>(w.h * a.group + hl) * D;
      // Every S of the tile before has landed (its last block's was waited for).
      {
        const uint4* src = reinterpret_cast<const uint4*>(a.q + (live ? (w.q.row0 + row) * a.q_stride + head : 0));
#pragma unroll
        for (int p = 0; p < G::PANELS; ++p) {
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            const uint4 v = live ? src[p * 8 + x] : make_uint4(0u, 0u, 0u, 0u);
            *reinterpret_cast<uint4*>(qs + p * (kCaRows * 128) + r * 128 + ((x ^ (r & 7)) << 4)) = v;
          }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
      const int pos = live ? w.q.kv - w.q.n + row : -1;  // keys 0 .. pos
      // The lowest position of the tile's rows: blocks that end below it need no mask.
      const int low = w.q.kv - w.q.n + w.t * a.qb;
      // A warp without a live pair (a request of a few rows fills the first
      // warp at most) only keeps the barriers going.
      const bool idle = !__any_sync(0xffffffffu, live);
      float m = kNegBig, l = 0.f;
      for (int j = 0; j < cnt; ++j, ++g) {
        ok = __all_sync(0xffffffffu, mbar_wait(&s_full[g & 1], (g >> 1) & 1, a.status, kStatusTimeoutFull));
        if (!ok) break;
        tc_fence_after();
        if (idle) {
          if (j > 0) ok = __all_sync(0xffffffffu, mbar_wait(pv_done, (g - 1) & 1, a.status, kStatusTimeoutFull));
          if (!ok) break;
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[g & 1]);
          continue;
        }
        const uint32_t tbuf = trow + (g & 1) * 64u;
        float s[64];
#pragma unroll
        for (int x = 0; x < 64; x += 16) {
          float t16[16];
          tc_ld16(tbuf + x, t16);
#pragma unroll
          for (int y = 0; y < 16; ++y) s[x + y] = t16[y];
        }
        tc_wait_ld();
        const int key0 = (w.off + j) * kCaBlock;
        if (key0 + kCaBlock - 1 > low) {
          const int lim = pos - key0;
#pragma unroll
          for (int x = 0; x < 64; ++x) {
            if (x > lim) s[x] = -INFINITY;
          }
        }
        float mx[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          mx[x] = fmaxf(fmaxf(fmaxf(s[8 * x], s[8 * x + 1]), fmaxf(s[8 * x + 2], s[8 * x + 3])),
                        fmaxf(fmaxf(s[8 * x + 4], s[8 * x + 5]), fmaxf(s[8 * x + 6], s[8 * x + 7])));
        }
        const float top = fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])),
                                fmaxf(fmaxf(mx[4], mx[5]), fmaxf(mx[6], mx[7]))) * a.scale_log2;
        const bool grow = top > m + 8.0f;  // false for a row with no key yet: m stays at its lowest
        const float na = grow ? top : m;
        const float alpha = ex2_approx(m - na);
        uint32_t pk[32];
        uint64_t sums[4] = {0, 0, 0, 0};
        const uint64_t scale2 = pair(a.scale_log2, a.scale_log2), shift2 = pair(-na, -na);
#pragma unroll
        for (int x = 0; x < 32; ++x) {
          const float2 z = unpair(fma2(pair(s[2 * x], s[2 * x + 1]), scale2, shift2));
          const uint64_t p = (x & 7) >= 8 - kCaFmaGroups ? exp2_fma2(z.x, z.y) : pair(ex2_approx(z.x), ex2_approx(z.y));
          sums[x & 3] = add2(sums[x & 3], p);
          const float2 pf = unpair(p);
          pk[x] = pack2(pf.x, pf.y);
        }
        const float2 sum = unpair(add2(add2(sums[0], sums[1]), add2(sums[2], sums[3])));
        l = fmaf(l, alpha, sum.x + sum.y);
        m = na;
        tc_st32(tbuf, pk);
        if (j > 0) {
          // O of the blocks before this one is complete and may be rescaled.
          // (Waited for in every block: a parity tells only neighbouring
          // phases apart.)
          ok = __all_sync(0xffffffffu, mbar_wait(pv_done, (g - 1) & 1, a.status, kStatusTimeoutFull));
          if (!ok) break;
          tc_fence_after();
          if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int x = 0; x < D; x += 16) {
              float o16[16];
              tc_ld16(trow + G::O_COL + x, o16);
              tc_wait_ld();
#pragma unroll
              for (int y = 0; y < 16; ++y) o16[y] *= alpha;
              tc_st16(trow + G::O_COL + x, o16);
            }
          }
        }
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[g & 1]);
      }
      if (!ok) break;
      ok = __all_sync(0xffffffffu, mbar_wait(pv_done, (g - 1) & 1, a.status, kStatusTimeoutFull));
      if (!ok) break;
      tc_fence_after();
      bf16* dst = a.out + (live ? (w.q.row0 + row) * a.out_stride + head : 0);
      if (cnt == w.len) {
        const float inv = ca_inverse(l);
#pragma unroll
        for (int x = 0; x < D; x += 16) {
          float o[16];
          tc_ld16(trow + G::O_COL + x, o);
          tc_wait_ld();
          if (live) {
            uint4* d4 = reinterpret_cast<uint4*>(dst + x);
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              d4[y] = make_uint4(pack2(o[8 * y] * inv, o[8 * y + 1] * inv), pack2(o[8 * y + 2] * inv, o[8 * y + 3] * inv),
                                 pack2(o[8 * y + 4] * inv, o[8 * y + 5] * inv),
                                 pack2(o[8 * y + 6] * inv, o[8 * y + 7] * inv));
            }
          }
        }
      } else {
        // A part: columns of four as [column / 4][pair], so neighbouring
        // threads' 16 bytes are neighbours.
        const long long tile0 = done - w.off, tile1 = tile0 + w.len;
        float* part = a.partials + static_cast<size_t>(2 * c + (w.off > 0 ? 0 : 1)) * ca_part_floats(D);
        if (live) {
          part[r] = m;
          part[kCaRows + r] = l;
        }
#pragma unroll
        for (int x = 0; x < D; x += 16) {
          float o[16];
          tc_ld16(trow + G::O_COL + x, o);
          tc_wait_ld();
          if (live) {
            float4* p4 = reinterpret_cast<float4*>(part + 2 * kCaRows);
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              p4[(x / 4 + y) * kCaRows + r] = make_float4(o[4 * y], o[4 * y + 1], o[4 * y + 2], o[4 * y + 3]);
            }
          }
        }
        // The ranges that hold the tile's first and last block, by the same
        // snapping as the ranges' own ends.
        long long c0 = tile0 / per, c1 = (tile1 - 1) / per;
        if ((c0 + 1) * per < tile1 && (c0 + 1) * per - tile0 < kCaMinPart) ++c0;
        if (c1 * per > tile0 && c1 * per - tile0 >= kCaMinPart && tile1 - c1 * per < kCaMinPart) --c1;
        __threadfence();
        __syncwarp();
        if (lane == 0) mbar_arrive(stored);
        ok = __all_sync(0xffffffffu, mbar_wait(stored, parts & 1, a.status, kStatusTimeoutFull));
        if (!ok) break;
        if (tid == 0) {
          const unsigned n = atomicAdd(&a.counters[c0], 1u) + 1u;
          const bool last = n == static_cast<unsigned>(c1 - c0 + 1);
          if (last) a.counters[c0] = 0u;
          *last_s = last;
          __threadfence();
          mbar_arrive(counted);
        }
        ok = __all_sync(0xffffffffu, mbar_wait(counted, parts & 1, a.status, kStatusTimeoutFull));
        if (!ok) break;
        ++parts;
        if (*last_s && live) ca_join<D>(a, c0, c1, r, dst);
      }
      tc_fence_before();  // O and S were read: the next tile's MMAs may write them
      done += cnt;
    } while (w.next(a));
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 4) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256) : "memory");
  }
}

}  // namespace lcrb
