// Attention of every request's new rows over its paged cache
// (lcr_chunk_attention) on the 5th-generation tensor cores: row i of the n
// rows of request b is at position p = kv_length - n + i and sees keys 0 .. p.
//
// Tiles. A tile is one KV head of one request and up to 128 of its (row, query
// head) pairs: QB = 128 / G' rows (G' = the group rounded up to a power of
// two) by the G heads of the group, pair r = row * G + head, so that a few
// rows of a decoding request fill the lowest lanes. Keys come in blocks of as
// many keys as a head has dimensions:
//
//   S = Q K^T          m128 k16, both from shared memory (K-major, 128-byte
//                      swizzle), into TMEM
//   softmax            one thread per pair (TMEM lane): maximum and sum in the
//                      log2 domain, held in fp32; P rounded to bf16 -- the
//                      tensor cores' operand; its share of the result's error
//                      is that of the output's own rounding -- and stored over
//                      S in TMEM
//   O += P V           m128 k16, P from TMEM, V in place as an MN-major operand
//                      (its rows are keys), O in TMEM
//
// The running maximum moves only when a block's exceeds it by more than 8 (a
// factor of 256): P and the sum use the same stale maximum, so O / l is
// unchanged, and rescaling O (a round trip through registers) is rare.
//
// One tile's chain (S, softmax, P V) is a sequence of latencies, and a softmax
// warp alone keeps no pipe busy, so several CTAs share an SM, each with a
// chain of its own: four for head_dim 64, two for head_dim 128 (what S and O
// leave of the 512 TMEM columns).
//
// Work. Lengths are known only on the device, and tiles cost from one block to
// thousands, so the blocks of all tiles (in order of request, KV head, rows)
// are laid end to end and every CTA takes an equal contiguous range of them:
// each CTA sums the requests' block counts (a closed form) and finds its range
// without a second launch. A tile that spans several ranges leaves one partial
// (m, l, O) for each in the workspace; the CTA that stores its partial last (a
// counter per split tile) joins them in range order, so the result does not
// depend on which one that is.
//
// Loads. One warp fills a ring of 128-byte wide panels of K and V in the
// swizzled layout, ahead across tiles. Where the pool is dense and a page holds
// a multiple of 16 positions, by tensor copies of 16 to 128 keys; else 16 bytes
// at a time (cp.async), each lane holding the cache rows of its keys, for any
// page size and strides (the first three cases below, on pages of 16: 59, 42
// and 801 us by tensor copies, 61, 51 and 878 by cp.async). Keys past the tile's
// last position are never read and enter as zeros, so what lies there cannot
// reach the sums.
//
// What it measured, with 32 query and 8 KV heads, and what bounds it:
//   64 requests of 1 - 5 rows on 128 - 4096 keys, heads of 64: 59 us for 279 MB
//     of keys and values, 4.7 TB/s, 0.72 of a copy's rate. Memory, and 9 us of
//     start (the scan, the first loads) and of joining split tiles. (With one row
//     each 58 us, and 100 with heads of 128, 5.6 TB/s.)
//   15 of these beside a chunk of 509 rows, heads of 128: 42 us for 130 MB, 0.47
//     of a copy's rate. The chain of a block, 4 - 5 thousand cycles while loads
//     come late, about ten blocks a CTA.
//   2048 rows on 32768 keys, heads of 64: 806 us (790 - 828 between runs), 661
//     TFLOP/s, 0.39 of a large product's rate. The chain again: 2900 cycles a
//     block, of them 1500 in the softmax warps (shared with the other CTAs'), the
//     rest the way to the tensor cores and back; tensor cores 41 % and
//     transcendental pipe 50 % busy, issue slots 57 %.
//   2048 rows on 8192 keys, heads of 128: 275 us, 873 TFLOP/s, 0.52. The chain, two
//     of them an SM, and a ring that holds one block's K and V: tensor cores 45 %,
//     transcendental pipe 37 %, issue slots 39 %; 2 GB out of L2, which is 27 % busy.
//   5 rows on 250 keys, heads of 64: 9.8 us, latency from end to end.
// Measured and no faster: P signalled in halves, so that P V starts early (812
// us for the third case, 811 without); the last 32 scores kept in registers
// between the two passes (809, spills); the next K waited for ahead of P (the
// second case 48 us: P V, whose slots the loads need, came late); blocks of 128
// keys with P beside S, for two CTAs an SM; two load warps for heads of 128.
//
// Warps: 0-3 softmax (warp w owns TMEM lanes 32 w .. + 31) and epilogue, 4
// TMEM allocation and MMA issue, 5 loads. Every wait is bounded.
#pragma once

#include "attn_prefill_tc.cuh"
#include "common.cuh"
#include "gemm_tc.cuh"

namespace lcrb {

constexpr int kCaThreads = 192;
constexpr int kCaRows = 128;      // (row, head) pairs per tile
// In units of a block of BLK keys (64 or 128); chosen by timing 64 requests of 1
// - 5 rows on 128 - 4096 keys (BLK 64: 77, 71, 71 us at a cost of 2, 3, 4) and a
// chunk of 509 rows beside 15 such requests (BLK 128: 49, 45 us at a reach of 2, 3).
template <int BLK>
constexpr int ca_tile_cost() {  // what a tile's start and end count for
  return BLK == 64 ? 3 : 2;
}
template <int BLK>
constexpr int ca_reach() {  // a range's end moves to a tile's end this near
  return BLK == 64 ? 4 : 3;
}
template <int BLK>
constexpr int ca_min_range() {  // units of a range at least (where there are as many); at least ca_reach
  return ca_reach<BLK>();
}
// Of 8 pairs of exponentials, on the FMA pipe (2048 rows on 32768 keys: 806 us, with
// none 828, medians of 40 runs of each in turn; 59 and 43 us with either in the
// first two cases).
constexpr int kCaFmaGroups = 1;

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
  int log2_qb;          // rows per tile: 2^log2_qb
  int log2_unit;        // keys per tensor copy: 2^log2_unit, at most a page and a block
  int pool_rows;        // rows of head_dim in a pool (tensor copies)
  unsigned page_mul, page_shift;  // key / page_size = umulhi(key, page_mul) >> page_shift (page_size > 1)
  float scale_log2;
  uint32_t* status;
  unsigned* counters;   // [grid], zero between calls
  float* partials;      // [2 * grid] parts of ca_part_floats(D)
};

constexpr size_t ca_part_floats(int d) { return static_cast<size_t>(kCaRows) * (d + 2); }

template <int D>
struct CaGeom {
  static constexpr int PANELS = D / 64;            // 128-byte wide panels
  static constexpr int BLOCK = D;                  // keys per block
  static constexpr int CTAS = D == 64 ? 4 : 2;     // per SM, by TMEM
  static constexpr int Q_BYTES = PANELS * kCaRows * 128;
  static constexpr int SLOT = BLOCK * 128;         // one panel of a block's K or V
  static constexpr int SLOTS = 4;
  static constexpr int LAG = 2;                    // loads in flight before the oldest is waited for
  static constexpr int BARS = 2 * SLOTS + 7;
  static constexpr size_t SMEM = Q_BYTES + SLOTS * SLOT + BARS * 8 + 64;
  static constexpr uint32_t TMEM = 2 * D;          // columns: S, with P over its first half, then O
  static constexpr uint32_t O_COL = D;
  static_assert(LAG < SLOTS, "a load is signalled before its slot's next use");
  static_assert(SLOTS % PANELS == 0, "the panels of a block's V lie side by side in the ring");
};

// Blocks of a request's tiles 0 .. t - 1 for one KV head (t < its tiles),
// each tile reaching to key s + (t + 1) * qb: the sum of ceil((s + i qb) / BLK)
// for i = 1 .. t, by shifts. (The host refuses steps of 2^31 blocks.)
template <int BLK>
__device__ __forceinline__ int ca_blocks_before(int s, int t, int log2_qb) {
  constexpr int LOG2_BLK = BLK == 64 ? 6 : 7;
  const unsigned a = static_cast<unsigned>(s) + BLK - 1, n = static_cast<unsigned>(t);
  if (log2_qb >= LOG2_BLK) return static_cast<int>(n * (a >> LOG2_BLK) + ((n * (n + 1) / 2) << (log2_qb - LOG2_BLK)));
  const int e = LOG2_BLK - log2_qb;
  auto below = [e](unsigned m) {  // sum of i >> e for i < m
    const unsigned k = m >> e;
    return ((k * (k - 1) / 2) << e) + k * (m - (k << e));
  };
  const unsigned a1 = a >> log2_qb;
  return static_cast<int>(below(a1 + n + 1) - below(a1 + 1));
}

// Ranges are cut in units of blocks with ca_tile_cost units added in front of
// every tile, about what a change of tiles costs (Q, the first S, the
// epilogue): a range with many short tiles gets fewer blocks.

template <int BLK>
__device__ __forceinline__ int ca_units_before(int s, int t, int log2_qb) {
  return ca_blocks_before<BLK>(s, t, log2_qb) + t * ca_tile_cost<BLK>();
}

// One request as the kernel sees it: malformed lengths are cut to what the
// arrays hold.
struct CaSeq {
  int row0, n;  // rows
  int kv;       // cached positions
  int s;        // max(0, kv - n): where the block count starts
  int tiles;
  int units;    // of one KV head
};

template <int BLK>
__device__ __forceinline__ CaSeq ca_seq(const ChunkAttnArgs& a, int b) {
  CaSeq q;
  q.row0 = min(max(0, a.row_starts[b]), a.rows);
  q.n = max(0, min(max(0, a.row_starts[b + 1]), a.rows) - q.row0);
  q.kv = min(max(0, a.kv_lengths[b]), a.max_pages * a.page_size);
  q.s = max(0, q.kv - q.n);
  q.tiles = (q.n + (1 << a.log2_qb) - 1) >> a.log2_qb;
  q.units = q.tiles == 0 ? 0
                         : ca_units_before<BLK>(q.s, q.tiles - 1, a.log2_qb) + (q.s + q.n + BLK - 1) / BLK + ca_tile_cost<BLK>();
  return q;
}

template <int BLK>
__device__ __forceinline__ int ca_tile_len(const CaSeq& q, int t, int log2_qb) {
  return (q.s + min(q.n, (t + 1) << log2_qb) + BLK - 1) / BLK;
}

// A CTA's walk over its range of units, segment by segment (a segment = its
// share of one tile, in whole blocks). Every warp walks for itself.
template <int BLK>
struct CaWalk {
  int b, h, t;
  CaSeq q;
  int len;   // blocks of the tile
  int at;    // units of the tile before this segment
  int left;  // units of the range from here on

  // To unit `from` of request b0's.
  __device__ __forceinline__ void find(const ChunkAttnArgs& a, int b0, int from) {
    b = b0;
    q = ca_seq<BLK>(a, b);
    h = from / q.units;
    const int rem = from - h * q.units;
    int lo = 0, hi = q.tiles - 1;  // the last tile that begins at or before rem
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (ca_units_before<BLK>(q.s, mid, a.log2_qb) <= rem) lo = mid;
      else hi = mid - 1;
    }
    t = lo;
    at = rem - ca_units_before<BLK>(q.s, t, a.log2_qb);
    len = ca_tile_len<BLK>(q, t, a.log2_qb);
  }
  __device__ __forceinline__ void open(const ChunkAttnArgs& a, int b0, int h0, int t0, int at0, int units) {
    b = b0;
    h = h0;
    t = t0;
    at = at0;
    left = units;
    q = ca_seq<BLK>(a, b);
    len = ca_tile_len<BLK>(q, t, a.log2_qb);
  }
  __device__ __forceinline__ int units() const { return min(len + ca_tile_cost<BLK>() - at, left); }
  __device__ __forceinline__ int off() const { return max(0, at - ca_tile_cost<BLK>()); }  // first block of the segment
  __device__ __forceinline__ int count() const { return max(0, at + units() - ca_tile_cost<BLK>()) - off(); }  // its blocks
  // Keys the tile's last row sees, of those cached.
  __device__ __forceinline__ int key_end(const ChunkAttnArgs& a) const {
    return max(0, q.kv - q.n + min(q.n, (t + 1) << a.log2_qb));
  }
  // To the start of the next tile (there is one).
  __device__ __forceinline__ void advance(const ChunkAttnArgs& a) {
    at = 0;
    if (++t == q.tiles) {
      t = 0;
      if (++h == a.kv_heads) {
        h = 0;
        do {
          q = ca_seq<BLK>(a, ++b);
        } while (q.n == 0);
      }
    }
    len = ca_tile_len<BLK>(q, t, a.log2_qb);
  }
  // Past this segment; false at the end of the range.
  __device__ __forceinline__ bool next(const ChunkAttnArgs& a) {
    left -= units();
    if (left <= 0) return false;
    advance(a);
    return true;
  }
};

// How far an end of a range that lies `at` units into a tile of `units` moves:
// splitting a tile costs its CTAs about as much as `reach` units (a part stored,
// counted and joined). Ends are at least `reach` apart, so that only one of a
// tile's moves to each of its own ends.
__device__ __forceinline__ int ca_snap(int at, int units, int reach) {
  return at <= reach ? -at : units - at <= reach ? units - at : 0;
}
// The range that unit `y` of the tile [begin, begin + units) falls to.
__device__ __forceinline__ int ca_owner(int y, int begin, int units, int per, int reach) {
  const int c = y / per, from = c * per - begin, to = from + per;
  if (from > 0 && ca_snap(from, units, reach) > 0) return c - 1;
  if (to < units && ca_snap(to, units, reach) < 0) return c + 1;
  return c;
}

// mbar_wait with its slow path out of line: the kernel waits in many places,
// and its loops should stay within the instruction caches.
__device__ __noinline__ bool ca_wait_slow(uint64_t* bar, uint32_t parity, uint32_t* status, uint32_t code) {
  return mbar_wait(bar, parity, status, code);
}
__device__ __forceinline__ bool ca_wait(uint64_t* bar, uint32_t parity, uint32_t* status, uint32_t code) {
  return mbar_try_wait(bar, parity) || ca_wait_slow(bar, parity, status, code);
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
  const int bytes = live ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ float max3(float x, float y, float z) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
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

// One tensor copy: rows `row` .. of a pool, 64 columns of panel `panel`.
__device__ __forceinline__ void ca_tma(uint32_t dst, const CUtensorMap* map, int row, int panel, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::
          "r"(dst),
      "l"(map), "r"(0), "r"(row), "r"(panel), "r"(smem_addr(bar))
      : "memory");
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
__device__ __forceinline__ void tc_st16u(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tc_ld32(uint32_t taddr, float (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
        "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
        "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(taddr)
      : "memory");
}

// Descriptor of 16 keys of V as the MN-major B operand: rows (keys) of 128
// bytes, 8-row groups 1024 bytes apart, panels of 64 dimensions `panel` bytes
// apart.
__device__ __forceinline__ uint64_t ca_vdesc(uint32_t smem_addr, uint32_t panel) {
  return static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(panel >> 4) << 16) | (64ull << 32) |
         (1ull << 46) | (2ull << 61);
}
// One lane of a converged warp, the same at every use of the result.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}
// bf16 operands, fp32 accumulator, M = 128, N = n (tc_idesc as a constant).
constexpr uint32_t ca_idesc(int n) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(kTcTileM >> 4) << 24);
}

// 1 / l, 0 for a row that saw no key (whose l is at most 2^-125 for each
// masked key), NaN for NaN.
__device__ __forceinline__ float ca_inverse(float l) { return l > 1e-20f ? 1.0f / l : (l == l ? 0.f : l); }

// 32 scores of this lane, those past column lim masked.
__device__ __forceinline__ void ca_fetch(uint32_t taddr, float (&v)[32], bool masked, int lim) {
  tc_ld32(taddr, v);
  tc_wait_ld();
  if (masked) {
    asm volatile("" ::: "memory");  // a branch, not 32 predicated selects in every block
#pragma unroll
    for (int x = 0; x < 32; ++x) {
      if (x > lim) v[x] = -INFINITY;
    }
  }
}
__device__ __forceinline__ float ca_most(const float (&v)[32], float top) {
  float mx[4] = {top, v[0], v[1], v[2]};
#pragma unroll
  for (int x = 3; x < 31; x += 2) mx[(x / 2) & 3] = max3(mx[(x / 2) & 3], v[x], v[x + 1]);
  return max3(max3(mx[0], mx[1], mx[2]), mx[3], v[31]);
}
// Their weights as bf16 pairs, and the weights' sums.
__device__ __forceinline__ void ca_weigh(const float (&v)[32], uint64_t scale2, uint64_t shift2, uint64_t (&sums)[2],
                                         uint32_t (&pk)[16]) {
#pragma unroll
  for (int x = 0; x < 16; ++x) {
    const float2 z = unpair(fma2(pair(v[2 * x], v[2 * x + 1]), scale2, shift2));
    const uint64_t p = (x & 7) >= 8 - kCaFmaGroups ? exp2_fma2(z.x, z.y) : pair(ex2_approx(z.x), ex2_approx(z.y));
    sums[x & 1] = add2(sums[x & 1], p);
    const float2 pf = unpair(p);
    pk[x] = pack2(pf.x, pf.y);
  }
}

// Joins the parts of a split tile, of ranges c0 .. c1 in that order. A thread
// takes 8 columns of a pair at a time.
template <int D>
__device__ __forceinline__ void ca_join(const ChunkAttnArgs& a, int c0, int c1, int pairs, bf16* out, int tid) {
#pragma unroll 1
  for (int item = tid; item < pairs * (D / 8); item += kCaRows) {
    const int pair_r = item % pairs, x = item / pairs;
    float m = kNegBig, l = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int k0 = c0; k0 <= c1; k0 += 4) {
      float pm[4], pl[4];
      float4 v[4][2];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = min(k0 + i, c1);
        const float* part = a.partials + static_cast<size_t>(2 * k + (k == c0 ? 1 : 0)) * ca_part_floats(D);
        pm[i] = k0 + i <= c1 ? __ldcg(part + pair_r) : kNegBig;
        pl[i] = __ldcg(part + kCaRows + pair_r);
        const float4* p4 = reinterpret_cast<const float4*>(part + 2 * kCaRows) + pair_r;
        v[i][0] = __ldcg(p4 + 2 * x * kCaRows);
        v[i][1] = __ldcg(p4 + (2 * x + 1) * kCaRows);
      }
      const float nm = fmaxf(fmaxf(fmaxf(m, pm[0]), fmaxf(pm[1], pm[2])), pm[3]);
      const float wa = ex2_approx(m - nm);
      m = nm;
      l *= wa;
#pragma unroll
      for (int y = 0; y < 8; ++y) acc[y] *= wa;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float wb = k0 + i <= c1 ? ex2_approx(pm[i] - nm) : 0.f;
        l = fmaf(pl[i], wb, l);
        acc[0] = fmaf(v[i][0].x, wb, acc[0]);
        acc[1] = fmaf(v[i][0].y, wb, acc[1]);
        acc[2] = fmaf(v[i][0].z, wb, acc[2]);
        acc[3] = fmaf(v[i][0].w, wb, acc[3]);
        acc[4] = fmaf(v[i][1].x, wb, acc[4]);
        acc[5] = fmaf(v[i][1].y, wb, acc[5]);
        acc[6] = fmaf(v[i][1].z, wb, acc[6]);
        acc[7] = fmaf(v[i][1].w, wb, acc[7]);
      }
    }
    const float inv = ca_inverse(l);
    const int row = pair_r / a.group;
    *reinterpret_cast<uint4*>(out + row * a.out_stride + (pair_r - row * a.group) * D + 8 * x) =
        make_uint4(pack2(acc[0] * inv, acc[1] * inv), pack2(acc[2] * inv, acc[3] * inv), pack2(acc[4] * inv, acc[5] * inv),
                   pack2(acc[6] * inv, acc[7] * inv));
  }
}

template <int D, bool TMA>
__global__ void __launch_bounds__(kCaThreads, CaGeom<D>::CTAS) chunk_attn_kernel(const ChunkAttnArgs a,
                                                                                const __grid_constant__ CUtensorMap kmap,
                                                                                const __grid_constant__ CUtensorMap vmap) {
  using G = CaGeom<D>;
  constexpr int SLOTS = G::SLOTS, BLOCK = G::BLOCK, COST = ca_tile_cost<BLOCK>();
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* qs = smem;
  uint8_t* ring = smem + G::Q_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + SLOTS * G::SLOT);
  uint64_t* empty = full + SLOTS;
  uint64_t* q_full = empty + SLOTS;
  uint64_t* s_full = q_full + 1;
  uint64_t* p_full = s_full + 1;
  uint64_t* pv_done = p_full + 1;
  uint64_t* drain = pv_done + 1;
  uint64_t* stored = drain + 1;    // this CTA's part is in the workspace
  uint64_t* counted = stored + 1;  // and counted: *last_s
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(full + G::BARS);
  int* last_s = reinterpret_cast<int*>(tmem_slot + 1);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // TMEM first: an SM starts its next CTA only when this one has allocated
  // (a CTA that allocated 2 us into its run held the next one up as long).
  if (warp == 4) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)),
                 "r"(G::TMEM)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 0) {
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(q_full, 4);
    mbar_init(s_full, 1);
    mbar_init(p_full, 4);
    mbar_init(pv_done, 1);
    mbar_init(drain, 1);
    mbar_init(stored, 4);
    mbar_init(counted, 1);
    mbar_fence_init();
  }

  // --- This CTA's range of units --------------------------------------------
  // Scratch of the scan, in the ring before its first use.
  struct Start {
    int part[kCaThreads / 32];
    int b, h, t, at;
    int edge[2];
  };
  Start* st = reinterpret_cast<Start*>(ring);
  const int per_thread = (a.sequences + kCaThreads - 1) / kCaThreads;
  const int b0 = min(a.sequences, tid * per_thread), b1 = min(a.sequences, b0 + per_thread);
  int mine = 0;
  for (int b = b0; b < b1; ++b) mine += ca_seq<BLOCK>(a, b).units * a.kv_heads;
  int incl = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += x;
  }
  if (lane == 31) st->part[warp] = incl;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  int before = incl - mine, total = 0;
#pragma unroll
  for (int x = 0; x < kCaThreads / 32; ++x) {
    const int p = st->part[x];
    if (x < warp) before += p;
    total += p;
  }
  // As many ranges as CTAs, fewer where each would be short.
  const int ranges = min(static_cast<int>(gridDim.x), max(1, total / ca_min_range<BLOCK>()));
  const int per = (total + ranges - 1) / ranges;
  const int c = blockIdx.x;
  // Both ends, snapped; the thread whose requests hold an end finds it.
#pragma unroll 1
  for (int k = 0; k < 2; ++k) {
    const long long raw = static_cast<long long>(c + k) * per;
    if (raw >= total) {
      if (tid == 0) st->edge[k] = total;
    } else if (raw >= before && raw < before + mine) {
      int at = static_cast<int>(raw) - before, b = b0;
      for (int n = ca_seq<BLOCK>(a, b).units * a.kv_heads; at >= n; n = ca_seq<BLOCK>(a, b).units * a.kv_heads) {
        at -= n;
        ++b;
      }
      CaWalk<BLOCK> e;
      e.find(a, b, at);
      const int shift = ca_snap(e.at, e.len + COST, ca_reach<BLOCK>());
      const int edge = static_cast<int>(raw) + shift;
      st->edge[k] = edge;
      if (k == 0) {
        e.at += shift;
        if (shift > 0 && edge < total) e.advance(a);
        st->b = e.b;
        st->h = e.h;
        st->t = e.t;
        st->at = e.at;
      }
    }
  }
  __syncthreads();
  const int lo = st->edge[0], hi = st->edge[1];
  const bool some = lo < hi;
  const int start_b = st->b, start_h = st->h, start_t = st->t, start_at = st->at;
  __syncthreads();  // the scratch becomes the ring

  const uint32_t tmem = *tmem_slot;
  const bool aligned = (smem_addr(smem) & 1023u) == 0;
  if (!aligned && tid == 0) atomicOr(a.status, kStatusBadSmem | kStatusAbort);
  CaWalk<BLOCK> w;
  if (some) w.open(a, start_b, start_h, start_t, start_at, hi - lo);

  if (!aligned || !some) {
    // Nothing is in flight.
  } else if (warp == 5 && TMA) {
    // --- Loads by tensor copies ----------------------------------------------
    // A slot's keys come in units that lie within a page: lane u looks up unit
    // u of a block (one block ahead) and lane 0 copies it. The keys of the
    // unit that the tile's last position ends in are copied one by one, zeros
    // after them up to a multiple of 16: the MMA warp uses no later ones.
    int issued = 0;  // slots (the panels of a block's K, of its V, ...) issued
    bool ok = true;
    const uint32_t ring_addr = smem_addr(ring);
    auto page_of = [&](int key) { return static_cast<int>(__umulhi(static_cast<unsigned>(key), a.page_mul) >> a.page_shift); };
    const bool leader = elect_one();
    if (leader) {
      prefetch_tensormap(&kmap);
      prefetch_tensormap(&vmap);
    }
    do {
      const int cnt = w.count(), off = w.off(), key_end = w.key_end(a);
      const int32_t* table = a.tables + static_cast<size_t>(w.b) * a.max_pages;
      int page = -1;
      auto look = [&](int j) {
        const int key = j * BLOCK + (lane << a.log2_unit);
        page = lane < (BLOCK >> a.log2_unit) && key < key_end ? __ldg(table + page_of(key)) : -1;
      };
      if (cnt > 0) look(off);
      for (int j = off; j < off + cnt && ok; ++j) {
        // This lane's unit as a row of the pool; past its end (which reads as
        // zeros) for a page outside it.
        const int key = j * BLOCK + (lane << a.log2_unit);
        const bool in = page >= 0 && page < a.pool_pages;
        if (!in && lane < (BLOCK >> a.log2_unit) && key < key_end) atomicOr(a.status, kStatusBadPage);
        const int row = in ? (page * a.kv_heads + w.h) * a.page_size + key - page_of(key) * a.page_size : a.pool_rows;
        if (j + 1 < off + cnt) look(j + 1);
        const int live = min(max(key_end - j * BLOCK, 0), BLOCK);
        const int units = live >> a.log2_unit;
        const int done = units << a.log2_unit, rest = max(16, (live + 15) & ~15) - done;  // rest < 0: the block is full
        const int last = __shfl_sync(0xffffffffu, row, units & 31);
        int at[BLOCK / 16];
#pragma unroll
        for (int u = 0; u < BLOCK / 16; ++u) at[u] = __shfl_sync(0xffffffffu, row, u);
#pragma unroll 1
        for (int x = 0; x < 2 * G::PANELS; ++x) {  // K's panels, then V's
          const int slot = issued % SLOTS;
          if (issued >= SLOTS) ok = ca_wait(&empty[slot], ((issued / SLOTS) - 1) & 1, a.status, kStatusTimeoutEmpty);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          const uint32_t dst = ring_addr + slot * G::SLOT;
          const int panel = x % G::PANELS;
          // Unrolled, so that the copies' operands reach uniform registers
          // side by side (in a loop a copy took 170 cycles).
          if (leader) {
#pragma unroll
            for (int u = 0; u < BLOCK / 16; ++u) {
              if (u < units) ca_tma(dst + (u << a.log2_unit) * 128, x < G::PANELS ? &kmap : &vmap, at[u], panel, &full[slot]);
            }
          }
          if (rest > 0) {
            const uint4* base = reinterpret_cast<const uint4*>(x < G::PANELS ? a.keys : a.values) + panel * 8 + (lane & 7);
            for (int r = lane >> 3; r < rest; r += 4) {
              const bool in = done + r < live && last < a.pool_rows;
              const int key = done + r;
              cp_async16(dst + key * 128 + (((lane & 7) ^ (key & 7)) << 4),
                         base + (in ? static_cast<long long>(last + r) * (D / 8) : 0ll), in);
            }
            cp_async_commit();
            cp_async_wait<0>();
            fence_proxy_async_smem();
            __syncwarp();
          }
          if (leader) mbar_arrive_expect_tx(&full[slot], static_cast<uint32_t>(done) * 128);
          ++issued;
        }
      }
    } while (ok && w.next(a));
    // Copies in flight land before the CTA ends.
    if (!ok && lane == 0) {
      for (int i = max(0, issued - SLOTS); i < issued; ++i) mbar_wait(&full[i % SLOTS], (i / SLOTS) & 1, nullptr, 0);
    }
  } else if (warp == 5) {
    // --- Loads row by row ----------------------------------------------------
    constexpr int LOOK = BLOCK / 32;  // lane l looks up keys l, l + 32, ... of a block
    int issued = 0;                   // slots (the panels of a block's K, of its V, ...) issued
    bool ok = true;
    // Signals the slot issued LAG calls ago.
    auto signal = [&](int i) {
      cp_async_wait<G::LAG>();
      fence_proxy_async_smem();
      __syncwarp();
      if (i >= 0 && lane == 0) mbar_arrive(&full[i % SLOTS]);
    };
    const uint32_t ring_addr = smem_addr(ring);
    do {
      const int cnt = w.count();
      const int key_end = w.key_end(a), off = w.off();
      const int32_t* table = a.tables + static_cast<size_t>(w.b) * a.max_pages;
      const long long head = w.h * a.head_stride;
      auto page_of = [&](int key) {
        return a.page_size == 1 ? key : static_cast<int>(__umulhi(static_cast<unsigned>(key), a.page_mul) >> a.page_shift);
      };
      // A block's pages are looked up one block ahead, and used only when its
      // turn comes, so that the look-up is not waited for.
      int page[LOOK];
      auto look = [&](int j) {
#pragma unroll
        for (int i = 0; i < LOOK; ++i) {
          const int key = j * BLOCK + i * 32 + lane;
          page[i] = key < key_end ? __ldg(table + page_of(key)) : -1;
        }
      };
      if (cnt > 0) look(off);
      for (int j = off; j < off + cnt && ok; ++j) {
        uint32_t row[LOOK];  // cache rows of this lane's keys, in 16-byte units; ~0u: zeros
#pragma unroll
        for (int i = 0; i < LOOK; ++i) {
          const int key = j * BLOCK + i * 32 + lane;
          const bool in = page[i] >= 0 && page[i] < a.pool_pages;
          if (!in && key < key_end) atomicOr(a.status, kStatusBadPage);
          const long long slot = key - page_of(key) * a.page_size;
          row[i] = in ? static_cast<uint32_t>((page[i] * a.page_stride + head + slot * D) >> 3) : 0xffffffffu;
        }
        if (j + 1 < off + cnt) look(j + 1);
#pragma unroll 1
        for (int x = 0; x < 2 * G::PANELS; ++x) {  // K's panels, then V's
          const int slot = issued % SLOTS;
          if (issued >= SLOTS) ok = ca_wait(&empty[slot], ((issued / SLOTS) - 1) & 1, a.status, kStatusTimeoutEmpty);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          // Lane l copies piece l % 8 of the rows l / 8, l / 8 + 4, ...
          const uint4* base = reinterpret_cast<const uint4*>(x < G::PANELS ? a.keys : a.values) + x % G::PANELS * 8 + (lane & 7);
          const uint32_t dst = ring_addr + slot * G::SLOT + (lane >> 3) * 128;
#pragma unroll
          for (int i = 0; i < BLOCK / 4; ++i) {
            const uint32_t at = __shfl_sync(0xffffffffu, row[i / 8], (lane >> 3) + 4 * (i % 8));
            const bool live = at != 0xffffffffu;
            // Row r's pieces are rotated by r % 8 = lane / 8 + 4 (i % 2).
            cp_async16(dst + i * 512 + (((lane & 7) ^ ((lane >> 3) + 4 * (i & 1))) << 4), base + (live ? at : 0u), live);
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
    // The whole warp walks and waits; one elected lane issues. Addresses come
    // from warp-uniform values, so that they live in uniform registers, which
    // the MMA takes them from (moved there from a single lane's registers, an
    // issue took 125 cycles; so, 40).
    const bool leader = elect_one();
    constexpr uint32_t idesc_s = ca_idesc(BLOCK);
    constexpr uint32_t idesc_pv = ca_idesc(D) | (1u << 16);  // V MN-major
    const uint32_t base = __shfl_sync(0xffffffffu, tmem, 0);
    const uint32_t ring_addr = __shfl_sync(0xffffffffu, smem_addr(ring), 0);
    const uint64_t qdesc = tc_desc_sw128(__shfl_sync(0xffffffffu, smem_addr(qs), 0));
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      const bool done = __all_sync(0xffffffffu, ca_wait(bar, parity, a.status, kStatusTimeoutFull));
      tc_fence_after();
      return done;
    };
    uint32_t slot = 0, phase = 0, g = 0;  // ring slot and its phase; blocks so far
    auto step = [&] {
      if (++slot == SLOTS) {
        slot = 0;
        phase ^= 1u;
      }
    };
    uint32_t tile = 0;
    bool ok = true;
    do {
      const int cnt = w.count(), off = w.off(), key_end = w.key_end(a);
      if (cnt == 0) continue;
      auto panels = [&] {  // the next K's or V's first slot, once it has landed
        const uint32_t first = slot;
#pragma unroll
        for (int p = 0; p < G::PANELS; ++p) {
          ok = ok && wait(&full[slot], phase);
          step();
        }
        return first;
      };
      // S goes over the P of the block before: its P V is waited for.
      auto issue_s = [&](uint32_t k0) {
        if (g > 0) ok = ok && wait(pv_done, (g - 1) & 1);
        if (!ok) return;
        const uint64_t kdesc = tc_desc_sw128(ring_addr + k0 * G::SLOT);
        if (leader) {
#pragma unroll
          for (int p = 0; p < G::PANELS; ++p) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              tc_mma(base, qdesc + p * (kCaRows * 128 / 16) + 2 * k, kdesc + p * (G::SLOT / 16) + 2 * k, idesc_s,
                     p + k > 0 ? 1u : 0u);
            }
          }
          tc_commit(s_full);
#pragma unroll
          for (int p = 0; p < G::PANELS; ++p) tc_commit(&empty[k0 + p]);
        }
      };
      ok = wait(q_full, tile & 1);
      const uint32_t first = panels();
      issue_s(first);
      for (int j = 0; j < cnt && ok; ++j) {
        const bool more = j + 1 < cnt;
        const uint32_t v0 = panels();
        ok = ok && wait(p_full, g & 1);
        if (!ok) break;
        const uint64_t vdesc = ca_vdesc(ring_addr + v0 * G::SLOT, G::SLOT);
        if (leader) {
#pragma unroll
          for (int k = 0; k < BLOCK / 16; ++k) {
            // (Keys that no row sees weigh nothing.)
            if (k == 0 || (off + j) * BLOCK + 16 * k < key_end) {
              tc_mma_ts(base + G::O_COL, base + k * 8u, vdesc + k * 2048 / 16, idesc_pv, j + k > 0 ? 1u : 0u);
            }
          }
          tc_commit(pv_done);  // first what the chain waits for
#pragma unroll
          for (int p = 0; p < G::PANELS; ++p) tc_commit(&empty[v0 + p]);
        }
        ++g;
        if (more) {
          // (Not before P V: the next K may come late, and its copies may need
          // V's slots.)
          const uint32_t k0 = panels();
          issue_s(k0);
        }
      }
      ++tile;
    } while (ok && w.next(a));
    if (leader) {
      if (!ok) atomicOr(a.status, kStatusAbort);
      tc_commit(drain);
    }
    mbar_wait(drain, 0, nullptr, 0);  // the MMAs in flight land even after an abort
  } else {
    // --- Softmax and epilogue: thread = pair r of the tile = TMEM lane --------
    const int r = tid;
    const int row_r = r / a.group, head_r = r - row_r * a.group;
    const uint32_t trow = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    int g = 0;
    bool ok = true;
    uint32_t parts = 0;  // parts stored so far
    int done = lo;       // units before this segment
    do {
      const int cnt = w.count(), off = w.off();
      if (cnt == 0) {
        done += w.units();
        continue;
      }
      const int row0 = w.t << a.log2_qb;  // of the request
      const int pairs = min(1 << a.log2_qb, w.q.n - row0) * a.group;
      const bool live = r < pairs;
      const int row = row0 + row_r;
      const long long head = static_cast<long long>(w.h * a.group + head_r) * D;
      // Every S of the tile before has landed (its last block's was waited for).
      {
        const uint4* src = reinterpret_cast<const uint4*>(a.q + (live ? (w.q.row0 + row) * a.q_stride + head : 0));
#pragma unroll 1
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
      const int low = w.q.kv - w.q.n + row0;  // blocks that end at or below it need no mask
      // A warp without a live pair (a decoding request fills the first warp at
      // most) only keeps the barriers going. Sharing such a tile's keys out over
      // all four warps, with copies of Q in their lanes, shortened the chain by
      // a fifth but was slower: 71 us instead of 65 for 64 requests of 1 - 5
      // rows on 128 - 4096 keys (heads of 64), the extra warps in the way of
      // the other CTAs' and four copies of O to join.
      const bool idle = !__any_sync(0xffffffffu, live);
      float m = kNegBig, l = 0.f;
      for (int j = 0; j < cnt; ++j, ++g) {
        // S of this block, and with it P V of the block before, have landed.
        ok = __all_sync(0xffffffffu, ca_wait(s_full, g & 1, a.status, kStatusTimeoutFull));
        if (!ok) break;
        tc_fence_after();
        if (idle) {
          if (lane == 0) mbar_arrive(p_full);
          continue;
        }
        const int lim = pos - (off + j) * BLOCK;  // keys of the block past it are masked
        const bool masked = (off + j + 1) * BLOCK - 1 > low;
        float top = -INFINITY;
#pragma unroll 1
        for (int c = 0; c < BLOCK; c += 32) {
          float v[32];
          ca_fetch(trow + c, v, masked, lim - c);
          top = ca_most(v, top);
        }
        top *= a.scale_log2;
        const bool grow = top > m + 8.0f;  // false for a row with no key yet: m stays at its lowest
        const float na = grow ? top : m;
        if (__any_sync(0xffffffffu, grow)) {
          const float alpha = ex2_approx(m - na);
          l *= alpha;
          if (j > 0) {
#pragma unroll 1
            for (int x = 0; x < D; x += 16) {
              float o16[16];
              tc_ld16(trow + G::O_COL + x, o16);
              tc_wait_ld();
#pragma unroll
              for (int y = 0; y < 16; ++y) o16[y] *= alpha;
              tc_st16(trow + G::O_COL + x, o16);
            }
          }
          m = na;
        }
        uint64_t sums[2] = {0, 0};
        const uint64_t scale2 = pair(a.scale_log2, a.scale_log2), shift2 = pair(-m, -m);
#pragma unroll 1
        for (int c = 0; c < BLOCK; c += 32) {
          float v[32];
          uint32_t pk[16];
          ca_fetch(trow + c, v, masked, lim - c);
          ca_weigh(v, scale2, shift2, sums, pk);
          tc_st16u(trow + c / 2, pk);  // over scores that have been read
        }
        const float2 sum = unpair(add2(sums[0], sums[1]));
        l += sum.x + sum.y;
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full);
      }
      if (!ok) break;
      ok = __all_sync(0xffffffffu, ca_wait(pv_done, (g - 1) & 1, a.status, kStatusTimeoutFull));
      if (!ok) break;
      tc_fence_after();
      if (cnt == w.len) {
        const float inv = ca_inverse(l);
        bf16* dst = a.out + (live ? (w.q.row0 + row) * a.out_stride + head : 0);
#pragma unroll 1
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
        // A part: columns of four as [column / 4][lane], so neighbouring
        // threads' 16 bytes are neighbours.
        float* part = a.partials + static_cast<size_t>(2 * c + (off > 0 ? 0 : 1)) * ca_part_floats(D);
        if (live) {
          part[r] = m;
          part[kCaRows + r] = l;
        }
        float4* p4 = reinterpret_cast<float4*>(part + 2 * kCaRows) + r;
#pragma unroll 1
        for (int x = 0; x < D; x += 16) {
          float o[16];
          tc_ld16(trow + G::O_COL + x, o);
          tc_wait_ld();
          if (live) {
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              p4[(x / 4 + y) * kCaRows] = make_float4(o[4 * y], o[4 * y + 1], o[4 * y + 2], o[4 * y + 3]);
            }
          }
        }
        // The ranges of the tile's first and last block.
        const int tile0 = done - w.at, units = w.len + COST;
        const int c0 = ca_owner(tile0 + COST, tile0, units, per, ca_reach<BLOCK>()),
                  c1 = ca_owner(tile0 + units - 1, tile0, units, per, ca_reach<BLOCK>());
        __syncwarp();
        if (lane == 0) mbar_arrive(stored);
        ok = __all_sync(0xffffffffu, ca_wait(stored, parts & 1, a.status, kStatusTimeoutFull));
        if (!ok) break;
        if (tid == 0) {
          __threadfence();  // what the CTA's threads stored before they met, too
          const bool last = atomicAdd(&a.counters[c0], 1u) == static_cast<unsigned>(c1 - c0);
          if (last) a.counters[c0] = 0u;
          *last_s = last;
          __threadfence();
          mbar_arrive(counted);
        }
        ok = __all_sync(0xffffffffu, ca_wait(counted, parts & 1, a.status, kStatusTimeoutFull));
        if (!ok) break;
        ++parts;
        if (*last_s) {
          ca_join<D>(a, c0, c1, pairs, a.out + (w.q.row0 + row0) * a.out_stride + w.h * a.group * D, tid);
        }
      }
      tc_fence_before();  // O and S were read: the next tile's MMAs may write them
      done += w.units();
    } while (w.next(a));
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 4) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(G::TMEM) : "memory");
  }
}

}  // namespace lcrb
