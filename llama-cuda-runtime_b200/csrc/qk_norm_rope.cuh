// Per-head RMSNorm of q and k, rotary positions and the paged cache write in
// one pass over the projection's rows (lcr_qk_norm_rope_kv).
//
// Per head x of D elements: y = x * rsqrt(mean(x^2) + eps) * gain, then for
// i < D/2 with angle t = position * inv_freq[i]
//   out[i]       = y[i] cos t - y[i + D/2] sin t
//   out[i + D/2] = y[i + D/2] cos t + y[i] sin t
// in fp32, rounded to bf16 once. The angle is formed as a rounded product
// plus its error e (one fma), and the pair (cos, sin) is turned by that error
// to second order: at position 32768 the plain fp32 product is off by up to
// 1e-3, which would show in bf16, and at 2^20 by 2^-5. The rest, e^3 / 6, is
// below 1e-5 up to angles of 2^20 (the first order alone: 5e-4 there); positions
// are whole in fp32 up to 2^24.
#pragma once

#include "common.cuh"

namespace lcrb {

struct QkNormRopeArgs {
  bf16* q_out;
  long long q_stride;
  bf16* keys;
  bf16* values;
  long long page_stride, head_stride;
  int page_size, pool_pages;
  const bf16* qkv;
  long long qkv_stride;
  int rows, heads, kv_heads;
  const bf16* q_gain;
  const bf16* k_gain;
  float eps;
  const float* inv_freq;
  const int32_t* positions;
  const int32_t* slots;
};

__device__ __forceinline__ float2 rope_pair(int position, float inv_freq) {
  const float p = static_cast<float>(position);
  const float t = __fmul_rn(p, inv_freq);
  const float err = fmaf(p, inv_freq, -t);
  float s, c;
  sincosf(t, &s, &c);
  const float half = -0.5f * err * err;
  return make_float2(fmaf(half, c, fmaf(-err, s, c)), fmaf(half, s, fmaf(err, c, s)));
}

// Two bf16 in one conversion.
__device__ __forceinline__ uint32_t qk_pack(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

constexpr int kQkThreads = 192;
constexpr int kQkAhead = 2;  // pieces of a row that a thread holds ahead
constexpr int kQkCtas = 4;   // per SM

// A group of D/16 lanes owns a head: each lane holds 8 elements of its lower
// and 8 of its upper half (a piece), so the rotation needs no exchange and the
// sum of squares log2(D/16) shuffles. HBM bound: every CTA walks over rows and
// loads the next row's pieces (64 bytes a thread), position and slot before it
// works on the present one, so that loads are always in flight; the angles'
// pairs, by head_dim / 2 threads, are double-buffered, with one barrier a row.
// 8192 rows of 32 + 16 heads of 128: 37.0 us for 201 MB, 5.4 TB/s, 0.83 of a
// copy's rate, and 34.1 us without norms (a CTA for each row, without loads
// ahead: 51); 320 rows of heads of 64: 2.7 us, latency.
template <int D>
__global__ void __launch_bounds__(kQkThreads, kQkCtas) qk_norm_rope_kernel(const QkNormRopeArgs a) {
  constexpr int HALF = D / 2;
  constexpr int LANES = D / 16;
  __shared__ float2 cs[2][HALF];
  const int tid = threadIdx.x;
  const int items = (a.heads + 2 * a.kv_heads) * LANES;
  const int piece = (tid % LANES) * 8;
  const float freq = tid < HALF ? a.inv_freq[tid] : 0.f;
  uint4 next[kQkAhead][2];
  int next_pos, next_slot;
  auto fetch = [&](int r, int it, uint4 (&v)[2]) {
    const bf16* src = a.qkv + r * a.qkv_stride + (it < items ? it / LANES : 0) * D + piece;
    v[0] = ldg16(src);
    v[1] = ldg16(src + HALF);
  };
  auto ahead = [&](int r) {
#pragma unroll
    for (int k = 0; k < kQkAhead; ++k) fetch(r, tid + k * kQkThreads, next[k]);
    next_pos = a.positions[r];
    next_slot = a.slots[r];
  };
  ahead(blockIdx.x);
  int buf = 0;
  for (int r = blockIdx.x; r < a.rows; r += gridDim.x, buf ^= 1) {
    uint4 now[kQkAhead][2];
#pragma unroll
    for (int k = 0; k < kQkAhead; ++k) {
      now[k][0] = next[k][0];
      now[k][1] = next[k][1];
    }
    const int slot = next_slot;
    if (tid < HALF) cs[buf][tid] = rope_pair(next_pos, freq);
    if (r + static_cast<int>(gridDim.x) < a.rows) ahead(r + gridDim.x);
    const int page = slot / a.page_size;
    const bool cached = slot >= 0 && page < a.pool_pages;
    const long long at = cached ? page * a.page_stride + static_cast<long long>(slot - page * a.page_size) * D : 0;
    __syncthreads();
    // (Every lane of a group takes part in the shuffles: a group is live or not.)
    auto work = [&](int it, const uint4 (&v)[2]) {
      const bool live = it < items;
      const int h = live ? it / LANES : 0;
      float lo[8], hi[8];
      unpack8(v[0], lo);
      unpack8(v[1], hi);
      const bool is_v = h >= a.heads + a.kv_heads, is_q = h < a.heads;
      const bf16* gain = is_q ? a.q_gain : a.k_gain;
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(lo[e], lo[e], fmaf(hi[e], hi[e], ss));
#pragma unroll
      for (int off = LANES / 2; off >= 1; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
      uint4 wl = v[0], wh = v[1];
      if (!is_v) {
        if (gain != nullptr) {
          const float scale = rsqrtf(ss * (1.0f / D) + a.eps);
          float g[8];
          unpack8(ldg16(gain + piece), g);
#pragma unroll
          for (int e = 0; e < 8; ++e) lo[e] = lo[e] * scale * g[e];
          unpack8(ldg16(gain + HALF + piece), g);
#pragma unroll
          for (int e = 0; e < 8; ++e) hi[e] = hi[e] * scale * g[e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float2 t = cs[buf][piece + e];
          const float x = lo[e], y = hi[e];
          lo[e] = x * t.x - y * t.y;
          hi[e] = y * t.x + x * t.y;
        }
        wl = make_uint4(qk_pack(lo[0], lo[1]), qk_pack(lo[2], lo[3]), qk_pack(lo[4], lo[5]), qk_pack(lo[6], lo[7]));
        wh = make_uint4(qk_pack(hi[0], hi[1]), qk_pack(hi[2], hi[3]), qk_pack(hi[4], hi[5]), qk_pack(hi[6], hi[7]));
      }
      if (!live || (!is_q && !cached)) return;
      bf16* dst = is_q ? a.q_out + r * a.q_stride + h * D
                       : (is_v ? a.values + (h - a.heads - a.kv_heads) * a.head_stride
                               : a.keys + (h - a.heads) * a.head_stride) + at;
      *reinterpret_cast<uint4*>(dst + piece) = wl;
      *reinterpret_cast<uint4*>(dst + piece + HALF) = wh;
    };
#pragma unroll
    for (int k = 0; k < kQkAhead; ++k) {
      if (k * kQkThreads < items) work(tid + k * kQkThreads, now[k]);
    }
    for (int first = kQkAhead * kQkThreads; first < items; first += kQkThreads) {  // wider rows
      uint4 v[2];
      fetch(r, first + tid, v);
      work(first + tid, v);
    }
  }
}

}  // namespace lcrb
