// Per-head RMSNorm of q and k, rotary positions and the paged cache write in
// one pass over the projection's rows (lcr_qk_norm_rope_kv).
//
// Per head x of D elements: y = x * rsqrt(mean(x^2) + eps) * gain, then for
// i < D/2 with angle t = position * inv_freq[i]
//   out[i]       = y[i] cos t - y[i + D/2] sin t
//   out[i + D/2] = y[i + D/2] cos t + y[i] sin t
// in fp32, rounded to bf16 once. The angle is formed as a rounded product
// plus its error (one fma), and the pair (cos, sin) is turned by that error
// to first order: at position 32768 the plain fp32 product is off by up to
// 2e-3, which would show in bf16; the second-order rest is below 1e-5 up to
// position 10^6.
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
  return make_float2(fmaf(-err, s, c), fmaf(err, c, s));
}

// Two bf16 in one conversion.
__device__ __forceinline__ uint32_t qk_pack(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

constexpr int kQkThreads = 192;
constexpr int kQkItems = 2;  // a thread's pieces in flight

// One CTA per row. A group of D/16 lanes owns a head: each lane holds 8
// elements of its lower and 8 of its upper half, so the rotation needs no
// exchange and the sum of squares log2(D/16) shuffles. HBM bound: a thread's
// loads (64 bytes) are issued before the row's angles are formed, and ten CTAs
// share an SM, so that one row's latencies hide under the others' transfers.
template <int D>
__global__ void __launch_bounds__(kQkThreads) qk_norm_rope_kernel(const QkNormRopeArgs a) {
  constexpr int HALF = D / 2;
  constexpr int LANES = D / 16;
  __shared__ float2 cs[HALF];
  const int r = blockIdx.x, tid = threadIdx.x;
  const bf16* row = a.qkv + r * a.qkv_stride;
  const int items = (a.heads + 2 * a.kv_heads) * LANES;
  const int piece = (tid % LANES) * 8;
  uint4 rl[kQkItems], rh[kQkItems];
  auto load = [&](int first) {
#pragma unroll
    for (int k = 0; k < kQkItems; ++k) {
      const int it = first + k * kQkThreads;
      const bf16* src = row + (it < items ? it / LANES : 0) * D + piece;
      rl[k] = ldg16(src);
      rh[k] = ldg16(src + HALF);
    }
  };
  load(tid);
  const int slot = a.slots[r];
  const int page = slot / a.page_size;
  const bool cached = slot >= 0 && page < a.pool_pages;
  const long long at = cached ? page * a.page_stride + static_cast<long long>(slot - page * a.page_size) * D : 0;
  if (tid < HALF) cs[tid] = rope_pair(a.positions[r], a.inv_freq[tid]);
  __syncthreads();
  // Every lane takes part in the shuffles: the loop count is uniform.
  for (int first = tid; first - tid < items; first += kQkItems * kQkThreads) {
    if (first != tid) load(first);
#pragma unroll
    for (int k = 0; k < kQkItems; ++k) {
      const int it = first + k * kQkThreads;
      const bool live = it < items;
      const int h = live ? it / LANES : 0;
      float lo[8], hi[8];
      unpack8(rl[k], lo);
      unpack8(rh[k], hi);
      const bool is_v = h >= a.heads + a.kv_heads, is_q = h < a.heads;
      const bf16* gain = is_q ? a.q_gain : a.k_gain;
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(lo[e], lo[e], fmaf(hi[e], hi[e], ss));
#pragma unroll
      for (int off = LANES / 2; off >= 1; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
      if (!live) continue;
      uint4 wl = rl[k], wh = rh[k];
      if (!is_v) {
        if (gain != nullptr) {
          const float scale = rsqrtf(ss * (1.0f / D) + a.eps);
          float gl[8], gh[8];
          unpack8(ldg16(gain + piece), gl);
          unpack8(ldg16(gain + HALF + piece), gh);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            lo[e] = lo[e] * scale * gl[e];
            hi[e] = hi[e] * scale * gh[e];
          }
        }
        float ol[8], oh[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float2 t = cs[piece + e];
          ol[e] = lo[e] * t.x - hi[e] * t.y;
          oh[e] = hi[e] * t.x + lo[e] * t.y;
        }
        wl = make_uint4(qk_pack(ol[0], ol[1]), qk_pack(ol[2], ol[3]), qk_pack(ol[4], ol[5]), qk_pack(ol[6], ol[7]));
        wh = make_uint4(qk_pack(oh[0], oh[1]), qk_pack(oh[2], oh[3]), qk_pack(oh[4], oh[5]), qk_pack(oh[6], oh[7]));
      }
      bf16* dst;
      if (is_q) {
        dst = a.q_out + r * a.q_stride + h * D + piece;
      } else {
        if (!cached) continue;
        const int kvh = is_v ? h - a.heads - a.kv_heads : h - a.heads;
        dst = (is_v ? a.values : a.keys) + at + kvh * a.head_stride + piece;
      }
      *reinterpret_cast<uint4*>(dst) = wl;
      *reinterpret_cast<uint4*>(dst + HALF) = wh;
    }
  }
}

}  // namespace lcrb
