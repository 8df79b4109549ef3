// Attention of every request's new rows over its paged cache
// (lcr_chunk_attention): row i of the n rows of request b is at position p =
// kv_length - n + i and sees keys 0 .. p.
#pragma once

#include "common.cuh"

namespace lcrb {

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
  float scale_log2;
  uint32_t* status;
};

// One warp per (row, query head), the lanes over the head's dimensions: one
// online-softmax pass over the visible keys.
template <int D>
__global__ void __launch_bounds__(256) chunk_attn_kernel(const ChunkAttnArgs a) {
  constexpr int PER = D / 32;
  const int heads = a.kv_heads * a.group;
  const long long w = (blockIdx.x * 256ll + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (w >= static_cast<long long>(a.rows) * heads) return;
  const int r = static_cast<int>(w / heads), h = static_cast<int>(w % heads), kvh = h / a.group;
  int lo = 0, hi = a.sequences;  // the request that owns row r
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a.row_starts[mid + 1] > r) hi = mid;
    else lo = mid + 1;
  }
  if (lo >= a.sequences || r < a.row_starts[lo]) return;
  const int b = lo, n = a.row_starts[b + 1] - a.row_starts[b];
  const long long cap = static_cast<long long>(a.max_pages) * a.page_size;
  const int kv = static_cast<int>(min(static_cast<long long>(max(0, a.kv_lengths[b])), cap));
  const int p = kv - n + (r - a.row_starts[b]);
  float q[PER], o[PER];
  for (int e = 0; e < PER; ++e) {
    q[e] = bf2f(__bfloat16_as_ushort(a.q[r * a.q_stride + h * D + lane * PER + e]));
    o[e] = 0.f;
  }
  float m = kNegBig, l = 0.f;
  for (int j = 0; j <= p; ++j) {
    const int page = a.tables[static_cast<size_t>(b) * a.max_pages + j / a.page_size];
    const bool ok = page >= 0 && page < a.pool_pages;
    if (!ok && lane == 0) atomicOr(a.status, kStatusBadPage);
    const long long at = ok ? page * a.page_stride + kvh * a.head_stride + static_cast<long long>(j % a.page_size) * D : 0;
    float s = 0.f;
    for (int e = 0; e < PER; ++e) s = fmaf(q[e], ok ? __bfloat162float(a.keys[at + lane * PER + e]) : 0.f, s);
    for (int off = 16; off >= 1; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    s *= a.scale_log2;
    const float mn = fmaxf(m, s), alpha = exp2f(m - mn), x = exp2f(s - mn);
    l = l * alpha + x;
    for (int e = 0; e < PER; ++e) o[e] = fmaf(x, ok ? __bfloat162float(a.values[at + lane * PER + e]) : 0.f, o[e] * alpha);
    m = mn;
  }
  const float inv = l > 0.f ? 1.0f / l : 0.f;
  for (int e = 0; e < PER; ++e) a.out[r * a.out_stride + h * D + lane * PER + e] = __float2bfloat16_rn(o[e] * inv);
}

}  // namespace lcrb
