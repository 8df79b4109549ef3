// C entry points of the ragged step over a paged cache (include/lcr_b200.h):
// argument checks and launches.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "chunk_attn.cuh"
#include "common.cuh"
#include "lcr_b200.h"
#include "qk_norm_rope.cuh"
#include "step_plan.cuh"
#include "tmap.h"
#include "token_probs.cuh"
#include "verify_drafts.cuh"

using namespace lcrb;

namespace {

cudaStream_t cs(lcr_stream_t s) { return reinterpret_cast<cudaStream_t>(s); }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// What lcr_qk_norm_rope_kv and lcr_chunk_attention ask of a cache.
int check_view(const char* what, const lcr_kv_view* v, int pool_pages) {
  LCRB_REQUIRE(v && v->keys && v->values, LCR_ERR_INVALID, "%s: null cache", what);
  LCRB_REQUIRE(v->page_size > 0 && v->num_kv_heads > 0 && pool_pages > 0, LCR_ERR_INVALID,
               "%s: page size %d, %d KV heads, %d pool pages", what, v->page_size, v->num_kv_heads, pool_pages);
  LCRB_REQUIRE(v->head_dim == 64 || v->head_dim == 128, LCR_ERR_SHAPE, "%s is compiled for head_dim 64 or 128, got %d",
               what, v->head_dim);
  LCRB_REQUIRE(v->page_stride > 0 && v->head_stride > 0 && v->page_stride % 8 == 0 && v->head_stride % 8 == 0 &&
                   aligned16(v->keys) && aligned16(v->values),
               LCR_ERR_SHAPE, "%s needs 16-byte aligned cache rows (strides %d, %d)", what, v->page_stride,
               v->head_stride);
  LCRB_REQUIRE(static_cast<long long>(pool_pages) * v->page_size <= INT32_MAX, LCR_ERR_SHAPE,
               "%s: a pool of %d pages of %d positions passes 31 bits", what, pool_pages, v->page_size);
  return LCR_OK;
}

// Division of a number below 2^31 by the page size: with 2^s >= page_size, mul =
// ceil(2^(31 + s) / page_size) is exact.
void page_division(int page_size, unsigned* mul, unsigned* shift) {
  int s = 0;
  while ((1ll << s) < page_size) ++s;
  if (s == 0) return;
  *shift = static_cast<unsigned>(s - 1);
  *mul = static_cast<unsigned>(((1ull << (31 + s)) + page_size - 1) / page_size);
}

// Of the current device.
int multiprocessors() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
    cudaGetLastError();
    return 148;
  }
  return sms;
}

// A launch in clusters of `ctas` CTAs along x.
template <class Args>
int launch_cluster(void (*kernel)(Args), int grid, int ctas, int threads, size_t smem, cudaStream_t s, const Args& args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(ctas);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args);
  return e == cudaSuccess ? LCR_OK : fail(LCR_ERR_CUDA, "kernel launch: %s", cudaGetErrorString(e));
}

// CTAs of the chunk attention on the current device; the workspace holds a
// status word, a counter for each, and two parts for each.
int attention_ctas(int head_dim) { return (head_dim == 64 ? CaGeom<64>::CTAS : CaGeom<128>::CTAS) * multiprocessors(); }
size_t attention_header(size_t ctas) { return 256 + (ctas * sizeof(unsigned) + 255) / 256 * 256; }

template <int D, bool TMA>
int launch_chunk_attention(const ChunkAttnArgs& a, const CUtensorMap& kmap, const CUtensorMap& vmap, int grid,
                           cudaStream_t s) {
  constexpr size_t smem = CaGeom<D>::SMEM;
  auto kernel = chunk_attn_kernel<D, TMA>;
  LCRB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
  return launch_kernel(kernel, dim3(static_cast<unsigned>(grid)), dim3(kCaThreads), smem, s, false, a, kmap, vmap);
}

template <int D>
int chunk_attention(ChunkAttnArgs& a, int grid, cudaStream_t s) {
  CUtensorMap kmap = {}, vmap = {};
  const long long rows = static_cast<long long>(a.pool_pages) * a.kv_heads * a.page_size;
  // Tensor copies see a pool as rows of head_dim, and a copy lies within a page.
  const bool dense = a.head_stride == static_cast<long long>(a.page_size) * D && a.page_stride == a.kv_heads * a.head_stride;
  if (dense && a.page_size % 16 == 0 && rows < INT32_MAX) {
    a.log2_unit = 4;
    while ((2 << a.log2_unit) <= CaGeom<D>::BLOCK && a.page_size % (2 << a.log2_unit) == 0) ++a.log2_unit;
    a.pool_rows = static_cast<int>(rows);
    LCRB_TRY(make_kmajor_map(&kmap, a.keys, a.pool_rows, D, 1, 1 << a.log2_unit, 1));
    LCRB_TRY(make_kmajor_map(&vmap, a.values, a.pool_rows, D, 1, 1 << a.log2_unit, 1));
    return launch_chunk_attention<D, true>(a, kmap, vmap, grid, s);
  }
  return launch_chunk_attention<D, false>(a, kmap, vmap, grid, s);
}

}  // namespace

extern "C" int lcr_plan_step(int32_t* block_tables, int max_pages, const int32_t* held, int32_t* held_out,
                             int32_t* free_pages, const int32_t* free_count, int32_t* free_count_out, int pool_pages,
                             const int32_t* cached, const int32_t* new_tokens, const int32_t* finished, int sequences,
                             int page_size, int max_rows, int32_t* row_starts, int32_t* kv_lengths,
                             int32_t* positions, int32_t* slots, int32_t* row_sequence, lcr_stream_t stream) {
  LCRB_REQUIRE(sequences > 0 && max_pages > 0 && pool_pages > 0 && page_size > 0 && max_rows >= 0, LCR_ERR_INVALID,
               "plan_step: %d requests, %d pages each, pool of %d pages of %d, %d rows", sequences, max_pages,
               pool_pages, page_size, max_rows);
  LCRB_REQUIRE(block_tables && held && held_out && free_pages && free_count && free_count_out && cached && new_tokens &&
                   row_starts && kv_lengths && (max_rows == 0 || (positions && slots && row_sequence)),
               LCR_ERR_INVALID, "plan_step: null pointer");
  LCRB_REQUIRE(sequences <= LCR_PLAN_MAX_SEQUENCES, LCR_ERR_SHAPE, "plan_step: %d requests; at most %d", sequences,
               LCR_PLAN_MAX_SEQUENCES);
  LCRB_REQUIRE(static_cast<long long>(sequences) * max_pages <= INT32_MAX &&
                   static_cast<long long>(max_pages) * page_size <= INT32_MAX &&
                   static_cast<long long>(pool_pages) * page_size <= INT32_MAX,
               LCR_ERR_SHAPE, "plan_step: tables or pool pass 31 bits");
  StepPlanArgs a = {};
  a.tables = block_tables;
  a.max_pages = max_pages;
  a.held = held;
  a.held_out = held_out;
  a.free_pages = free_pages;
  a.free_count = free_count;
  a.free_count_out = free_count_out;
  a.pool_pages = pool_pages;
  a.cached = cached;
  a.new_tokens = new_tokens;
  a.finished = finished;
  a.sequences = sequences;
  a.page_size = static_cast<uint32_t>(page_size);
  page_division(page_size, &a.page_mul, &a.page_shift);
  a.max_rows = max_rows;
  a.row_starts = row_starts;
  a.kv_lengths = kv_lengths;
  a.positions = positions;
  a.slots = slots;
  a.row_sequence = row_sequence;
  // The limit is the kernel's, not the launch's: always the largest call's, as
  // other threads may be planning.
  constexpr int kPerSequence = 5 * sizeof(int32_t);
  const size_t smem = kPerSequence * static_cast<size_t>(sequences);
  LCRB_CUDA(cudaFuncSetAttribute(step_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 kPerSequence * LCR_PLAN_MAX_SEQUENCES));
  return launch_kernel(step_plan_kernel, dim3(kPlanCtas), dim3(kPlanThreads), smem, cs(stream), false, a);
}

extern "C" int lcr_qk_norm_rope_kv(void* q_out, int64_t q_stride, const lcr_kv_view* view, int pool_pages,
                                   const void* qkv, int64_t qkv_stride, int rows, int num_heads, const void* q_gain,
                                   const void* k_gain, float eps, const float* inv_freq, const int32_t* positions,
                                   const int32_t* slots, lcr_stream_t stream) {
  if (rows == 0) return LCR_OK;
  LCRB_REQUIRE(q_out && qkv && inv_freq && positions && slots && rows > 0 && num_heads > 0 && eps >= 0.f,
               LCR_ERR_INVALID, "qk_norm_rope_kv: null pointer or bad size");
  LCRB_TRY(check_view("qk_norm_rope_kv", view, pool_pages));
  const int64_t width = static_cast<int64_t>(num_heads + 2 * view->num_kv_heads) * view->head_dim;
  LCRB_REQUIRE(qkv_stride >= width && q_stride >= static_cast<int64_t>(num_heads) * view->head_dim, LCR_ERR_INVALID,
               "qk_norm_rope_kv: row strides %lld (of %lld elements) and %lld", static_cast<long long>(qkv_stride),
               static_cast<long long>(width), static_cast<long long>(q_stride));
  LCRB_REQUIRE(qkv_stride % 8 == 0 && q_stride % 8 == 0 && aligned16(qkv) && aligned16(q_out) && aligned16(q_gain) &&
                   aligned16(k_gain),
               LCR_ERR_SHAPE, "qk_norm_rope_kv needs 16-byte aligned rows and gains");
  QkNormRopeArgs a = {};
  a.q_out = static_cast<bf16*>(q_out);
  a.q_stride = q_stride;
  a.keys = static_cast<bf16*>(view->keys);
  a.values = static_cast<bf16*>(view->values);
  a.page_stride = view->page_stride;
  a.head_stride = view->head_stride;
  a.page_size = view->page_size;
  a.pool_pages = pool_pages;
  a.qkv = static_cast<const bf16*>(qkv);
  a.qkv_stride = qkv_stride;
  a.rows = rows;
  a.heads = num_heads;
  a.kv_heads = view->num_kv_heads;
  a.q_gain = static_cast<const bf16*>(q_gain);
  a.k_gain = static_cast<const bf16*>(k_gain);
  a.eps = eps;
  a.inv_freq = inv_freq;
  a.positions = positions;
  a.slots = slots;
  auto kernel = view->head_dim == 64 ? qk_norm_rope_kernel<64> : qk_norm_rope_kernel<128>;
  return launch_kernel(kernel, dim3(static_cast<unsigned>(std::min(rows, kQkCtas * multiprocessors()))), dim3(kQkThreads), 0,
                       cs(stream), false, a);
}

extern "C" size_t lcr_chunk_attention_scratch_bytes(int num_heads, int head_dim) {
  (void)num_heads;
  const size_t ctas = static_cast<size_t>(attention_ctas(head_dim));
  return attention_header(ctas) + 2 * ctas * ca_part_floats(std::max(64, head_dim)) * sizeof(float);
}

extern "C" int lcr_chunk_attention(void* out, int64_t out_stride, const void* q, int64_t q_stride,
                                   const lcr_kv_view* view, int max_pages, int pool_pages, const int32_t* row_starts,
                                   const int32_t* kv_lengths, int sequences, int rows, int num_heads, float scale,
                                   void* scratch, size_t scratch_bytes, lcr_stream_t stream) {
  if (rows == 0 || sequences == 0) return LCR_OK;
  LCRB_REQUIRE(out && q && row_starts && kv_lengths && scratch && sequences > 0 && rows > 0 && num_heads > 0 &&
                   max_pages > 0,
               LCR_ERR_INVALID, "chunk_attention: null pointer or bad size");
  LCRB_TRY(check_view("chunk_attention", view, pool_pages));
  LCRB_REQUIRE(view->page_table != nullptr, LCR_ERR_INVALID, "chunk_attention: no page tables");
  LCRB_REQUIRE(num_heads % view->num_kv_heads == 0 && num_heads / view->num_kv_heads <= 128, LCR_ERR_SHAPE,
               "chunk_attention: %d query heads on %d KV heads", num_heads, view->num_kv_heads);
  const int64_t width = static_cast<int64_t>(num_heads) * view->head_dim;
  LCRB_REQUIRE(q_stride >= width && out_stride >= width, LCR_ERR_INVALID,
               "chunk_attention: row strides %lld and %lld of %lld elements", static_cast<long long>(q_stride),
               static_cast<long long>(out_stride), static_cast<long long>(width));
  LCRB_REQUIRE(q_stride % 8 == 0 && out_stride % 8 == 0 && aligned16(q) && aligned16(out) && aligned16(scratch),
               LCR_ERR_SHAPE, "chunk_attention needs 16-byte aligned rows and scratch");
  LCRB_REQUIRE(scale > 0.f && std::isfinite(scale), LCR_ERR_INVALID, "chunk_attention: scale %g must be positive",
               static_cast<double>(scale));
  LCRB_REQUIRE(static_cast<double>(pool_pages) * view->page_stride + static_cast<double>(view->num_kv_heads) * view->head_stride <
                   34359738368.0,
               LCR_ERR_SHAPE, "chunk_attention: a pool of more than 2^35 elements");
  LCRB_REQUIRE(static_cast<long long>(max_pages) * view->page_size <= INT32_MAX, LCR_ERR_SHAPE,
               "chunk_attention: tables of %d pages of %d positions pass 31 bits", max_pages, view->page_size);
  LCRB_REQUIRE(scratch_bytes >= lcr_chunk_attention_scratch_bytes(num_heads, view->head_dim), LCR_ERR_INVALID,
               "chunk_attention: %zu bytes of scratch; it needs %zu", scratch_bytes,
               lcr_chunk_attention_scratch_bytes(num_heads, view->head_dim));
  ChunkAttnArgs a = {};
  a.out = static_cast<bf16*>(out);
  a.out_stride = out_stride;
  a.q = static_cast<const bf16*>(q);
  a.q_stride = q_stride;
  a.keys = static_cast<const bf16*>(view->keys);
  a.values = static_cast<const bf16*>(view->values);
  a.tables = view->page_table;
  a.max_pages = max_pages;
  a.pool_pages = pool_pages;
  a.page_size = view->page_size;
  a.page_stride = view->page_stride;
  a.head_stride = view->head_stride;
  a.row_starts = row_starts;
  a.kv_lengths = kv_lengths;
  a.sequences = sequences;
  a.rows = rows;
  a.kv_heads = view->num_kv_heads;
  a.group = num_heads / view->num_kv_heads;
  a.scale_log2 = scale * kLog2e;
  a.log2_qb = 7;
  while (a.log2_qb > 0 && (a.group << a.log2_qb) > kCaRows) --a.log2_qb;
  page_division(view->page_size, &a.page_mul, &a.page_shift);
  const int ctas = attention_ctas(view->head_dim);
  char* work = static_cast<char*>(scratch);
  a.status = reinterpret_cast<uint32_t*>(work);
  a.counters = reinterpret_cast<unsigned*>(work + 256);
  a.partials = reinterpret_cast<float*>(work + attention_header(static_cast<size_t>(ctas)));
  // As many CTAs as the tables' capacity could give ranges.
  const double tiles = a.kv_heads * (std::ldexp(static_cast<double>(rows), -a.log2_qb) + sequences);
  const double blocks = tiles * ((static_cast<double>(max_pages) * view->page_size + rows) / view->head_dim + 1 + ca_tile_cost<64>());
  LCRB_REQUIRE(blocks < 2147483647.0, LCR_ERR_SHAPE,
               "chunk_attention: %d rows of %d requests over tables of %d positions are too many blocks", rows, sequences,
               max_pages * view->page_size);
  const int grid = static_cast<int>(std::min(static_cast<double>(ctas), std::max(1.0, blocks / ca_min_range<128>())));
  return view->head_dim == 64 ? chunk_attention<64>(a, grid, cs(stream)) : chunk_attention<128>(a, grid, cs(stream));
}

extern "C" int lcr_chunk_attention_status(void* scratch, lcr_stream_t stream) {
  LCRB_REQUIRE(scratch, LCR_ERR_INVALID, "chunk_attention_status: null scratch");
  uint32_t st = 0;
  LCRB_CUDA(cudaMemcpyAsync(&st, scratch, sizeof st, cudaMemcpyDeviceToHost, cs(stream)));
  LCRB_CUDA(cudaStreamSynchronize(cs(stream)));
  if (st == 0) return LCR_OK;
  // A call that gave up may have left its counters up.
  LCRB_CUDA(cudaMemsetAsync(scratch, 0, attention_header(static_cast<size_t>(attention_ctas(64))), cs(stream)));
  LCRB_CUDA(cudaStreamSynchronize(cs(stream)));
  if (st & kStatusBadPage) return fail(LCR_ERR_POOL, "page table entry outside the pool (status 0x%x)", st);
  return fail(LCR_ERR_TIMEOUT, "a device-side wait gave up (status 0x%x)", st);
}

extern "C" int lcr_token_probs(float* probs, int64_t probs_stride, const float* logits, int64_t logits_stride, int rows,
                               int vocab, const float* temperature, int temperatures, const int32_t* row_sequence,
                               lcr_stream_t stream) {
  if (rows == 0) return LCR_OK;
  LCRB_REQUIRE(probs && logits && rows > 0 && vocab > 0, LCR_ERR_INVALID, "token_probs: null pointer or bad size");
  LCRB_REQUIRE(probs_stride >= vocab && logits_stride >= vocab, LCR_ERR_INVALID,
               "token_probs: row strides %lld and %lld of %d ids", static_cast<long long>(probs_stride),
               static_cast<long long>(logits_stride), vocab);
  LCRB_REQUIRE(temperature == nullptr || temperatures >= (row_sequence != nullptr ? 1 : rows), LCR_ERR_INVALID,
               "token_probs: %d temperatures of %d rows", temperatures, rows);
  TokenProbsArgs a = {probs, probs_stride, logits, logits_stride, rows, vocab, temperature, temperatures, row_sequence, 0};
  // CTAs for a row: enough to keep it in shared memory, and for few rows as many
  // as fill the GPU (one row of 32000 ids: 3.8 us with 8, 5.4 with the 2 it takes
  // to keep it; 16 rows 4.9 and 5.6; 64 rows the same).
  int ctas = 1;
  while (ctas < kProbsMaxCtas && (vocab > ctas * kProbsSlice || (rows * ctas < 256 && vocab > ctas * 2048))) ctas *= 2;
  LCRB_REQUIRE(rows <= INT32_MAX / ctas, LCR_ERR_SHAPE, "token_probs: %d rows", rows);
  a.slice = ((vocab + ctas - 1) / ctas + 3) / 4 * 4;
  const bool vec = aligned16(probs) && aligned16(logits) && probs_stride % 4 == 0 && logits_stride % 4 == 0;
  const auto kernel = vec ? token_probs_kernel<true> : token_probs_kernel<false>;
  LCRB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kProbsSlice * 4));
  return launch_cluster(kernel, rows * ctas, ctas, kProbsThreads, sizeof(float) * std::min(a.slice, kProbsSlice), cs(stream), a);
}

extern "C" int lcr_verify_drafts_bounded(int32_t* tokens, int32_t* accepted, const float* target_probs,
                                         int64_t target_stride, int target_rows, const int32_t* target_starts,
                                         const int32_t* drafts, const int32_t* draft_counts, const float* draft_probs,
                                         const float* uniforms, int sequences, int max_drafts, int vocab,
                                         lcr_stream_t stream) {
  if (sequences == 0) return LCR_OK;
  LCRB_REQUIRE(tokens && accepted && target_probs && target_starts && draft_counts && uniforms && sequences > 0 &&
                   target_rows >= 0 && max_drafts >= 0 && vocab > 0 && (max_drafts == 0 || drafts),
               LCR_ERR_INVALID, "verify_drafts: null pointer or bad size");
  LCRB_REQUIRE(target_stride >= vocab, LCR_ERR_INVALID, "verify_drafts: row stride %lld of %d ids",
               static_cast<long long>(target_stride), vocab);
  VerifyArgs a = {tokens,       accepted,    target_probs, target_stride, target_rows, target_starts, drafts,
                  draft_counts, draft_probs, uniforms,     sequences,     max_drafts,  vocab};
  // CTAs for a request: as many as run at once (two on an SM) for all of them
  // (64 requests of 128256 ids: 41, 25, 19.5 and 23 us with 1, 2, 4 and 8).
  const int sms = multiprocessors();
  int ctas = 1;
  while (ctas < kVerifyMaxCtas && static_cast<long long>(sequences) * ctas <= sms) ctas *= 2;
  return launch_cluster(verify_drafts_kernel, sequences * ctas, ctas, kVerifyThreads, 0, cs(stream), a);
}

extern "C" int lcr_verify_drafts(int32_t* tokens, int32_t* accepted, const float* target_probs, int64_t target_stride,
                                 const int32_t* target_starts, const int32_t* drafts, const int32_t* draft_counts,
                                 const float* draft_probs, const float* uniforms, int sequences, int max_drafts,
                                 int vocab, lcr_stream_t stream) {
  return lcr_verify_drafts_bounded(tokens, accepted, target_probs, target_stride, INT32_MAX, target_starts, drafts,
                                   draft_counts, draft_probs, uniforms, sequences, max_drafts, vocab, stream);
}
