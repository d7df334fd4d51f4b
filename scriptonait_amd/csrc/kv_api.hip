// C entry points of the paged key-value cache (declared in
// include/llmhip_kv.h): what the host can check, and the launches.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <string.h>

#include "kv_check.h"

using namespace llmhip;

namespace {

int check_cache(const llmhip_kv_cache* c) {
  ARG(c, "cache is null");
  ARG(c->dtype <= LLMHIP_E4M3, "unknown cache dtype");
  ARG(c->k_pool && c->v_pool, "k_pool and v_pool are required");
  ARG((c->dtype == LLMHIP_E4M3) == (c->k_scale != nullptr) && (c->dtype == LLMHIP_E4M3) == (c->v_scale != nullptr),
      "k_scale and v_scale go with an E4M3 cache, and only with one");
  ARG(c->pages >= 1 && c->page >= 1 && c->heads >= 1, "pages, page and heads must be at least 1");
  SUPPORTED(c->pages <= kMaxInt && c->page <= kMaxInt && c->heads <= kMaxHeads, "pages, page or heads too large");
  SUPPORTED(c->head_dim >= 8 && c->head_dim <= kMaxHeadDim && c->head_dim % 8 == 0,
            "head_dim must be a multiple of 8 up to 256");
  for (int i = 0; i < 3; ++i) ARG(c->k_stride[i] >= 0 && c->v_stride[i] >= 0, "pool strides must not be negative");
  const uint32_t elem = size_of(c->dtype), bytes = elem == 1 ? 8 : 16;
  SUPPORTED(rows_on(c->k_pool, c->k_stride, 3, elem, bytes) && rows_on(c->v_pool, c->v_stride, 3, elem, bytes),
            "pool rows must be aligned to 16 bytes (8 for E4M3)");
  return LLMHIP_OK;
}

int check_dtype(const llmhip_kv_cache* c, uint32_t dtype) {
  ARG(dtype <= LLMHIP_F16, "dtype must be F32, BF16 or F16");
  ARG(dtype == c->dtype || c->dtype == LLMHIP_E4M3, "dtype is neither the cache's nor beside an E4M3 cache");
  return LLMHIP_OK;
}

void set_pools(const llmhip_kv_cache* c, const void** pool, const float** scale, int64_t (*stride)[3]) {
  pool[0] = c->k_pool;
  pool[1] = c->v_pool;
  scale[0] = c->k_scale;
  scale[1] = c->v_scale;
  memcpy(stride[0], c->k_stride, sizeof c->k_stride);
  memcpy(stride[1], c->v_stride, sizeof c->v_stride);
}

}  // namespace

extern "C" {

int llmhip_kv_plan(llmhip_ctx* ctx, size_t pages, size_t page, int32_t* ring, const int32_t* free_state, size_t R,
                   const int32_t* lens, const int32_t* new_tokens, const int32_t* release, int32_t* table,
                   size_t table_pages, size_t table_ld, int32_t* out_lens, int32_t* granted, int32_t* start, size_t T,
                   int64_t* slots, int32_t* positions, int32_t* out_free_state, void* stream) {
  ARG(pages >= 1 && page >= 1, "pages and page must be at least 1");
  SUPPORTED(pages <= kMaxInt && page <= kMaxInt, "pages or page too large");
  ARG(ring && free_state && out_free_state, "ring, free_state and out_free_state are required");
  ARG(R == 0 || (lens && out_lens && granted), "lens, out_lens and granted are required");
  ARG(R == 0 || table_pages == 0 || table, "table is null");
  ARG(start, "start is null");
  ARG(T == 0 || (slots && positions), "slots and positions are required");
  SUPPORTED(R <= kMaxInt - 1024 && T <= kMaxInt - 1024, "R or T too large");
  TRY(check_table(table_pages, table_ld, page));
  ON_DEVICE(info);
  // Workgroups read what each request asks for, and the tokens' pages, while
  // others write the results.
  const Span lens_span(lens, R), state(free_state, 2);
  const Span table_span(table, R && table_pages ? (R - 1) * table_ld + table_pages : 0);
  const Span inputs[] = {lens_span, {new_tokens, R}, {release, R}, state, {ring, pages}, table_span};
  const Span outputs[] = {{out_lens, R}, {out_free_state, 2}, {granted, R}, {start, R + 1}, {slots, T}, {positions, T}};
  for (const Span& out : outputs)
    for (const Span& in : inputs)
      ARG(out.apart(in) || (&out == &outputs[0] && &in == &inputs[0] && out.same(in)) ||
              (&out == &outputs[1] && &in == &inputs[3] && out.same(in)),
          "an output overlaps an input (only out_lens may be lens, and out_free_state free_state)");
  for (int i = 0; i < 5; ++i)
    ARG(inputs[i].apart(table_span) && (i == 4 || inputs[i].apart(inputs[4])), "ring or table overlaps another input");
  PlanArgs a{};
  a.ring = ring;
  a.free_state = free_state;
  a.out_free_state = out_free_state;
  a.lens = lens;
  a.new_tokens = new_tokens;
  a.release = release;
  a.table = table;
  a.out_lens = out_lens;
  a.granted = granted;
  a.start = start;
  a.slots = slots;
  a.positions = positions;
  a.table_ld = table_ld;
  a.pages = (uint32_t)pages;
  a.page = (uint32_t)page;
  a.table_pages = (uint32_t)table_pages;
  a.R = (uint32_t)R;
  a.T = (uint32_t)T;
  a.by_page = FastDiv::of(a.page);
  a.status = info.status;
  return launched(launch_kv_plan(a, static_cast<hipStream_t>(stream)), "llmhip_kv_plan");
}

int llmhip_kv_append(llmhip_ctx* ctx, const llmhip_kv_cache* cache, uint32_t dtype, size_t T, const void* k,
                     int64_t k_token, int64_t k_head, const void* v, int64_t v_token, int64_t v_head,
                     const int64_t* slots, size_t q_heads, const void* q, int64_t q_token, int64_t q_head, void* out_q,
                     int64_t out_q_token, int64_t out_q_head, const int32_t* positions, const llmhip_rope* rope,
                     void* stream) {
  TRY(check_cache(cache));
  TRY(check_dtype(cache, dtype));
  ARG((q == nullptr) == (out_q == nullptr) && (q == nullptr) == (q_heads == 0), "q, out_q and q_heads go together");
  ARG(!rope || rope->dims == 0 || rope->freqs, "rope->freqs is null");
  ARG(!rope || rope->style <= LLMHIP_ROPE_NEIGHBOURS, "unknown rope style");
  ARG(!rope || (rope->dims % 2 == 0 && rope->dims <= cache->head_dim), "rope->dims must be even and at most head_dim");
  const uint32_t dims = rope ? rope->dims : 0u;
  SUPPORTED(T <= ((size_t)1 << 23) && q_heads <= kMaxHeads, "T (over 2^23) or q_heads too large");
  if (T == 0) return LLMHIP_OK;
  ARG(k && v && slots, "k, v and slots are required");
  ARG(!dims || positions, "positions are required with rope");
  const int64_t k_stride[2] = {k_token, k_head}, v_stride[2] = {v_token, v_head}, q_stride[2] = {q_token, q_head},
                out_q_stride[2] = {out_q_token, out_q_head};
  const uint64_t pool_extents[3] = {cache->pages, cache->page, cache->heads}, q_extents[2] = {T, q_heads};
  ARG(rows_apart(cache->k_stride, pool_extents, 3, cache->head_dim) && rows_apart(cache->v_stride, pool_extents, 3, cache->head_dim),
      "rows of a pool overlap");
  ARG(!q || rows_apart(out_q_stride, q_extents, 2, cache->head_dim), "rows of out_q overlap");
  // The widest vectors that the rows' starts and the pairs' places allow: a
  // vector of 16 bytes, or of 8, or single values; of neighbouring pairs two
  // vectors are one access.
  const uint32_t elem = size_of(dtype), kv_elem = size_of(cache->dtype), dim = cache->head_dim;
  const bool neighbours = rope && rope->style == LLMHIP_ROPE_NEIGHBOURS;
  uint32_t vec = (neighbours ? 8 : 16) / elem;
  for (const uint32_t least = 8 / elem; vec >= least; vec /= 2) {
    const uint32_t access = neighbours ? 2 * vec : vec, bytes = access * elem, kv_bytes = access * kv_elem;
    if (dims % (2 * vec) || (dim - dims) % (2 * vec)) continue;
    if (!rows_on(k, k_stride, 2, elem, bytes) || !rows_on(v, v_stride, 2, elem, bytes)) continue;
    if (q && (!rows_on(q, q_stride, 2, elem, bytes) || !rows_on(out_q, out_q_stride, 2, elem, bytes))) continue;
    if (rows_on(cache->k_pool, cache->k_stride, 3, kv_elem, kv_bytes) &&
        rows_on(cache->v_pool, cache->v_stride, 3, kv_elem, kv_bytes))
      break;
  }
  if (vec < 8 / elem) vec = 1;
  ON_DEVICE(info);
  AppendArgs a{};
  a.x[0] = q;
  a.x[1] = k;
  a.x[2] = v;
  a.out_q = out_q;
  set_pools(cache, const_cast<const void**>(a.pool), a.scale, a.pool_stride);
  if (q) memcpy(a.x_stride[0], q_stride, sizeof a.x_stride[0]);
  memcpy(a.x_stride[1], k_stride, sizeof a.x_stride[1]);
  memcpy(a.x_stride[2], v_stride, sizeof a.x_stride[2]);
  if (q) memcpy(a.oq_stride, out_q_stride, sizeof a.oq_stride);
  a.slots = slots;
  a.positions = positions;
  a.T = (uint32_t)T;
  a.q_heads = (uint32_t)q_heads;
  a.heads = cache->heads;
  a.dim = dim;
  a.dims = dims;
  a.pages = cache->pages;
  a.page = cache->page;
  a.status = info.status;
  if (dims) memcpy(a.freqs, rope->freqs, dims / 2 * sizeof(double));
  return launched(launch_kv_append(a, dtype, cache->dtype, neighbours, vec, static_cast<hipStream_t>(stream)),
                  "llmhip_kv_append");
}

int llmhip_kv_attend_workspace(llmhip_ctx* ctx, const llmhip_kv_cache* cache, size_t q_heads, size_t* bytes) {
  ARG(bytes, "bytes is null");
  TRY(check_cache(cache));
  ARG(q_heads >= 1 && q_heads % cache->heads == 0, "q_heads must be a multiple of the cache's heads");
  SUPPORTED(q_heads <= kMaxHeads, "q_heads too large");
  ARG(ctx, "ctx is null");
  *bytes = AttendPlan(cache->heads, cache->head_dim, q_heads, ctx_info(ctx).cus).bytes();
  return LLMHIP_OK;
}

int llmhip_kv_attend(llmhip_ctx* ctx, const llmhip_kv_cache* cache, uint32_t dtype, size_t B, size_t q_heads,
                     const void* q, int64_t q_request, int64_t q_head, const int32_t* table, size_t table_pages,
                     size_t table_ld, const int32_t* lens, size_t window, float scale, void* out, int64_t out_request,
                     int64_t out_head, float* out_lse, void* workspace, size_t workspace_bytes, void* stream) {
  TRY(check_cache(cache));
  TRY(check_dtype(cache, dtype));
  ARG(cache->dtype != LLMHIP_E4M3 || dtype != LLMHIP_F32, "dtype beside an E4M3 cache is BF16 or F16");
  ARG(q_heads >= 1 && q_heads % cache->heads == 0, "q_heads must be a multiple of the cache's heads");
  SUPPORTED(q_heads <= kMaxHeads && B <= kMaxBatch, "B or q_heads too large");
  TRY(check_table(table_pages, table_ld, cache->page));
  if (B == 0) return LLMHIP_OK;
  ARG(q && out && lens, "q, out and lens are required");
  const int64_t out_stride[2] = {out_request, out_head};
  const uint64_t out_extents[2] = {B, q_heads};
  ARG(rows_apart(out_stride, out_extents, 2, cache->head_dim), "rows of out overlap");
  ARG(table || table_pages == 0, "table is null");
  ARG(workspace && reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "workspace must be given, aligned to 16 bytes");
  ON_DEVICE(info);
  const AttendPlan plan(cache->heads, cache->head_dim, q_heads, info.cus);
  ARG(workspace_bytes >= plan.bytes(), "workspace is smaller than llmhip_kv_attend_workspace says");
  AttendArgs a{};
  a.q = q;
  a.out = out;
  a.lse = out_lse;
  set_pools(cache, a.pool, a.scale, a.pool_stride);
  a.table = table;
  a.lens = lens;
  a.q_stride[0] = q_request;
  a.q_stride[1] = q_head;
  a.out_stride[0] = out_request;
  a.out_stride[1] = out_head;
  a.table_ld = table_ld;
  a.workspace = static_cast<float*>(workspace);
  a.B = (uint32_t)B;
  a.q_heads = (uint32_t)q_heads;
  a.heads = cache->heads;
  a.dim = cache->head_dim;
  a.pages = cache->pages;
  a.page = cache->page;
  a.table_pages = (uint32_t)table_pages;
  a.window = window < kMaxInt ? (uint32_t)window : 0u;
  a.score_scale = scale;
  a.group = plan.group;
  a.blocks = plan.blocks;
  a.vheads = plan.vheads;
  a.cus = info.cus;
  a.part_words = plan.part_words;
  a.part_offset = kCutWords;
  a.by_page = FastDiv::of(a.page);
  a.by_dim = FastDiv::of(a.dim);
  a.status = info.status;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const bool bf16 = dtype == LLMHIP_BF16;
  hipError_t e;
  if (cache->dtype == LLMHIP_E4M3) e = bf16 ? launch_attend_e4m3_bf16(a, s) : launch_attend_e4m3_f16(a, s);
  else if (cache->dtype == LLMHIP_F32) e = launch_attend_f32(a, s);
  else e = bf16 ? launch_attend_bf16(a, s) : launch_attend_f16(a, s);
  return launched(e, "llmhip_kv_attend");
}

}  // extern "C"
