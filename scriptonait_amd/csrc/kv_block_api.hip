// C entry points of the cache of 8 bits with a scale for each block of tokens
// and head (declared in include/llmhip_kv.h).
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <string.h>

#include "kv_block_tasks.h"
#include "kv_check.h"

using namespace llmhip;

namespace {

constexpr uint32_t kMaxBlock = 256;
constexpr size_t kMaxNewTokens = 16;

int check_blocks(const llmhip_kv_blocks* c) {
  ARG(c, "cache is null");
  ARG(c->dtype == LLMHIP_I8 || c->dtype == LLMHIP_E4M3, "the cache's dtype must be I8 or E4M3");
  ARG(c->k_pool && c->v_pool && c->k_scale && c->v_scale, "k_pool, v_pool, k_scale and v_scale are required");
  ARG(c->pages >= 1 && c->page >= 1 && c->heads >= 1, "pages, page and heads must be at least 1");
  ARG(c->block >= 1 && c->page % c->block == 0, "block must be at least 1 and divide page");
  SUPPORTED(c->pages <= kMaxInt && c->page <= kMaxInt && c->heads <= kMaxHeads, "pages, page or heads too large");
  SUPPORTED(c->block <= kMaxBlock, "block must be at most 256");
  SUPPORTED(c->head_dim >= 8 && c->head_dim <= kMaxHeadDim && c->head_dim % 8 == 0,
            "head_dim must be a multiple of 8 up to 256");
  for (int i = 0; i < 3; ++i)
    ARG(c->k_stride[i] >= 0 && c->v_stride[i] >= 0 && c->k_scale_stride[i] >= 0 && c->v_scale_stride[i] >= 0,
        "strides of pools and scales must not be negative");
  SUPPORTED(rows_on(c->k_pool, c->k_stride, 3, 1, 8) && rows_on(c->v_pool, c->v_stride, 3, 1, 8),
            "pool rows must be aligned to 8 bytes");
  ARG(reinterpret_cast<uintptr_t>(c->k_scale) % 4 == 0 && reinterpret_cast<uintptr_t>(c->v_scale) % 4 == 0,
      "scales must be aligned to 4 bytes");
  return LLMHIP_OK;
}

int check_dtype(uint32_t dtype) {
  ARG(dtype <= LLMHIP_F16, "dtype must be F32, BF16 or F16");
  return LLMHIP_OK;
}

// Rows that a call writes: [n][m] of dim values each.
int check_out(const void* p, const int64_t* strides, size_t n, size_t m, uint32_t dim, const char* what) {
  const uint64_t extents[2] = {n, m};
  ARG(strides[0] >= 0 && strides[1] >= 0, "strides of what is written must not be negative");
  ARG(!p || rows_disjoint(strides, extents, 2, dim), what);
  return LLMHIP_OK;
}

// Whether a row of dim values and one of the same array's `from` values on meet:
// its directions' strides, the largest first, each of which steps past all that the
// ones behind it span. So only two steps of each can bring them together.
bool rows_meet(int64_t from, const int64_t* strides, const uint64_t* extents, int n, uint32_t dim) {
  if (n == 0) return from < (int64_t)dim && from > -(int64_t)dim;
  if (*extents < 2) return rows_meet(from, strides + 1, extents + 1, n - 1, dim);
  const int64_t below = from / *strides - (from % *strides < 0);
  for (int64_t step = below; step <= below + 1; ++step)
    if ((uint64_t)(step < 0 ? -step : step) < *extents && rows_meet(from - step * *strides, strides + 1, extents + 1, n - 1, dim))
      return true;
  return false;
}

// Whether the rows of two operands, [n][m] of dim values each, are apart: in
// memory of their own, or of the same strides and beside one another. (Neither's own
// rows overlap.)
bool pair_disjoint(const void* p, const void* q, const int64_t (*strides)[2], size_t n, size_t m, uint32_t dim, uint32_t elem) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(p), y = reinterpret_cast<uintptr_t>(q), between = x <= y ? y - x : x - y;
  const int64_t* low = strides[x <= y ? 0 : 1];
  if (between >= ((unsigned __int128)(uint64_t)low[0] * (n - 1) + (unsigned __int128)(uint64_t)low[1] * (m - 1) + dim) * elem) return true;
  if ((n > 1 && strides[0][0] != strides[1][0]) || (m > 1 && strides[0][1] != strides[1][1]) || between % elem) return false;
  const bool tokens_first = m < 2 || (n > 1 && low[0] >= low[1]);
  const int64_t ordered[2] = {low[!tokens_first], low[tokens_first]};
  const uint64_t extents[2] = {tokens_first ? n : m, tokens_first ? m : n};
  return !rows_meet((int64_t)(between / elem), ordered, extents, 2, dim);
}

BlockScales scales_of(const llmhip_kv_blocks* c) {
  BlockScales s{};
  s.scale[0] = c->k_scale;
  s.scale[1] = c->v_scale;
  memcpy(s.stride[0], c->k_scale_stride, sizeof c->k_scale_stride);
  memcpy(s.stride[1], c->v_scale_stride, sizeof c->v_scale_stride);
  s.by_block = FastDiv::of(c->block);
  return s;
}

template <class P>
void set_pools(const llmhip_kv_blocks* c, P* pool, int64_t (*stride)[3]) {
  pool[0] = c->k_pool;
  pool[1] = c->v_pool;
  memcpy(stride[0], c->k_stride, sizeof c->k_stride);
  memcpy(stride[1], c->v_stride, sizeof c->v_stride);
}

}  // namespace

extern "C" {

int llmhip_kv_block_append(llmhip_ctx* ctx, const llmhip_kv_blocks* cache, uint32_t dtype, size_t T, const void* k,
                           int64_t k_token, int64_t k_head, const void* v, int64_t v_token, int64_t v_head,
                           const int64_t* slots, size_t q_heads, const void* q, int64_t q_token, int64_t q_head,
                           void* out_q, int64_t out_q_token, int64_t out_q_head, const int32_t* positions,
                           const llmhip_rope* rope, void* stream) {
  TRY(check_blocks(cache));
  TRY(check_dtype(dtype));
  ARG((q == nullptr) == (out_q == nullptr) && (q == nullptr) == (q_heads == 0), "q, out_q and q_heads go together");
  ARG(!rope || rope->dims == 0 || rope->freqs, "rope->freqs is null");
  ARG(!rope || rope->style <= LLMHIP_ROPE_NEIGHBOURS, "unknown rope style");
  ARG(!rope || (rope->dims % 2 == 0 && rope->dims <= cache->head_dim), "rope->dims must be even and at most head_dim");
  const uint32_t dims = rope ? rope->dims : 0u, dim = cache->head_dim;
  SUPPORTED(T <= ((size_t)1 << 23) && q_heads <= kMaxHeads, "T (over 2^23) or q_heads too large");
  if (T == 0) return LLMHIP_OK;
  ARG(k && v && slots, "k, v and slots are required");
  ARG(!dims || positions, "positions are required with rope");
  const uint64_t pool_extents[3] = {cache->pages, cache->page, cache->heads},
                 scale_extents[3] = {cache->pages, cache->page / cache->block, cache->heads};
  ARG(rows_disjoint(cache->k_stride, pool_extents, 3, dim) && rows_disjoint(cache->v_stride, pool_extents, 3, dim),
      "rows of a pool overlap");
  ARG(rows_disjoint(cache->k_scale_stride, scale_extents, 3, 1) && rows_disjoint(cache->v_scale_stride, scale_extents, 3, 1),
      "scales overlap");
  const int64_t out_q_stride[2] = {out_q_token, out_q_head};
  TRY(check_out(out_q, out_q_stride, T, q_heads, dim, "rows of out_q overlap"));
  const bool neighbours = rope && rope->style == LLMHIP_ROPE_NEIGHBOURS;
  const uint32_t vec = append_vec(size_of(dtype), neighbours, dims, dim);
  ON_DEVICE(info);
  BlockAppendArgs a{};
  a.x[0] = q;
  a.x[1] = k;
  a.x[2] = v;
  a.out_q = out_q;
  set_pools(cache, a.pool, a.pool_stride);
  a.block_scales = scales_of(cache);
  const int64_t strides[3][2] = {{q_token, q_head}, {k_token, k_head}, {v_token, v_head}};
  memcpy(a.x_stride, strides, sizeof strides);
  memcpy(a.oq_stride, out_q_stride, sizeof out_q_stride);
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
  return launched(launch_kv_block_append(a, dtype, cache->dtype, neighbours, vec, static_cast<hipStream_t>(stream)),
                  "llmhip_kv_block_append");
}

int llmhip_kv_block_read(llmhip_ctx* ctx, const llmhip_kv_blocks* cache, uint32_t dtype, size_t T, const int64_t* slots,
                         void* out_k, int64_t out_k_token, int64_t out_k_head, void* out_v, int64_t out_v_token,
                         int64_t out_v_head, void* stream) {
  TRY(check_blocks(cache));
  TRY(check_dtype(dtype));
  SUPPORTED(T <= ((size_t)1 << 23), "T too large (over 2^23)");
  ARG(T == 0 || out_k || out_v, "out_k or out_v is required");
  if (T == 0) return LLMHIP_OK;
  ARG(slots, "slots are required");
  const int64_t strides[2][2] = {{out_k_token, out_k_head}, {out_v_token, out_v_head}};
  TRY(check_out(out_k, strides[0], T, cache->heads, cache->head_dim, "rows of out_k overlap"));
  TRY(check_out(out_v, strides[1], T, cache->heads, cache->head_dim, "rows of out_v overlap"));
  ARG(!out_k || !out_v || pair_disjoint(out_k, out_v, strides, T, cache->heads, cache->head_dim, size_of(dtype)),
      "rows of out_k and out_v overlap");
  ON_DEVICE(info);
  BlockReadArgs a{};
  a.out[0] = out_k;
  a.out[1] = out_v;
  memcpy(a.out_stride, strides, sizeof strides);
  set_pools(cache, a.pool, a.pool_stride);
  a.block_scales = scales_of(cache);
  a.slots = slots;
  a.T = (uint32_t)T;
  a.heads = cache->heads;
  a.dim = cache->head_dim;
  a.pages = cache->pages;
  a.page = cache->page;
  a.status = info.status;
  return launched(launch_kv_block_read(a, dtype, cache->dtype, static_cast<hipStream_t>(stream)), "llmhip_kv_block_read");
}

int llmhip_kv_block_attend_workspace(llmhip_ctx* ctx, const llmhip_kv_blocks* cache, size_t new_tokens, size_t q_heads,
                                     size_t* bytes) {
  ARG(bytes, "bytes is null");
  TRY(check_blocks(cache));
  ARG(new_tokens >= 1, "new_tokens must be at least 1");
  SUPPORTED(new_tokens <= kMaxNewTokens, "new_tokens must be at most 16");
  ARG(q_heads >= 1 && q_heads % cache->heads == 0, "q_heads must be a multiple of the cache's heads");
  SUPPORTED(q_heads <= kMaxHeads, "q_heads too large");
  ARG(ctx, "ctx is null");
  *bytes = AttendPlan(cache->heads, cache->head_dim, q_heads * new_tokens, ctx_info(ctx).cus).bytes();
  return LLMHIP_OK;
}

int llmhip_kv_block_attend(llmhip_ctx* ctx, const llmhip_kv_blocks* cache, uint32_t dtype, size_t B, size_t new_tokens,
                           size_t q_heads, const void* q, int64_t q_request, int64_t q_token, int64_t q_head,
                           const int32_t* table, size_t table_pages, size_t table_ld, const int32_t* lens,
                           size_t window, float scale, void* out, int64_t out_request, int64_t out_token,
                           int64_t out_head, float* out_lse, void* workspace, size_t workspace_bytes, void* stream) {
  TRY(check_blocks(cache));
  ARG(dtype == LLMHIP_BF16 || dtype == LLMHIP_F16, "dtype must be BF16 or F16");
  ARG(new_tokens >= 1, "new_tokens must be at least 1");
  SUPPORTED(new_tokens <= kMaxNewTokens, "new_tokens must be at most 16");
  ARG(q_heads >= 1 && q_heads % cache->heads == 0, "q_heads must be a multiple of the cache's heads");
  SUPPORTED(q_heads <= kMaxHeads && B <= kMaxBatch, "B or q_heads too large");
  TRY(check_table(table_pages, table_ld, cache->page));
  if (B == 0) return LLMHIP_OK;
  ARG(q && out && lens, "q, out and lens are required");
  const int64_t out_stride[3] = {out_request, out_token, out_head};
  const uint64_t out_extents[3] = {B, new_tokens, q_heads};
  ARG(out_request >= 0 && out_token >= 0 && out_head >= 0, "strides of what is written must not be negative");
  ARG(rows_disjoint(out_stride, out_extents, 3, cache->head_dim), "rows of out overlap");
  ARG(table || table_pages == 0, "table is null");
  ARG(workspace && reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "workspace must be given, aligned to 16 bytes");
  ON_DEVICE(info);
  const size_t queries = q_heads * new_tokens;
  const AttendPlan plan(cache->heads, cache->head_dim, queries, info.cus);
  ARG(workspace_bytes >= plan.bytes(), "workspace is smaller than llmhip_kv_block_attend_workspace says");
  BlockAttendArgs a{};
  a.q = q;
  a.out = out;
  a.lse = out_lse;
  set_pools(cache, a.pool, a.pool_stride);
  a.block_scales = scales_of(cache);
  a.table = table;
  a.lens = lens;
  a.q_stride[0] = q_request;
  a.q_stride[1] = q_head;
  a.q_token = q_token;
  a.out_stride[0] = out_request;
  a.out_stride[1] = out_head;
  a.out_token = out_token;
  a.table_ld = table_ld;
  a.workspace = static_cast<float*>(workspace);
  a.B = (uint32_t)B;
  a.tokens = (uint32_t)new_tokens;
  a.per_token = (uint32_t)q_heads / cache->heads;
  a.by_per_token = FastDiv::of(a.per_token);
  a.q_heads = (uint32_t)queries;
  a.heads = cache->heads;
  a.dim = cache->head_dim;
  a.pages = cache->pages;
  a.page = cache->page;
  a.table_pages = (uint32_t)table_pages;
  a.seen_window = window < kMaxInt - kMaxNewTokens ? (uint32_t)window : 0u;
  a.window = a.seen_window ? a.seen_window + a.tokens - 1u : 0u;
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
  const hipError_t e = cache->dtype == LLMHIP_I8 ? (bf16 ? launch_block_attend_i8_bf16(a, s) : launch_block_attend_i8_f16(a, s))
                                                 : (bf16 ? launch_block_attend_e4m3_bf16(a, s) : launch_block_attend_e4m3_f16(a, s));
  return launched(e, "llmhip_kv_block_attend");
}

}  // extern "C"
