/*
 * llmhip_kv.h — C ABI of the paged key-value cache that serves a decode
 * loop around llmhip_sampler.h's steps: which pages and slots the next
 * tokens take, their rotary positions and their way into the cache, and the
 * attention of one new token for each request over its pages.
 *
 * The reference keeps one ring cache for each generation and attends one
 * query at a time (crates/llm-core/src/model.rs:329-402); pages serve many
 * generations from one pool. A decode step is
 *   llmhip_kv_plan     pages for the tokens that each request adds
 *   llmhip_kv_append   for each layer: rotated queries and keys; keys and
 *                      values into their slots
 *   llmhip_kv_attend   for each layer: attention over the request's pages
 *   llmhip_decode_step the sampler, on the logits of the last layer
 *
 * Conventions as in llmhip_sampler.h: plain pointers and sizes, the caller
 * owns every buffer, an int status comes back, calls are stream-ordered and
 * return once their kernels are enqueued. No entry here allocates memory,
 * synchronizes or copies, so all of them can be recorded into a HIP graph.
 * Sizes and pointers are checked on the host. What only the device knows
 * (lengths, page ids, slots) is checked by the kernels: an entry outside its
 * range is left out as each function says, never followed, and sets
 * LLMHIP_KSTATUS_BAD_INDEX in the flags that llmhip_ctx_status returns.
 */
#ifndef LLMHIP_KV_H
#define LLMHIP_KV_H

#include "llmhip_sampler.h"

#ifdef __cplusplus
extern "C" {
#endif

/* A length, page id, slot or free-page count was outside its range. */
#define LLMHIP_KSTATUS_BAD_INDEX 2u

/* Element types. E4M3 is the 8-bit float with 4 exponent bits, no infinities. */
enum { LLMHIP_F32 = 0, LLMHIP_BF16 = 1, LLMHIP_F16 = 2, LLMHIP_E4M3 = 3 };

/*
 * The cache of one layer: two pools of `pages` pages of `page` tokens, each
 * token `heads` rows of `head_dim` values. Element [p][t][h][d] of a pool is
 * at p*stride[0] + t*stride[1] + h*stride[2] + d (strides in elements, so
 * pages that hold heads before tokens, or keys next to values, are views).
 * A slot is page id * page + token. head_dim is a multiple of 8 up to 256;
 * pool rows are aligned to 16 bytes (8 for E4M3).
 * E4M3 values stand for value * scale[head]; k_scale and v_scale are device
 * [heads] f32 then, and null for the other types.
 */
typedef struct llmhip_kv_cache {
  void* k_pool;
  void* v_pool;
  const float* k_scale;
  const float* v_scale;
  int64_t k_stride[3];
  int64_t v_stride[3];
  uint32_t dtype;
  uint32_t pages;
  uint32_t page;
  uint32_t heads;
  uint32_t head_dim;
} llmhip_kv_cache;

/*
 * Rotary positions: pair i of the first `dims` values of a head row is
 * turned by position * freqs[i] radians (freqs is a host array of dims / 2,
 * read during the call). Pair i is values (i, i + dims/2) in
 * LLMHIP_ROPE_HALVES and (2i, 2i + 1) in LLMHIP_ROPE_NEIGHBOURS.
 * Angles are computed in binary64.
 */
enum { LLMHIP_ROPE_HALVES = 0, LLMHIP_ROPE_NEIGHBOURS = 1 };
typedef struct llmhip_rope {
  const double* freqs;
  uint32_t dims;
  uint32_t style;
} llmhip_rope;

/*
 * Pages for the tokens that R requests add to their caches.
 *
 *   ring, free_state  the pool's free page ids, a ring of `pages` entries:
 *                     free_state[0] is the first free one's place,
 *                     free_state[1] how many there are
 *   lens          device [R] tokens that each request's cache holds
 *   new_tokens    device nullable [R] tokens that each request adds; null
 *                 adds one to every request that is not released
 *   release       device nullable [R]; nonzero: the request's pages go back
 *                 to the pool, in the requests' order, behind the free ones
 *                 (this call does not hand them out again), and its cache
 *                 is empty before new_tokens are added
 *   table         device [R][table_ld] page ids, table_pages of them used;
 *                 new pages are written behind a request's present ones
 *   out_lens      device [R] lengths with the tokens added (may be lens)
 *   granted       device [R] tokens that each request may add: all it asked
 *                 for, or 0. Requests are served in order. One is refused
 *                 when its table cannot hold them, when they pass token T of
 *                 the batch, or when the free pages do not reach; after the
 *                 first that the free pages do not reach for, every request
 *                 that needs a page is refused in this call
 *   start         device [R + 1] each request's first token in the batch
 *                 (refused requests keep their gap) and their sum, at most
 *                 2^31 - 1
 *   slots         device [T] each token's slot; -1 in gaps and past the end
 *   positions     device [T] each token's position; 0 there
 *   out_free_state device [2] the pool's state after the call (may be
 *                 free_state). ring and table change in place
 *
 * A length outside [0, table_pages * page], a negative new_tokens, a free
 * state outside the ring and a page id outside the pool (a released one
 * too, which goes back as it is) set
 * LLMHIP_KSTATUS_BAD_INDEX: the length is clamped, the count taken as 0, the
 * pool as empty, and the token's slot is -1. Apart from out_lens and
 * out_free_state no output may overlap an input, and ring and table none
 * either: refused.
 */
int llmhip_kv_plan(llmhip_ctx* ctx, size_t pages, size_t page, int32_t* ring, const int32_t* free_state, size_t R,
                   const int32_t* lens, const int32_t* new_tokens, const int32_t* release, int32_t* table,
                   size_t table_pages, size_t table_ld, int32_t* out_lens, int32_t* granted, int32_t* start, size_t T,
                   int64_t* slots, int32_t* positions, int32_t* out_free_state, void* stream);

/*
 * T tokens' keys and values into their slots, and their queries rotated.
 *
 *   dtype      of k, v, q and out_q: F32, BF16 or F16; the cache's is the
 *              same or E4M3
 *   k, v       device [T][heads][head_dim], a token's and a head's stride
 *              in elements; rows are dense. Slices of one packed projection
 *              output are such views
 *   slots      device [T]: llmhip_kv_plan's. A token of slot < 0 (padding)
 *              writes no key or value. Two tokens of one call must not share
 *              a slot
 *   q, out_q   device nullable [T][q_heads][head_dim] with strides; every
 *              token's query is rotated (out_q may be q itself). q_heads
 *              need not be a multiple of heads here
 *   positions  device [T], with rope
 *   rope       host, nullable: null stores keys and queries as they are
 *
 * Values are rotated in binary32 and rounded once to the output's type, to
 * nearest even; an E4M3 cache takes value / scale[head], clamped to +-448.
 * A slot past the pool is skipped and flagged. Rows of a pool or of out_q that
 * overlap (strides below head_dim) are refused.
 */
int llmhip_kv_append(llmhip_ctx* ctx, const llmhip_kv_cache* cache, uint32_t dtype, size_t T, const void* k,
                     int64_t k_token, int64_t k_head, const void* v, int64_t v_token, int64_t v_head,
                     const int64_t* slots, size_t q_heads, const void* q, int64_t q_token, int64_t q_head, void* out_q,
                     int64_t out_q_token, int64_t out_q_head, const int32_t* positions, const llmhip_rope* rope,
                     void* stream);

/* Bytes of workspace that llmhip_kv_attend takes for this cache and q_heads,
 * whatever the batch. */
int llmhip_kv_attend_workspace(llmhip_ctx* ctx, const llmhip_kv_cache* cache, size_t q_heads, size_t* bytes);

/*
 * Attention of one token for each of B requests over its cache:
 *   s_t = scale * (q . k_t),  out = sum_t softmax(s)_t v_t,
 *   lse = ln(sum_t exp(s_t))
 * over the last min(lens[b], window) tokens (window 0: all of them). Query
 * head h reads cache head h / (q_heads / heads). A request of length 0 gets
 * zeros and an lse of -inf.
 *
 *   dtype      of q and out: the cache's, or BF16 or F16 with an E4M3 cache
 *   q, out     device [B][q_heads][head_dim], a request's and a head's stride
 *              in elements
 *   table      device [B][table_ld] page ids, table_pages of them used
 *   lens       device [B], with the newest token
 *   out_lse    device nullable [B][q_heads] f32
 *   workspace  device, llmhip_kv_attend_workspace bytes, aligned to 16
 *              bytes; its contents need no setting up and mean nothing after
 *              the call. Calls that overlap need one each
 *
 * A length outside [0, table_pages * page] is clamped, and tokens on a page
 * id outside the pool are left out; both are flagged. Rows of out that overlap
 * are refused.
 * Scores, maxima, sums and outputs are accumulated in binary32, exponentials
 * and logarithms are the hardware's to base 2; a score that times log2(e)
 * passes binary32's largest number gives a row of NaN. With 16-bit queries each
 * softmax weight meets the values as the sum of two 16-bit numbers: off by at
 * most 2^-17 of itself, or in an F16 cache by 2^-23 of itself or 2^-44 of the
 * largest weight. An infinite value that a token of a weight above 0 holds
 * makes its column infinite, or NaN beside one of the other sign.
 */
int llmhip_kv_attend(llmhip_ctx* ctx, const llmhip_kv_cache* cache, uint32_t dtype, size_t B, size_t q_heads,
                     const void* q, int64_t q_request, int64_t q_head, const int32_t* table, size_t table_pages,
                     size_t table_ld, const int32_t* lens, size_t window, float scale, void* out, int64_t out_request,
                     int64_t out_head, float* out_lse, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* LLMHIP_KV_H */
