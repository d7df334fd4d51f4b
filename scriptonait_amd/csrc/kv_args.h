// Arguments of the paged key-value cache's kernels, passed by value.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/llmhip_kv.h"
#include "kv_index.h"
#include "kv_split.h"

namespace llmhip {

constexpr uint32_t kMaxHeadDim = 256;
constexpr uint32_t kCutWords = 4 * kMaxRanges;  // attention: workspace words before the partial answers

struct PlanArgs {
  int32_t* ring;
  const int32_t* free_state;
  int32_t* out_free_state;
  const int32_t* lens;
  const int32_t* new_tokens;  // nullable
  const int32_t* release;     // nullable
  int32_t* table;
  int32_t* out_lens;
  int32_t* granted;
  int32_t* start;
  int64_t* slots;
  int32_t* positions;
  uint64_t table_ld;
  uint32_t pages, page, table_pages, R, T;
  bool tokens, requests;  // what a launch writes: slots, positions and new pages; all else
  FastDiv by_page;
  uint32_t* status;
};

struct AppendArgs {
  const void* x[3];  // queries, keys, values
  void* out_q;
  void* pool[2];
  const float* scale[2];  // E4M3: one for each head
  int64_t x_stride[3][2];
  int64_t oq_stride[2];
  int64_t pool_stride[2][3];
  const int64_t* slots;
  const int32_t* positions;
  uint32_t T, q_heads, heads, dim, dims, pages, page;
  FastDiv by_token, by_row;  // units of a token, units of a head row
  uint32_t tokens_per_group;
  uint32_t* status;
  double freqs[kMaxHeadDim / 2];
};

// For each block of tokens and head: where its scale is, and which block a
// token of a page is in.
struct BlockScales {
  float* scale[2];
  int64_t stride[2][3];  // page, block, head
  FastDiv by_block;
};

struct BlockAppendArgs : AppendArgs {
  BlockScales block_scales;
  uint32_t kv_tokens, kv_groups, kv_parts;  // groups of tokens whose keys and values are written, and workgroups for each
  uint32_t turn_tokens;                     // tokens whose cosines and sines LDS holds
  bool short_slots;              // the pool has less than 2^31 tokens
  FastDiv by_half, by_heads, by_page;
};

struct BlockReadArgs {
  void* out[2];  // nullable
  const void* pool[2];
  int64_t out_stride[2][2];
  int64_t pool_stride[2][3];
  BlockScales block_scales;
  const int64_t* slots;
  uint32_t T, heads, dim, pages, page;
  bool short_slots;  // the pool has less than 2^31 tokens
  FastDiv by_token, by_row, by_page;  // units of a token, units of a head row
  uint32_t tokens_per_group;
  uint32_t* status;
};

struct AttendArgs {
  const void* q;
  void* out;
  float* lse;  // nullable
  const void* pool[2];
  const float* scale[2];
  const int32_t* table;
  const int32_t* lens;
  int64_t q_stride[2], out_stride[2];
  int64_t pool_stride[2][3];
  uint64_t table_ld;
  float* workspace;
  uint32_t B, q_heads, heads, dim, pages, page, table_pages, window;
  float score_scale;
  uint32_t group, blocks, vheads;  // query heads of a cache head, in blocks of 16; blocks of all heads
  uint32_t cus;                    // the device's compute units
  uint32_t team, splits;           // a workgroup's blocks of heads, and waves for each
  uint32_t ranges;                 // 0: a workgroup takes one request of one team
  uint32_t start_words;            // LDS words of the requests' starts, a multiple of 4
  uint32_t part_words;             // workspace words of a partial answer, a multiple of 4
  uint32_t part_offset;            // and of the first one
  FastDiv by_page, by_dim;
  uint32_t* status;
};

// A cache head's queries are those of all new tokens: `group` and `q_heads`
// count them, a query is number token * per_token + head of its cache head.
struct BlockAttendArgs : AttendArgs {
  BlockScales block_scales;
  int64_t q_token, out_token;  // strides
  uint32_t tokens, per_token;
  uint32_t seen_window;  // of one token; `window` is that of all of them
  FastDiv by_per_token;
};

hipError_t launch_kv_plan(const PlanArgs& a, hipStream_t s);
hipError_t launch_kv_append(const AppendArgs& a, uint32_t dtype, uint32_t kv_dtype, bool neighbours, uint32_t vec,
                            hipStream_t s);
hipError_t launch_kv_block_append(const BlockAppendArgs& a, uint32_t dtype, uint32_t kv_dtype, bool neighbours, uint32_t vec,
                                  hipStream_t s);
hipError_t launch_kv_block_read(const BlockReadArgs& a, uint32_t dtype, uint32_t kv_dtype, hipStream_t s);
hipError_t launch_attend_f32(const AttendArgs& a, hipStream_t s);
hipError_t launch_attend_bf16(const AttendArgs& a, hipStream_t s);
hipError_t launch_attend_f16(const AttendArgs& a, hipStream_t s);
hipError_t launch_attend_e4m3_bf16(const AttendArgs& a, hipStream_t s);
hipError_t launch_attend_e4m3_f16(const AttendArgs& a, hipStream_t s);
hipError_t launch_block_attend_i8_bf16(const BlockAttendArgs& a, hipStream_t s);
hipError_t launch_block_attend_i8_f16(const BlockAttendArgs& a, hipStream_t s);
hipError_t launch_block_attend_e4m3_bf16(const BlockAttendArgs& a, hipStream_t s);
hipError_t launch_block_attend_e4m3_f16(const BlockAttendArgs& a, hipStream_t s);

}  // namespace llmhip
