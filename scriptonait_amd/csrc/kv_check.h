// What the key-value cache's entry points check on the host, before the
// context, so that a wrong call says what is wrong with it also where there is
// no device.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include <algorithm>

#include "ctx_info.h"
#include "device_scope.h"
#include "kv_args.h"

namespace llmhip {

inline int arg_fail(const char* what) {
  set_last_error(what);
  return LLMHIP_ERR_INVALID_ARGUMENT;
}
inline int unsupported(const char* what) {
  set_last_error(what);
  return LLMHIP_ERR_UNSUPPORTED;
}
inline int launched(hipError_t e, const char* what) {
  if (e == hipSuccess) return LLMHIP_OK;
  char buf[256];
  snprintf(buf, sizeof buf, "%s: %s (%d)", what, hipGetErrorString(e), (int)e);
  set_last_error(buf);
  return e == hipErrorOutOfMemory ? LLMHIP_ERR_OUT_OF_MEMORY : LLMHIP_ERR_HIP;
}

#define ARG(cond, what) \
  if (!(cond)) return arg_fail(what)
#define SUPPORTED(cond, what) \
  if (!(cond)) return unsupported(what)

// Memory of an argument; a null one has none.
struct Span {
  uintptr_t at;
  size_t bytes;
  template <class T>
  Span(const T* p, size_t n) : at(reinterpret_cast<uintptr_t>(p)), bytes(p ? n * sizeof(T) : 0) {}
  bool apart(const Span& o) const { return !bytes || !o.bytes || at + bytes <= o.at || o.at + o.bytes <= at; }
  bool same(const Span& o) const { return at == o.at && bytes == o.bytes; }
};

constexpr size_t kMaxInt = 0x7fffffff;
constexpr size_t kMaxBatch = 65535;
constexpr size_t kMaxHeads = 65535;

inline uint32_t size_of(uint32_t dtype) { return dtype == LLMHIP_F32 ? 4u : dtype == LLMHIP_E4M3 ? 1u : 2u; }

// Whether every row of an operand starts on `bytes`.
inline bool rows_on(const void* p, const int64_t* strides, int n, uint32_t elem, uint32_t bytes) {
  if (reinterpret_cast<uintptr_t>(p) % bytes) return false;
  for (int i = 0; i < n; ++i)
    if ((uint64_t)strides[i] * elem % bytes) return false;
  return true;
}

// Whether neighbours in each direction have `dim` values to themselves.
inline bool rows_apart(const int64_t* strides, const uint64_t* extents, int n, uint32_t dim) {
  for (int i = 0; i < n; ++i)
    if (extents[i] > 1 && strides[i] < (int64_t)dim && strides[i] > -(int64_t)dim) return false;
  return true;
}

// Whether no two rows of `dim` values lie over one another: each direction steps
// past all that the directions with smaller steps span. Strides are not negative.
inline bool rows_disjoint(const int64_t* strides, const uint64_t* extents, int n, uint32_t dim) {
  int order[4];
  for (int i = 0; i < n; ++i) order[i] = i;
  std::sort(order, order + n, [&](int x, int y) { return strides[x] < strides[y]; });
  unsigned __int128 span = dim;
  for (int i = 0; i < n; ++i) {
    const int k = order[i];
    if (extents[k] < 2) continue;
    if ((uint64_t)strides[k] < span) return false;
    span += (unsigned __int128)(uint64_t)strides[k] * (extents[k] - 1);
  }
  return true;
}

inline int check_table(size_t table_pages, size_t table_ld, size_t page) {
  ARG(table_ld >= table_pages, "table_ld < table_pages");
  SUPPORTED(table_pages <= kMaxInt && (table_pages + 1) * page <= kMaxInt - 256, "table_pages * page must be below 2^31");
  return LLMHIP_OK;
}

#define TRY(expr)                       \
  do {                                  \
    const int st_ = (expr);             \
    if (st_ != LLMHIP_OK) return st_;   \
  } while (0)

#define ON_DEVICE(info)                                                    \
  ARG(ctx, "ctx is null");                                                 \
  const CtxInfo info = ctx_info(ctx);                                      \
  Device scope(info.device);                                               \
  if (!scope.ok) return launched(hipErrorInvalidDevice, "hipSetDevice")

// Sizes of the attention's work and workspace. q_heads: of a token, or of all
// of a request's new tokens.
struct AttendPlan {
  uint32_t group, blocks, vheads, part_words;
  size_t parts;  // partial answers: two for each range and block of query heads
  AttendPlan(uint32_t heads, uint32_t head_dim, size_t q_heads, uint32_t cus) {
    group = (uint32_t)q_heads / heads;
    blocks = (group + 15u) / 16u;
    vheads = blocks * heads;
    part_words = (std::min(group, 16u) * (head_dim + 2u) + 3u) / 4u * 4u;
    // Workgroups of up to 8 blocks fill the card, or two of up to 4: a range
    // for each 8 of the blocks at most, and one range at least.
    parts = 2 * std::max<size_t>(vheads, (size_t)8 * cus);
  }
  size_t bytes() const { return (kCutWords + parts * part_words) * 4; }
};

}  // namespace llmhip
