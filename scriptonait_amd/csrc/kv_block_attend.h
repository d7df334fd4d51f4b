// The attention kernels' launches for a cache with a scale for each block of
// tokens and head (llmhip_kv_block_attend).
//
// A lane's scores are those of a group of 8 neighbouring tokens, so a block of
// whole groups costs a lane one scale of keys and one of values for a tile: the
// first goes into the factor that the scores are multiplied with anyway, the
// second into the numerators, before they are split into two bfloat16. Other
// blocks (of one token, say) take a scale for each token. Several new tokens
// are further columns of the same products: the matrix cores take 16 queries of
// a cache head at once, whose tokens are read once.
#pragma once
#include "kv_attend.h"

namespace llmhip {

template <template <int, bool> class WIDE, template <int, bool> class WIDE_EACH, template <int, bool> class NARROW>
hipError_t launch_block_attend(const BlockAttendArgs& a, hipStream_t s) {
  const bool each = a.block_scales.by_block.d % 8u != 0u;
  if (a.dim % 16u == 0u || a.dim <= 32u)
    return each ? launch_attend_dims<WIDE_EACH, BlockAttendArgs>(a, s) : launch_attend_dims<WIDE, BlockAttendArgs>(a, s);
  if (a.dim < 128u) return each ? launch_attend_engine<NARROW<128, true>>(a, s) : launch_attend_engine<NARROW<128, false>>(a, s);
  return each ? launch_attend_engine<NARROW<256, true>>(a, s) : launch_attend_engine<NARROW<256, false>>(a, s);
}

}  // namespace llmhip
