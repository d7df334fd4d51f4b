// The attention kernels' launches for a cache with a scale for each block of
// tokens and head (llmhip_kv_block_attend).
//
// A lane's scores are those of a group of 8 neighbouring tokens. Their scales of
// keys go into the factor that scores are multiplied with anyway, those of values
// into the numerators, before they are split into two bfloat16. A block of whole
// groups has one scale of each for a lane and tile; other blocks (of one token,
// say) one for each token. Several new tokens are further columns of the same
// products: the matrix cores take 16 queries of a cache head at once, whose tokens
// are read once.
//
// What bounds it is reading the cache once: 2.2 GB of 256 requests in 337-362 us (box
// to box, E4M3 level; 6.1-6.5 TB/s). Not at that bound: 269 MB of one request in 49
// to 56 and 7 for the join, with 16 tiles a wave. Four new tokens of 64 requests 63
// and 10 us (66 with a scale for each token), one 54 and 6: partial answers are
// four times as large, 20 MB written and read.
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
