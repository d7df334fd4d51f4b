// Attention of bf16 queries over E4M3 codes with a scale for each block.
#include "kv_block_attend.h"

namespace llmhip {

template <int DIM, bool FULL>
using BlockE4M3BF16Wide = BlockEngine<BF16, E4M3, DIM, FULL, DIM == 32 ? 8 : 16, false>;
template <int DIM, bool FULL>
using BlockE4M3BF16WideEach = BlockEngine<BF16, E4M3, DIM, FULL, DIM == 32 ? 8 : 16, true>;
template <int DIM, bool EACH>
using BlockE4M3BF16Narrow = BlockEngine<BF16, E4M3, DIM, false, 8, EACH>;

hipError_t launch_block_attend_e4m3_bf16(const BlockAttendArgs& a, hipStream_t s) {
  return launch_block_attend<BlockE4M3BF16Wide, BlockE4M3BF16WideEach, BlockE4M3BF16Narrow>(a, s);
}

}  // namespace llmhip
