// Attention of f16 queries over whole numbers of 8 bits with a scale for each block.
#include "kv_block_attend.h"

namespace llmhip {

template <int DIM, bool FULL>
using BlockI8F16Wide = BlockEngine<F16, I8, DIM, FULL, DIM == 32 ? 8 : 16, false>;
template <int DIM, bool FULL>
using BlockI8F16WideEach = BlockEngine<F16, I8, DIM, FULL, DIM == 32 ? 8 : 16, true>;
template <int DIM, bool EACH>
using BlockI8F16Narrow = BlockEngine<F16, I8, DIM, false, 8, EACH>;

hipError_t launch_block_attend_i8_f16(const BlockAttendArgs& a, hipStream_t s) {
  return launch_block_attend<BlockI8F16Wide, BlockI8F16WideEach, BlockI8F16Narrow>(a, s);
}

}  // namespace llmhip
