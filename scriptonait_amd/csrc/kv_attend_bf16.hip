// Attention of bf16 queries over a cache of the same type.
#include "kv_attend.h"

namespace llmhip {

template <int DIM, bool FULL>
using EngineBF16 = Engine16<BF16, BF16, DIM, FULL, 8>;

hipError_t launch_attend_bf16(const AttendArgs& a, hipStream_t s) { return launch_attend_dims<EngineBF16>(a, s); }

}  // namespace llmhip
