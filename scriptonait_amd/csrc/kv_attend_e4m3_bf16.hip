// Attention of bf16 queries over an E4M3 cache.
#include "kv_attend.h"

namespace llmhip {

template <int DIM, bool FULL>
using Engine = Engine16<BF16, E4M3, DIM, FULL>;

hipError_t launch_attend_e4m3_bf16(const AttendArgs& a, hipStream_t s) { return launch_attend_dims<Engine>(a, s); }

}  // namespace llmhip
