// Attention of f16 queries over a cache of the same type.
#include "kv_attend.h"

namespace llmhip {

template <int DIM, bool FULL>
using Engine = Engine16<F16, F16, DIM, FULL>;

hipError_t launch_attend_f16(const AttendArgs& a, hipStream_t s) { return launch_attend_dims<Engine>(a, s); }

}  // namespace llmhip
