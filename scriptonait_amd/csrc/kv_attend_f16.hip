// Attention of f16 queries over a cache of the same type.
#include "kv_attend.h"

namespace llmhip {

template <int DIM, bool FULL>
using EngineF16 = Engine16<F16, F16, DIM, FULL, 8>;

hipError_t launch_attend_f16(const AttendArgs& a, hipStream_t s) { return launch_attend_dims<EngineF16>(a, s); }

}  // namespace llmhip
