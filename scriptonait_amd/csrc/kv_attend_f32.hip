// Attention over a binary32 cache.
#include "kv_attend.h"

namespace llmhip {

hipError_t launch_attend_f32(const AttendArgs& a, hipStream_t s) { return launch_attend_dims<Engine32>(a, s); }

}  // namespace llmhip
