// Attention of f16 queries over an E4M3 cache.
#include "kv_attend.h"

namespace llmhip {

template <int DIM, bool FULL>
using WideF16 = Engine16<F16, E4M3, DIM, FULL, DIM == 32 ? 8 : 16>;
template <int DIM>
using NarrowF16 = Engine16<F16, E4M3, DIM, false, 8>;

hipError_t launch_attend_e4m3_f16(const AttendArgs& a, hipStream_t s) {
  if (a.dim % 16u == 0u || a.dim <= 32u) return launch_attend_dims<WideF16>(a, s);
  return a.dim < 128u ? launch_attend_engine<NarrowF16<128>>(a, s) : launch_attend_engine<NarrowF16<256>>(a, s);
}

}  // namespace llmhip
