// The rotation of a rotary position: cosine and sine of its angle.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace llmhip {

struct Turn {
  double cos, sin;
};

// cos and sin of x: x - k pi/2 with pi/2 in two parts (k < 2^31 keeps the
// rest's error below 2^-70), then the Taylor sums. At pi/4 the first left
// out terms are 4e-14 (sin, x^15 / 15!) and 1e-12 (cos, x^14 / 14!), far
// below half a step of binary32; FINE: 5e-17 and 2e-18.
template <bool FINE>
__device__ __forceinline__ Turn turn_of(double x) {
  const double k = rint(x * 0.63661977236758134308);
  double r = __builtin_fma(-k, 1.57079632679489661923, x);
  r = __builtin_fma(-k, 6.123233995736766036e-17, r);
  const double z = r * r;
  double s = 1.0 / 6227020800.0, c = 1.0 / 479001600.0;
  if (FINE) {
    s = __builtin_fma(-1.0 / 1307674368000.0, z, s);
    c = __builtin_fma(__builtin_fma(1.0 / 20922789888000.0, z, -1.0 / 87178291200.0), z, c);
  }
  s = __builtin_fma(s, z, -1.0 / 39916800.0);
  s = __builtin_fma(s, z, 1.0 / 362880.0);
  s = __builtin_fma(s, z, -1.0 / 5040.0);
  s = __builtin_fma(s, z, 1.0 / 120.0);
  s = __builtin_fma(s, z, -1.0 / 6.0);
  s = __builtin_fma(s * z, r, r);
  c = __builtin_fma(c, z, -1.0 / 3628800.0);
  c = __builtin_fma(c, z, 1.0 / 40320.0);
  c = __builtin_fma(c, z, -1.0 / 720.0);
  c = __builtin_fma(c, z, 1.0 / 24.0);
  c = __builtin_fma(c, z, -0.5);
  c = __builtin_fma(c, z, 1.0);
  const int32_t quarter = (int32_t)(int64_t)k & 3;
  const double cc = quarter & 1 ? s : c, ss = quarter & 1 ? c : s;
  return {quarter == 1 || quarter == 2 ? -cc : cc, quarter >= 2 ? -ss : ss};
}

__device__ __forceinline__ float2 cos_sin(double x) {
  const Turn t = turn_of<false>(x);
  return {(float)t.cos, (float)t.sin};
}

}  // namespace llmhip
