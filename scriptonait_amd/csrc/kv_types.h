// Element types of the key-value cache's kernels: as stored, and as binary32.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/llmhip_kv.h"

namespace llmhip {

struct F32 {
  using Raw = float;
  static constexpr uint32_t kId = LLMHIP_F32;
  __device__ static __forceinline__ float load(Raw x) { return x; }
  __device__ static __forceinline__ Raw store(float x) { return x; }
};
struct BF16 {
  using Raw = __bf16;
  static constexpr uint32_t kId = LLMHIP_BF16;
  __device__ static __forceinline__ float load(Raw x) { return (float)x; }
  __device__ static __forceinline__ Raw store(float x) { return (Raw)x; }
};
struct F16 {
  using Raw = _Float16;
  static constexpr uint32_t kId = LLMHIP_F16;
  __device__ static __forceinline__ float load(Raw x) { return (float)x; }
  __device__ static __forceinline__ Raw store(float x) { return (Raw)x; }
};
// 4 exponent bits, 3 mantissa bits, largest value 448, no infinities: the
// conversion instructions of gfx950 take and give this format.
struct E4M3 {
  using Raw = uint8_t;
  static constexpr uint32_t kId = LLMHIP_E4M3;
  static constexpr float kMax = 448.0f;
  __device__ static __forceinline__ float load(Raw x) { return __builtin_amdgcn_cvt_f32_fp8((int)x, 0); }
  // NaN passes both comparisons' false sides and stays NaN.
  __device__ static __forceinline__ Raw store(float x) {
    x = x > kMax ? kMax : x;
    x = x < -kMax ? -kMax : x;
    return (Raw)(__builtin_amdgcn_cvt_pk_fp8_f32(x, 0.0f, 0, false) & 0xff);
  }
};

// N values of one row, moved as one access.
template <class T, int N>
struct alignas(sizeof(typename T::Raw) * N) Pack {
  typename T::Raw v[N];
};

}  // namespace llmhip
