// Index arithmetic of the paged key-value cache: everything that decides
// where a kernel reads and writes. Compiled for the device by the kernels
// and for the host by the CPU tests, which check that no input leaves the
// ranges.
#pragma once
#include <stdint.h>

#if defined(__HIPCC__)
#define LLMHIP_HD __host__ __device__ __forceinline__
#else
#define LLMHIP_HD inline
#endif

namespace llmhip {

// n / d for 0 <= n < 2^31 and 1 <= d < 2^31 without a division: with
// l = ceil(log2 d) and m = floor(2^32 (2^l - d) / d) + 1, the quotient is
// (mulhi(m, n) + n) >> l; n below 2^31 keeps the sum below 2^32.
struct FastDiv {
  uint32_t d, mul, shift;
  static FastDiv of(uint32_t d) {
    uint32_t l = 0;
    while (((uint64_t)1 << l) < d) ++l;
    return {d, (uint32_t)((((((uint64_t)1 << l) - d) << 32) / d) + 1u), l};
  }
  LLMHIP_HD uint32_t div(uint32_t n) const { return ((uint32_t)(((uint64_t)mul * n) >> 32) + n) >> shift; }
  LLMHIP_HD uint32_t mod(uint32_t n) const { return n - div(n) * d; }
};

// A length or page count as a kernel uses it: inside [0, most], and whether it was.
LLMHIP_HD uint32_t clamp_len(int32_t len, uint32_t most, bool& bad) {
  if (len < 0 || (uint32_t)len > most) {
    bad = true;
    return len < 0 ? 0u : most;
  }
  return (uint32_t)len;
}

// Page and token of a slot; false for a slot that writes nothing (bad is set
// when it is no padding either).
LLMHIP_HD bool split_slot(int64_t slot, uint32_t pages, uint32_t page, uint32_t& p, uint32_t& t, bool& bad) {
  if (slot < 0) return false;
  if ((uint64_t)slot >= (uint64_t)pages * page) {
    bad = true;
    return false;
  }
  p = (uint32_t)((uint64_t)slot / page);
  t = (uint32_t)((uint64_t)slot % page);
  return true;
}

// The same of a pool below 2^31 tokens, without 64-bit divisions.
LLMHIP_HD bool split_short_slot(int64_t slot, uint32_t pages, FastDiv page, uint32_t& p, uint32_t& t, bool& bad) {
  if (slot < 0) return false;
  if ((uint64_t)slot >= (uint64_t)pages * page.d) {
    bad = true;
    return false;
  }
  p = page.div((uint32_t)slot);
  t = (uint32_t)slot - p * page.d;
  return true;
}

// First token that a request's newest token sees.
LLMHIP_HD uint32_t window_start(uint32_t len, uint32_t window) { return window && len > window ? len - window : 0u; }

}  // namespace llmhip
