// Sizes of the work that llmhip_kv_block_append's workgroups share. Compiled for
// the host by the launches and by a CPU test, which checks that no call's tables
// pass what a workgroup has.
#pragma once
#include <stdint.h>

#include <algorithm>

namespace llmhip {

constexpr uint32_t kAppendThreads = 256;
constexpr uint32_t kMaxQueryTokens = 8;    // of a workgroup of queries
constexpr uint32_t kMaxTurned = 256 + 15;  // tokens whose cosines and sines LDS holds: a block's, and some more

// Values of a vector, the widest that the pairs' places allow: of 16 bytes, or of
// 8, or single values; of neighbouring pairs two vectors are one access.
inline uint32_t append_vec(uint32_t elem, bool neighbours, uint32_t dims, uint32_t dim) {
  uint32_t vec = (neighbours ? 8 : 16) / elem;
  const uint32_t least = 8 / elem;
  while (vec >= least && (dims % (2 * vec) || (dim - dims) % (2 * vec))) vec /= 2;
  return vec < least ? 1u : vec;
}

// Units (two vectors) of a lane in registers: 32 values, 16 where they take more
// addresses. (16 for all, in five waves of a SIMD and not four: 16384 tokens with 32
// heads of queries 81 us and 85, without queries 45 and 36, 2047 in blocks of 64
// 24 and 18.)
constexpr uint32_t append_held(uint32_t vec) { return vec >= 4 ? 16 / vec : 8 / vec; }

// Tokens whose cosines and sines LDS holds: all of a step of one block, and some
// of its neighbours'. `longest`: tokens of a block that a call can write.
inline uint32_t append_turn_tokens(uint32_t longest, uint32_t vec, uint32_t dim) {
  return std::min(longest, kAppendThreads * append_held(vec) / (dim / (2 * vec)) + 2u) + 15u;
}

}  // namespace llmhip
