// How a call of the key-value cache's attention is split over workgroups.
// Compiled for the host by the kernels' launches and by the CPU tests, which
// check that no input leaves the workspace or the waves of a workgroup.
#pragma once
#include <stdint.h>

#include <algorithm>

namespace llmhip {

// The ranges that a call's work is cut into, and the requests of a call that
// is cut (their tiles' prefix sums live in LDS).
constexpr uint32_t kMaxRanges = 1024;
constexpr uint32_t kMaxSplitBatch = 2048;

struct AttendSplit {
  uint32_t team, splits;  // a workgroup's blocks of query heads, and waves for each
  uint32_t ranges;        // 0: a workgroup takes one request of one team
};

// waves: of a workgroup. tile: tokens of a tile; token_bytes: a token's key
// and value of one head. tokens: what the table holds.
inline AttendSplit attend_split(uint32_t waves, uint32_t tile, uint32_t token_bytes, uint32_t cus, uint32_t B,
                                uint32_t vheads, uint32_t tokens, uint32_t window) {
  // All waves have work: 12 heads are three teams of 4 with two waves each, not
  // two of 6 with one (head size 96: 130 us and 135; 3 heads of 64: 17 and 19).
  uint32_t cut_team = waves;
  while (vheads % cut_team) cut_team /= 2u;
  const uint32_t longest = (window ? std::min(tokens, window + tile) : tokens) / tile + 1u;
  // A workgroup of 8 waves, or two of 4, on each compute unit (two and three
  // times as many: 64 requests 104, 106, 110 us then, and 54, 80, 96 for one of
  // 131072 tokens of a single head). More requests, or tiles, than the line
  // takes are not cut, with a workgroup for each.
  const uint32_t groups = cus * (8u / waves);
  const bool cut = B <= kMaxSplitBatch && (uint64_t)B * longest <= 0x7fffffffu;
  // Nor are requests so short that a workgroup reads one whole sooner than
  // ranges are read and joined. The longest that the table or the window allow
  // counts, with as many waves for each head as there are workgroups for:
  //   up to 320 KiB a workgroup: 30 requests of up to 200 tokens of 8 heads of 128
  //     bf16 10.1 us whole, 15.9 cut; 3 of 60 tokens 5.9 and 9.0; one of 512 tokens
  //     of 2 heads of 64 f32 12.1 and 11.9, and one launch less.
  //   up to 1 MiB where the workgroups fill an eighth of the card: 300 of up to 100
  //     tokens 26.8 and 32.1, 200 of up to 1000 of one head 22.3 and 31.2. (Fewer:
  //     one of 2000 tokens of 8 heads 29.6 and 16.1.)
  //   up to 640 KiB there where rows are no whole cache lines: 37 of up to 1000 of
  //     12 heads of 80 f16, 737 KiB, 39.8 and 32.5.
  uint32_t team = cut_team;
  while (team > 1u && (uint64_t)B * (vheads / team) < groups) team /= 2u;
  const uint64_t takes = (uint64_t)B * (vheads / team), rounds = (takes + groups - 1u) / groups;
  const uint64_t bytes = ((uint64_t)longest + waves / team - 1u) / (waves / team) * waves * tile * token_bytes;
  const uint64_t few = takes < groups / 8u ? 320u : token_bytes / 2u % 128u ? 640u : 1024u;
  if (!cut || rounds == 0u || bytes <= few * 1024u / rounds) return {team, waves / team, 0u};
  const uint32_t teams = vheads / cut_team;
  return {cut_team, waves / cut_team, std::min(std::max(groups / teams, 1u), kMaxRanges)};
}

}  // namespace llmhip
