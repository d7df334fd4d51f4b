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
  // Nor are requests so short that workgroups read them whole, one for each
  // request and team, sooner than ranges are read and joined. A team is as
  // small then as there are workgroups for. Both times, in bytes that one
  // workgroup reads, for the longest requests that the table or the window allow:
  //   whole: its request's tiles, of which each has the time of 12 KiB before its
  //     bytes come, and 288 KiB; more workgroups than the card takes have turns.
  //   cut: 1280 KiB, and a quarter of a workgroup's share of all tiles (requests
  //     are shorter than the longest, and all waves work all of the time).
  // Measured over 7600 calls of 1 to 400 requests, 1 to 32 heads of 16 to 256
  // values with 1 to 32 queries each, all types, windows of 128 to 1000 tokens and
  // none, by the quotient of the two (us: medians; measured: geometric means):
  //   by the rule  to 0.5  -0.75     -1  -1.33     -2     -4   more
  //   whole, us       8.1   12.9   19.4   24.3   31.5   47.3   84.8
  //   cut, us        11.8   15.5   20.3   23.8   28.0   25.8   22.1
  //   measured       0.70   0.84   0.95   1.06   1.18   1.64   3.87
  // The better of the two is missed by 2.4% in the mean (all whole 14%, all cut
  // 21%), by 2.8% over 1200 calls that the numbers were not chosen by. So much for
  // caches of values, which those calls were. Of caches of 8 bits with block scales,
  // over 900 calls of 1 to 8 new tokens of 1 to 400 requests, it is missed by 3.4%
  // (all whole 13%, all cut 23%), most where requests have a tile or two of heads
  // of 256.
  uint32_t team = cut_team;
  while (team > 1u && (uint64_t)B * (vheads / team) < groups) team /= 2u;
  constexpr double kKiB = 1024.0;
  const double turns = std::max((double)B * (vheads / team) / groups, 1.0);
  const double tile_time = (double)tile * token_bytes + 12.0 * kKiB;
  const uint32_t wave_tiles = (uint32_t)(((uint64_t)longest + waves / team - 1u) / (waves / team));
  const double whole_time = turns * (wave_tiles * (double)waves * tile_time + 288.0 * kKiB);
  const double cut_time = 1280.0 * kKiB + 0.25 * B * longest * vheads / groups * tile_time;
  if (!cut || whole_time <= cut_time) return {team, waves / team, 0u};
  const uint32_t teams = vheads / cut_team;
  return {cut_team, waves / cut_team, std::min(std::max(groups / teams, 1u), kMaxRanges)};
}

}  // namespace llmhip
