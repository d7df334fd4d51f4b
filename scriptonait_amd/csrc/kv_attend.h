// Attention of one new token over its request's pages (llmhip_kv_attend).
//
// With s_t the scores in base-2 exponents and m a reference that no score
// passes by more than 8, a run of tokens is held as
//   m,  l = sum 2^(s_t - m),  o = sum 2^(s_t - m) v_t,
// runs are joined by l = sum_k l_k 2^(m_k - M), o likewise, and the answer
// is o / l. m moves only when a score passes it by more than 8: the
// numerators then stay below 2^8 and the largest is at least 1, and most
// tiles neither compare across lanes nor scale o. (Where they are held as F16
// m is 7 lower, for their small ones: 2^15, and at least 2^7.)
//
// The work is every request's tiles of tokens in one line, cut into equal
// ranges, so ragged lengths share the card evenly and one long request uses
// all of it. A workgroup takes one range: a wave for each of up to 8 cache
// heads, which so read a token's neighbouring rows at about the same time,
// and where there are fewer heads, several waves for each, equal parts of
// the range. (Reading 537 MB of 131072 tokens of 8 heads of 256 bytes this way
// takes 80 us, with workgroups of one head 86 us.) A request's run inside one
// wave goes straight to the output; runs that waves of one head share are
// joined in LDS, and what a workgroup leaves of a request that goes on
// elsewhere goes to the workspace, for join_kernel. What bounds it is reading
// the cache once.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "kv_args.h"
#include "kv_engines.h"
#include "wave_ops.h"

namespace llmhip {

// Waves of a workgroup: 8, two on each SIMD, where the registers allow it.
template <class E, bool GROUPED>
constexpr uint32_t kWavesOf = E::kDim > 128 || (!GROUPED && E::kDim > 64) ? 4 : 8;
constexpr float kLazyBits = 8.0f;
constexpr float kLn2 = 0.693147180559945309f, kLog2e = 1.44269504088896341f;
constexpr uint32_t kNoId = 0xffffffffu;

// A request's tiles: tile_first .. tile_first + count, the first one holding
// its window's first token.
__device__ __forceinline__ uint32_t tiles_of(uint32_t len, uint32_t window, uint32_t tile, uint32_t& first) {
  first = window_start(len, window) / tile;
  return len ? (len + tile - 1u) / tile - first : 0u;
}

// The line of all tiles: where each request's begin and end. Up to 64
// requests live in a wave's lanes, more of them in LDS.
struct Line {
  uint32_t B, total;
  uint32_t len, upto;      // lane r: request r's length, and the tiles up to and with it
  const uint32_t* starts;  // LDS [B + 1], or null

  // `words`: LDS for the starts and, before them, a word for each wave.
  __device__ __forceinline__ void lay(const AttendArgs& a, uint32_t tile, uint32_t* words, bool& bad) {
    const uint32_t most = a.table_pages * a.page, lane = lane_id();
    uint32_t first;
    B = a.B;
    if (B <= 64u) {
      starts = nullptr;
      len = lane < B ? clamp_len(a.lens[lane], most, bad) : 0u;
      upto = wave_incl_scan(tiles_of(len, a.window, tile, first));
      total = readlane_u32(upto, 63);
      return;
    }
    uint32_t* waves = words;
    uint32_t* start = words + 16;
    const uint32_t wave = threadIdx.x >> 6, n_waves = blockDim.x >> 6;
    total = 0u;
    for (uint32_t r0 = 0; r0 < B; r0 += blockDim.x) {
      const uint32_t r = r0 + threadIdx.x;
      const uint32_t n = r < B ? tiles_of(clamp_len(a.lens[r], most, bad), a.window, tile, first) : 0u;
      const uint32_t sum = wave_incl_scan(n);
      if (lane == 63u) waves[wave] = sum;
      __syncthreads();
      uint32_t before = total;
      for (uint32_t w = 0; w < n_waves; ++w) {
        before += w < wave ? waves[w] : 0u;
        total += waves[w];
      }
      if (r < B) start[r] = before + sum - n;
      __syncthreads();
    }
    if (threadIdx.x == 0u) start[B] = total;
    __syncthreads();
    total = readlane_u32(total, 0);
    starts = start;
  }
  __device__ __forceinline__ uint32_t start(uint32_t r) const {
    if (starts) return readlane_u32(starts[r], 0);
    return r ? readlane_u32(upto, r - 1u) : 0u;
  }
  __device__ __forceinline__ uint32_t end(uint32_t r) const {
    return readlane_u32(starts ? starts[r + 1u] : upto, starts ? 0u : r);
  }
  // The request that holds a tile; for all lanes of a wave.
  __device__ __forceinline__ uint32_t at(uint32_t tile) const {
    if (!starts) return (uint32_t)__builtin_popcountll(__ballot(upto <= tile));
    uint32_t i = 0, above = B;  // the last one that begins at or before it
    while (above - i > 1u) {
      const uint32_t mid = (i + above) >> 1;
      if (starts[mid] <= tile) i = mid;
      else above = mid;
    }
    return readlane_u32(i, 0);
  }
};

// Workgroups go to the 8 XCDs in turn: the number that puts neighbours in
// work on one of them.
__device__ __forceinline__ uint32_t near_block(uint32_t id, uint32_t n) {
  const uint32_t x = id & 7u, rest = n & 7u;
  return x * (n >> 3) + min(x, rest) + (id >> 3);
}

// What joins a request that several ranges share: written by each range
// about the request that came into it (request kNoId: none did).
struct Cut {
  uint32_t request, first, last, unused;
};

// The scales of a group of 8 tokens, of a cache that has one for each block of
// tokens and head, are spread over the group's 16 lanes: lane c < 8 loads that of
// token c's keys, lane 8 + c of its values, and a row broadcast gives all lanes
// what they multiply with. (A load for each token and lane: 64 requests with 4 new
// tokens and a scale for each token 75 us.)
struct GroupScales {
  float next, now;     // of the tile whose keys are loaded, and of the one at hand
  const float* base;   // the cache head's, of the lane's kind
  int64_t stride[2];   // page, block
};
struct NoScales {};
// Lane N's value of each row of 16 lanes.
template <int N>
__device__ __forceinline__ float row_lane(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x150 + N, 0xf, 0xf, true));
}
template <int FIRST>
__device__ __forceinline__ void row_lanes(float x, float* y) {
  y[0] = row_lane<FIRST>(x);
  y[1] = row_lane<FIRST + 1>(x);
  y[2] = row_lane<FIRST + 2>(x);
  y[3] = row_lane<FIRST + 3>(x);
  y[4] = row_lane<FIRST + 4>(x);
  y[5] = row_lane<FIRST + 5>(x);
  y[6] = row_lane<FIRST + 6>(x);
  y[7] = row_lane<FIRST + 7>(x);
}

// Query `qhead` of all of a request's (their number counts a cache head's
// queries, `head`'s begin at first): its row, and its place in the request's
// log-sum-exps. Several new tokens' queries of a cache head are its tokens' one
// after the other.
__device__ __forceinline__ int64_t query_row(const AttendArgs&, const int64_t* stride, int64_t, uint32_t, uint32_t qhead) {
  return (int64_t)qhead * stride[1];
}
__device__ __forceinline__ uint32_t query_lse(const AttendArgs&, uint32_t, uint32_t qhead) { return qhead; }
__device__ __forceinline__ int64_t query_row(const BlockAttendArgs& a, const int64_t* stride, int64_t token_stride, uint32_t head,
                                             uint32_t qhead) {
  const uint32_t i = qhead - head * a.group, token = a.by_per_token.div(i);
  return (int64_t)token * token_stride + (int64_t)(head * a.per_token + (i - token * a.per_token)) * stride[1];
}
__device__ __forceinline__ uint32_t query_lse(const BlockAttendArgs& a, uint32_t head, uint32_t qhead) {
  const uint32_t i = qhead - head * a.group, token = a.by_per_token.div(i);
  return (token * a.heads + head) * a.per_token + (i - token * a.per_token);
}
__device__ __forceinline__ int64_t q_token(const AttendArgs&) { return 0; }
__device__ __forceinline__ int64_t q_token(const BlockAttendArgs& a) { return a.q_token; }
__device__ __forceinline__ int64_t out_token(const AttendArgs&) { return 0; }
__device__ __forceinline__ int64_t out_token(const BlockAttendArgs& a) { return a.out_token; }

// GROUPED: pages are whole groups of tokens. ONCE: values are not found in a
// cache again.
template <class E, bool GROUPED, bool ONCE>
struct Run {
  static_assert(GROUPED || !E::kWhole, "no call has such pages");
  static constexpr int kIds = GROUPED ? 1 : E::kGroup;       // page ids of the lane's V tokens
  static constexpr int kKIds = GROUPED ? 1 : E::kProducts;   // and of its K tokens
  const typename E::Args& a;
  const int32_t* row;   // the request's table
  const char* base[2];  // the pools at the cache head
  uint32_t g, c, lo, hi;  // the lane, and the tokens that are seen
  float scale;            // of a score, in base-2 exponents
  E e;
  float ref, limit, sum = 0.0f;  // m (0 before the first finite score), what no score passes, the lane's part of l
  bool far = false;  // some |m| is 2^20 or more
  bool bad = false;
  enum { kAllValues, kFinite, kInfinite, kNoNumbers } values = kAllValues;  // which ones a pass adds
  struct PlainIds {
    uint32_t k[kKIds], v[kIds];
  };
  struct ScaledIds : PlainIds {
    uint32_t scale;  // of the token whose scale the lane loads
  };
  using Ids = std::conditional_t<E::kBlocks && !GROUPED, ScaledIds, PlainIds>;

  std::conditional_t<E::kBlocks, GroupScales, NoScales> scales;
  int lane_lo, lane_hi;  // kBlocks: the tokens that the lane's query sees

  __device__ __forceinline__ Run(const typename E::Args& args) : a(args) {}

  // First of the lane's tokens in a tile: V's group, and K's in product p.
  __device__ __forceinline__ uint32_t v_token(uint32_t t0) const { return t0 + E::kGroup * g; }
  __device__ __forceinline__ uint32_t k_token(uint32_t t0, uint32_t p) const {
    return t0 + E::kGroup * (c >> 2) + 4u * p + (c & 3u);
  }

  // Page id of token t, or of the nearest one that is seen: always a load, so
  // that the compiler can count the loads behind it when it waits.
  __device__ __forceinline__ uint32_t page_id(uint32_t t) const {
    return (uint32_t)row[a.by_page.div(min(max(t, lo), hi - 1u))];
  }
  __device__ __forceinline__ Ids fetch_ids(uint32_t t0) const {
    Ids x;
#pragma unroll
    for (int p = 0; p < kKIds; ++p) x.k[p] = page_id(k_token(t0, p));
#pragma unroll
    for (int i = 0; i < kIds; ++i) x.v[i] = page_id(v_token(t0) + i);
    if constexpr (E::kBlocks && !GROUPED) x.scale = page_id(v_token(t0) + (c & 7u));
    return x;
  }

  // Where a token of page id starts; an id outside the pool leads to its
  // first page (seen_of drops the token).
  __device__ __forceinline__ const char* token_row(int pool, uint32_t id, uint32_t in_page) const {
    id = id < a.pages ? id : 0u;
    return base[pool] + ((int64_t)id * a.pool_stride[pool][0] + (int64_t)in_page * a.pool_stride[pool][1]) * E::kElem;
  }
  __device__ __forceinline__ void load_keys(uint32_t t0, const Ids& x) {
#pragma unroll
    for (int p = 0; p < E::kProducts; ++p) {
      const uint32_t t = k_token(t0, p);
      e.load_k(p, token_row(0, x.k[GROUPED ? 0 : p], a.by_page.mod(t)), g, a.dim);
    }
  }
  __device__ __forceinline__ void load_values(uint32_t t0, const Ids& x) {
    const uint32_t t = v_token(t0);
    if constexpr (GROUPED) {
      const char* p = token_row(1, x.v[0], a.by_page.mod(t));
      const int64_t step = a.pool_stride[1][1] * E::kElem;
#pragma unroll
      for (int i = 0; i < E::kGroup; ++i) e.template load_v<ONCE>(i, p + i * step, c, a.dim);
    } else {
#pragma unroll
      for (int i = 0; i < E::kGroup; ++i) e.template load_v<ONCE>(i, token_row(1, x.v[i], a.by_page.mod(t + i)), c, a.dim);
    }
  }
  __device__ __forceinline__ void load_scales(uint32_t t0, const Ids& ids) {
    if constexpr (E::kBlocks) {
      uint32_t id, t;
      if constexpr (GROUPED) {
        id = ids.v[0];
        t = a.by_page.mod(v_token(t0)) + (E::kEach ? c & 7u : 0u);
      } else {
        id = ids.scale;
        t = a.by_page.mod(v_token(t0) + (c & 7u));
      }
      scales.next = scales.base[(int64_t)(id < a.pages ? id : 0u) * scales.stride[0] +
                                (int64_t)a.block_scales.by_block.div(t) * scales.stride[1]];
    }
  }
  // Which of the lane's tokens are seen, as bits; kAll in every lane of most
  // tiles. kBlocks: by the lane's query, and above those bits by any query.
  static constexpr uint32_t kAll = (1u << (E::kBlocks ? 2 : 1) * E::kGroup) - 1u;
  __device__ __forceinline__ uint32_t seen_of(uint32_t t0, const Ids& x) {
    bool outside = t0 < lo || t0 + E::kTile > hi;
    if constexpr (E::kBlocks) outside = (int)t0 < lane_lo || (int)(t0 + E::kTile) > lane_hi || outside;
#pragma unroll
    for (int i = 0; i < kIds; ++i) outside = outside || x.v[i] >= a.pages;
    if (!__any(outside)) return kAll;
    uint32_t seen = 0u;
#pragma unroll
    for (int i = 0; i < E::kGroup; ++i) {
      const uint32_t t = v_token(t0) + i, id = x.v[GROUPED ? 0 : i];
      const bool in = t >= lo && t < hi;
      bad = bad || (in && id >= a.pages);
      if constexpr (E::kBlocks) {
        seen |= in && id < a.pages ? 1u << (E::kGroup + i) : 0u;
        seen |= in && id < a.pages && (int)t >= lane_lo && (int)t < lane_hi ? 1u << i : 0u;
      } else {
        seen |= in && id < a.pages ? 1u << i : 0u;
      }
    }
    return seen;
  }

  // Tiles first .. last of the request, at least one. A tile's keys are loaded
  // when the tile before has used its own, its values likewise, and its page
  // ids two tiles ahead, so that no wait for one of them includes a younger
  // load. The last tile loads itself again (from the L2): a branch around the
  // loads would make every wait one for all of them.
  __device__ __forceinline__ void tiles(uint32_t first, uint32_t last) {
    const float before = sum;
    if (!E::kInfinities || values != kInfinite) {
      ref = 0.0f;
      far = false;
      limit = E::kNaNs && values == kNoNumbers ? INFINITY : -INFINITY;  // (marks are not scaled)
      sum = 0.0f;
      if (!E::kNaNs || values != kFinite) e.clear();
    }
    uint32_t t0 = readlane_u32(first, 0) * E::kTile;  // (the same in every lane: the loop's branch is the wave's)
    const uint32_t t_last = (readlane_u32(last, 0) - 1u) * E::kTile;
    const Ids now = fetch_ids(t0);
    Ids next = fetch_ids(min(t0 + E::kTile, t_last));
    load_keys(t0, now);
    load_scales(t0, now);
    load_values(t0, now);
    uint32_t seen = seen_of(t0, now);
    bool more;
    do {
      more = t0 != t_last;
      float s[E::kGroup];
      e.scores(s, g, a.dim);
      const uint32_t t1 = min(t0 + E::kTile, t_last);
      const Ids after = fetch_ids(min(t0 + 2u * E::kTile, t_last));
      load_keys(t1, next);
      if constexpr (E::kBlocks) {
        scales.now = scales.next;
        load_scales(t1, next);
      }
      add(s, seen);
      load_values(t1, next);
      seen = seen_of(t1, next);
      next = after;
      t0 = t1;
    } while (more);
    if (E::kInfinities && values == kInfinite) sum = before;
  }

  // Whether the tiles have to be read again, for sums that are not finite. Of
  // infinite values a second pass adds the finite values alone, a third the others,
  // which their signs decide. Of several new tokens' queries, which do not see
  // the same tokens, and values that are no numbers (0 times one is none) a second
  // pass counts for each query those that it sees, and a third adds the numbers
  // to NaN where there is one, to 0 elsewhere.
  __device__ __forceinline__ bool again() {
    if constexpr (E::kInfinities) {
      if (__builtin_expect(values != kAllValues || __any(e.infinite()), 0)) {
        values = values == kAllValues ? kFinite : values == kFinite ? kInfinite : kAllValues;
        return values != kAllValues;
      }
    }
    if constexpr (E::kNaNs) {
      if (__builtin_expect(values != kAllValues || (a.tokens > 1u && __any(e.infinite())), 0)) {
        if (values == kNoNumbers) e.spoil();
        values = values == kAllValues ? kNoNumbers : values == kNoNumbers ? kFinite : kAllValues;
        return values != kAllValues;
      }
    }
    return false;
  }

  // A tile's scores and values into ref, sum and o.
  __device__ __forceinline__ void add(float* s, uint32_t seen) {
    // What each token's score is multiplied with, and its numerator.
    float k_scale[E::kGroup], v_scale[E::kGroup];
    if constexpr (E::kBlocks) {
      if constexpr (E::kEach) {
        row_lanes<0>(scales.now, k_scale);
        row_lanes<8>(scales.now, v_scale);
#pragma unroll
        for (int i = 0; i < E::kGroup; ++i) k_scale[i] *= scale;
      } else {
        const float x = row_lane<0>(scales.now) * scale, y = row_lane<8>(scales.now);
#pragma unroll
        for (int i = 0; i < E::kGroup; ++i) {
          k_scale[i] = x;
          v_scale[i] = y;
        }
      }
    }
    const auto scale_of = [&](int i) {
      if constexpr (E::kBlocks) return k_scale[i];
      else return scale;
    };
    const bool edge = __any(seen != kAll) || ((E::kInfinities || E::kNaNs) && values != kAllValues);
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < E::kGroup; ++i) {
      const float x = s[i] * scale_of(i);
      top = fmaxf(top, !edge || (seen >> i & 1u) ? x : -INFINITY);
    }
    if (__any(top > limit)) raise(top);
    // The scaled score is not rounded before the reference is taken from it:
    // only the difference is, and that is small where it counts. The reference
    // is a rounded one, so the largest difference is as far from 0 as half of
    // its last bit: far references take the rounded scores' difference, which
    // is exact there.
    if (__builtin_expect(far, 0)) {
#pragma unroll
      for (int i = 0; i < E::kGroup; ++i) {
        s[i] = s[i] * scale_of(i) - ref;
        // (The limit is rounded too: by a last bit of 16 to past the largest F16.)
        if (E::kLift > 0.0f) s[i] = s[i] > E::kLift + kLazyBits ? E::kLift + kLazyBits : s[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < E::kGroup; ++i) s[i] = __builtin_fmaf(s[i], scale_of(i), -ref);
    }
#pragma unroll
    for (int i = 0; i < E::kGroup; ++i) s[i] = __builtin_amdgcn_exp2f(s[i]);
    if (edge) {
#pragma unroll
      for (int i = 0; i < E::kGroup; ++i) {
        const bool keep = seen >> i & 1u;
        s[i] = keep ? s[i] : 0.0f;
        if constexpr (E::kBlocks) {
          // (Whole numbers are finite whatever a place holds.)
          const bool any = seen >> (E::kGroup + i) & 1u;
          if constexpr (!std::is_same_v<typename E::KV, I8>) e.keep_v(i, any);
          v_scale[i] = any ? v_scale[i] : 0.0f;  // (of a block that no call has written it may be no number)
        } else {
          e.keep_v(i, keep);
        }
      }
      if constexpr (E::kInfinities) {
        if (__builtin_expect(values != kAllValues, 0)) {
#pragma unroll
          for (int i = 0; i < E::kGroup; ++i) {
            // A numerator above 0 whose two parts are.
            if (values == kInfinite) s[i] = s[i] > 0.0f ? 1.0f + 0x1p-12f : s[i];
            e.keep_finite(i, values == kFinite);
          }
        }
      }
      if constexpr (E::kNaNs) {
        if (__builtin_expect(values != kAllValues, 0)) {
#pragma unroll
          for (int i = 0; i < E::kGroup; ++i) {
            const bool marks = values == kNoNumbers;
            e.keep_numbers(i, marks);
            s[i] = marks ? (seen >> i & 1u ? 1.0f : 0.0f) : s[i];
            v_scale[i] = marks ? 1.0f : v_scale[i];
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < E::kGroup; ++i) sum += s[i];
    if constexpr (E::kBlocks) {
#pragma unroll
      for (int i = 0; i < E::kGroup; ++i) s[i] *= v_scale[i];
    }
    e.accumulate(s);
  }

  // Moves the reference of each query head to its largest score.
  __device__ __forceinline__ void raise(float top) {
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float low = top - E::kLift;
    const bool fresh = limit == -INFINITY, up = low > (fresh ? -INFINITY : ref);
    const float next = up ? low : ref;
    const float keep = fresh || !up ? 1.0f : __builtin_amdgcn_exp2f(ref - next);
    ref = next == INFINITY ? NAN : next;  // (past binary32: no weight of 0, but NaN)
    far = __any(fabsf(ref) >= 0x1p20f);
    limit = up || !fresh ? next + (E::kLift + kLazyBits) : -INFINITY;
    sum *= keep;
    f32x4 k;
#pragma unroll
    for (int i = 0; i < 4; ++i) k[i] = __shfl(keep, 4 * g + i, 64);
#pragma unroll
    for (int p = 0; p < E::kPanels; ++p)
#pragma unroll
      for (int j = 0; j < E::kVec; ++j) e.o[p][j] *= k;
  }

  __device__ __forceinline__ float total() const {
    float l = sum + __shfl_xor(sum, 16, 64);
    return l + __shfl_xor(l, 32, 64);
  }
};

__device__ __forceinline__ float lse_of(float m, float l) {
  return l == 0.0f ? -INFINITY : kLn2 * (m + __builtin_amdgcn_logf(l));
}

template <class E, bool GROUPED, bool ONCE>
__device__ __forceinline__ void attend(typename E::Args a) {
  constexpr uint32_t kWaves = kWavesOf<E, GROUPED>;
  extern __shared__ __attribute__((aligned(16))) uint32_t s_mem[];
  __shared__ int32_t s_slot[2 * kWaves];  // the request of each partial answer, or -1
  float* s_part = reinterpret_cast<float*>(s_mem + a.start_words);

  const uint32_t tid = threadIdx.x, lane = lane_id(), wave = readlane_u32(tid >> 6, 0);
  // Heads whose rows are no whole cache lines share lines with their
  // neighbours, and then an L2.
  const uint32_t block = a.dim * E::kElem % 128u ? near_block(blockIdx.x, gridDim.x) : blockIdx.x;
  const uint32_t teams = a.vheads / a.team, range = block / teams;
  const uint32_t mate = wave % a.team, share = wave / a.team;  // the wave's head in the team, and its part of the range
  const uint32_t vhead = block % teams * a.team + mate;
  const uint32_t head = vhead / a.blocks, q0 = vhead % a.blocks * 16u;  // first query head inside the group
  const uint32_t group = min(16u, a.group - q0);
  const uint32_t most = a.table_pages * a.page;
  bool bad = false;

  // The range of tiles: [begin, end) of the line, or one request's.
  Line line;
  uint32_t begin, end, quota = 1u, b = range;
  if (a.ranges) {
    line.lay(a, E::kTile, s_mem, bad);
    quota = max((line.total + a.ranges - 1u) / a.ranges, a.splits);
    begin = min(range * quota, line.total);
    end = min(begin + quota, line.total);
  } else {
    uint32_t first;
    begin = 0u;
    end = tiles_of(clamp_len(a.lens[b], most, bad), a.window, E::kTile, first);
  }
  // (Any wave may hold the bad length: each lays out a part of a long line.)
  if (bad && block % teams == 0u && (range == 0u || !a.ranges)) atomicOr(a.status, LLMHIP_KSTATUS_BAD_INDEX);

  Run<E, GROUPED, ONCE> run(a);
  run.g = lane >> 4;
  run.c = lane & 15u;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    run.base[i] = static_cast<const char*>(a.pool[i]) + (int64_t)head * a.pool_stride[i][2] * E::kElem;
  const bool e4m3 = E::KV::kId == LLMHIP_E4M3 && !E::kBlocks;  // (blocks: the scales are the tokens')
  run.scale = a.score_scale * kLog2e * (e4m3 ? a.scale[0][head] : 1.0f);
  const float vscale = e4m3 ? a.scale[1][head] : 1.0f;
  if constexpr (E::kBlocks) {
    const int kind = run.c >= 8u;
    run.scales.base = (kind ? a.block_scales.scale[1] : a.block_scales.scale[0]) +
                      (int64_t)head * (kind ? a.block_scales.stride[1][2] : a.block_scales.stride[0][2]);
#pragma unroll
    for (int i = 0; i < 2; ++i) run.scales.stride[i] = kind ? a.block_scales.stride[1][i] : a.block_scales.stride[0][i];
  }
  const uint32_t qhead = head * a.group + q0;  // the first of the output
  const auto out_of = [&](uint32_t r, uint32_t qi) {
    return static_cast<typename E::Q::Raw*>(a.out) + (int64_t)r * a.out_stride[0] +
           query_row(a, a.out_stride, out_token(a), head, qhead + qi);
  };
  const auto lse_at = [&](uint32_t r, uint32_t qi) {
    if constexpr (E::kBlocks) return a.lse + (uint64_t)r * a.q_heads + query_lse(a, head, qhead + qi);
    else return a.lse + (uint64_t)r * a.q_heads + qhead + qi;
  };

  const auto partial_of = [&](bool before) {
    return a.workspace + a.part_offset + (((uint64_t)range * a.vheads + vhead) * 2u + (before ? 0u : 1u)) * a.part_words;
  };
  const auto put_partial = [&](float* part, float m, float l) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t qi = 4u * run.g + i;
      if (qi >= group) continue;
#pragma unroll
      for (uint32_t p = 0; p < E::kPanels; ++p) {
        const uint32_t d = (p * 16u + run.c) * E::kVec;
        if (d >= a.dim) continue;
        // (In stores of 16 bytes, or 8: the compiler joins none, and 16 queries of
        // 64 requests, over whole numbers, take 66 us then, not 60.)
        using Store = float __attribute__((ext_vector_type(E::kVec < 4 ? E::kVec : 4)));
        constexpr int kEach = sizeof(Store) / 4;
#pragma unroll
        for (int j = 0; j < E::kVec; j += kEach) {
          Store x;
#pragma unroll
          for (int k = 0; k < kEach; ++k) x[k] = run.e.o[p][j + k][i];
          *reinterpret_cast<Store*>(part + qi * a.dim + d + j) = x;
        }
      }
    }
    if (lane < group) {
      part[group * a.dim + lane] = m;
      part[group * (a.dim + 1u) + lane] = l;
    }
  };

  const uint32_t tiles = end - begin, part = tiles / a.splits, over = tiles - part * a.splits;  // (no product passes 32 bits)
  uint32_t tile = begin + part * share + over * share / a.splits, slot = 2u * wave;
  const uint32_t stop = begin + part * (share + 1u) + over * (share + 1u) / a.splits;
  if (a.splits > 1u && lane < 2u) s_slot[slot + lane] = -1;
  if (a.ranges && tile < stop) b = line.at(tile);
  while (tile < stop) {
    const uint32_t from = a.ranges ? line.start(b) : 0u, to = a.ranges ? line.end(b) : end;
    if (to <= tile) {  // an empty request
      ++b;
      continue;
    }
    bool clamped = false;
    const uint32_t len =
        a.ranges && !line.starts ? readlane_u32(line.len, b) : readlane_u32(clamp_len(a.lens[b], most, clamped), 0);
    uint32_t zero_tile;
    tiles_of(len, a.window, E::kTile, zero_tile);
    const uint32_t last = min(stop, to);
    run.row = a.table + (uint64_t)b * a.table_ld;
    run.lo = window_start(len, a.window);
    run.hi = len;
    if constexpr (E::kBlocks) {
      run.lane_hi = (int)len + 1 - (int)a.tokens + (int)a.by_per_token.div(q0 + min(run.c, group - 1u));
      run.lane_lo = a.seen_window ? max(run.lane_hi - (int)a.seen_window, 0) : 0;
    }
    const typename E::Q::Raw* q = static_cast<const typename E::Q::Raw*>(a.q) + (int64_t)b * a.q_stride[0] +
                                  query_row(a, a.q_stride, q_token(a), head, qhead + (run.c < group ? run.c : 0u));
    run.e.load_q(q, run.g, a.dim, run.c < group);
    run.tiles(zero_tile + (tile - from), zero_tile + (last - from));
    if (run.again()) continue;
    const float l = run.total(), m = l == 0.0f ? -INFINITY : run.ref;
    if (tile == from && last == to) {  // all of the request
      const float inv = l == 0.0f ? 0.0f : vscale / l;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t qi = 4u * run.g + i;
        const float scale = __shfl(inv, qi, 64);
        if (qi >= group) continue;
        typename E::Q::Raw* out = out_of(b, qi);
#pragma unroll
        for (uint32_t p = 0; p < E::kPanels; ++p) {
          const uint32_t d = (p * 16u + run.c) * E::kVec;
          if (d >= a.dim) continue;
          Pack<typename E::Q, E::kVec> x;
#pragma unroll
          for (int j = 0; j < E::kVec; ++j) x.v[j] = E::Q::store(run.e.o[p][j][i] * scale);
          __builtin_memcpy(out + d, x.v, sizeof x.v);
        }
      }
      if (a.lse && lane < group) *lse_at(b, lane) = lse_of(m, l);
    } else if (a.splits > 1u) {
      put_partial(s_part + slot * a.part_words, m, l);
      if (lane == 0u) s_slot[slot] = (int32_t)b;
      ++slot;  // a wave leaves two at most: one that came in, one that goes on
    } else {
      put_partial(partial_of(from < begin), m, l);
    }
    tile = last;
    ++b;
  }
  if (__any(run.bad) && lane == 0u) atomicOr(a.status, LLMHIP_KSTATUS_BAD_INDEX);

  // Requests of length 0: a range has every ranges-th one.
  const auto empty = [&](uint32_t r) {
    for (uint32_t x = lane; x < group * a.dim; x += 64u) {
      const uint32_t qi = a.by_dim.div(x), d = x - qi * a.dim;
      out_of(r, qi)[d] = E::Q::store(0.0f);
      if (a.lse && d == 0u) *lse_at(r, qi) = -INFINITY;
    }
  };
  if (a.ranges) {
    for (uint32_t r = range + share * a.ranges; r < a.B; r += a.splits * a.ranges)
      if (line.start(r) == line.end(r)) empty(r);
    // For the join: the request that came into this range, and its ranges.
    if (vhead == 0u && share == 0u) {
      Cut cut = {kNoId, 0u, 0u, 0u};
      if (begin < end) {
        const uint32_t r = line.at(begin);
        if (line.start(r) < begin) cut = {r, line.start(r) / quota, (line.end(r) - 1u) / quota, 0u};
      }
      if (lane == 0u) reinterpret_cast<Cut*>(a.workspace)[range] = cut;
    }
  } else if (end == 0u && share == 0u) {
    empty(b);
  }
  if (a.splits == 1u) return;
  __syncthreads();

  // Join the partial answers of each request of the wave's head: one of each
  // share at most, all read at once (a missing one stands for the first
  // again, with weight 0). The head's waves do this together. At most two of
  // its requests go on outside the range.
  const int32_t holds = lane < 2u * a.splits ? s_slot[2u * ((lane >> 1) * a.team + mate) + (lane & 1u)] : -1;
  uint64_t rest = __ballot(holds >= 0);
  while (rest) {
    const uint32_t r = readlane_u32((uint32_t)holds, (uint32_t)__builtin_ctzll(rest));
    const uint64_t parts = __ballot(holds == (int32_t)r);
    rest &= ~parts;
    const auto part_at = [&](uint32_t i) { return s_part + (2u * ((i >> 1) * a.team + mate) + (i & 1u)) * a.part_words; };
    const uint32_t n = (uint32_t)__builtin_popcountll(parts);
    uint64_t set = parts;
    const float* part[kWaves];
#pragma unroll
    for (uint32_t k = 0; k < kWaves; ++k) {
      part[k] = k < n ? part_at((uint32_t)__builtin_ctzll(set)) : part[0];
      set &= set - 1u;
    }
    const bool before = a.ranges && line.start(r) < begin, after = a.ranges && line.end(r) > end;
    float* to = partial_of(before);
    for (uint32_t x = share * 64u + lane; x < group * a.dim; x += a.splits * 64u) {
      const uint32_t qi = a.by_dim.div(x), d = x - qi * a.dim, at_m = group * a.dim + qi, at_l = at_m + group;
      float m = -INFINITY, l = 0.0f, o = 0.0f, w[kWaves];
#pragma unroll
      for (uint32_t k = 0; k < kWaves; ++k) {
        w[k] = k < n ? part[k][at_m] : -INFINITY;
        m = fmaxf(m, w[k]);
      }
      const float top = m == -INFINITY ? 0.0f : m;
#pragma unroll
      for (uint32_t k = 0; k < kWaves; ++k) {
        w[k] = __builtin_amdgcn_exp2f(w[k] - top);
        l += part[k][at_l] * w[k];
        o += part[k][x] * w[k];
      }
      if (__builtin_expect(!isfinite(o), 0)) {  // without the missing parts: 0 times an infinite sum is NaN
        o = 0.0f;
        for (uint64_t left = parts; left; left &= left - 1u) {
          const float* p = part_at((uint32_t)__builtin_ctzll(left));
          o += p[x] * __builtin_amdgcn_exp2f(p[at_m] - top);
        }
      }
      if (before || after) {
        to[x] = o;
        if (d == 0u) {
          to[at_m] = m;
          to[at_l] = l;
        }
      } else {
        const float inv = l == 0.0f ? 0.0f : vscale / l;
        out_of(r, qi)[d] = E::Q::store(o * inv);
        if (a.lse && d == 0u) *lse_at(r, qi) = lse_of(m, l);
      }
    }
  }
}

template <class E, bool GROUPED, bool ONCE>
__global__ __launch_bounds__((kWavesOf<E, GROUPED> * 64)) void attend_kernel(AttendArgs a) {
  attend<E, GROUPED, ONCE>(a);
}
template <class E, bool GROUPED, bool ONCE>
__global__ __launch_bounds__((kWavesOf<E, GROUPED> * 64)) void block_attend_kernel(BlockAttendArgs a) {
  attend<E, GROUPED, ONCE>(a);
}

// The answers of requests that several ranges share. Row y of the grid is the
// boundary before range y + 1. All boundaries inside a request take equal
// parts of its value quads (of all query heads), so that a request of more
// parts has more workgroups; in a workgroup neighbouring threads take
// neighbouring quads, and where that leaves threads over, they take other
// parts of the same quads. The order of joining follows from the number of
// parts alone.
template <class Q, class KV, class Args>
__global__ __launch_bounds__(256) void join_kernel(Args a) {
  constexpr uint32_t kBatch = 8;
  __shared__ float s_m[256], s_l[256];
  __shared__ f32x4 s_o[256];
  const Cut cut = reinterpret_cast<const Cut*>(a.workspace)[blockIdx.y + 1u];
  if (cut.request == kNoId) return;
  const uint32_t tid = threadIdx.x, n = cut.last - cut.first + 1u, quads = a.q_heads * (a.dim / 4u);
  const uint32_t groups = (n - 1u) * gridDim.x, mine = (blockIdx.y - cut.first) * gridDim.x + blockIdx.x;
  uint32_t width = 8u;  // quads of a workgroup: a power of 2
  while (width < 256u && width * groups < quads) width *= 2u;
  const uint32_t quad = mine * width + (tid & (width - 1u)), shares = 256u / width, share = tid / width;
  if (mine * width >= quads) return;
  const uint32_t x = min(quad, quads - 1u) * 4u, qh = a.by_dim.div(x), d = x - qh * a.dim;
  const uint32_t head = qh / a.group, in_group = qh % a.group, vhead = head * a.blocks + in_group / 16u;
  const uint32_t group = min(16u, a.group - in_group / 16u * 16u), qi = in_group % 16u;
  const uint32_t at_o = qi * a.dim + d, at_m = group * a.dim + qi, at_l = at_m + group;
  const auto part_at = [&](uint32_t k) {
    return a.workspace + a.part_offset + (((uint64_t)(cut.first + k) * a.vheads + vhead) * 2u + (k ? 0u : 1u)) * a.part_words;
  };
  float m = -INFINITY, l = 0.0f;
  f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  for (uint32_t k0 = share; k0 < n; k0 += kBatch * shares) {
    float pm[kBatch], pl[kBatch];
    f32x4 po[kBatch];
#pragma unroll
    for (uint32_t j = 0; j < kBatch; ++j) {  // (the first one again where there is no more)
      const uint32_t k = k0 + j * shares < n ? k0 + j * shares : k0;
      const float* part = part_at(k);
      pm[j] = part[at_m];
      pl[j] = part[at_l];
      po[j] = *reinterpret_cast<const f32x4*>(part + at_o);
    }
    float next = m;
#pragma unroll
    for (uint32_t j = 0; j < kBatch; ++j) {
      pm[j] = k0 + j * shares < n ? pm[j] : -INFINITY;
      next = fmaxf(next, pm[j]);
    }
    const float top = next == -INFINITY ? 0.0f : next, keep = __builtin_amdgcn_exp2f(m - top);
    o *= keep;
    l *= keep;
#pragma unroll
    for (uint32_t j = 0; j < kBatch; ++j) {
      const float w = __builtin_amdgcn_exp2f(pm[j] - top);
      l += pl[j] * w;
      o += po[j] * w;
    }
    m = next;
  }
  if (__builtin_expect(!isfinite((o[0] + o[1]) + (o[2] + o[3])), 0)) {  // without the missing parts: 0 times an infinite sum is NaN
    o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t k = share; k < n; k += shares) {
      const float* part = part_at(k);
      o += *reinterpret_cast<const f32x4*>(part + at_o) * __builtin_amdgcn_exp2f(part[at_m] - (m == -INFINITY ? 0.0f : m));
    }
  }
  if (shares > 1u) {
    s_m[tid] = m;
    s_l[tid] = l;
    s_o[tid] = o;
    __syncthreads();
    if (share) return;
    float top = m;
    for (uint32_t k = 1; k < shares; ++k) top = fmaxf(top, s_m[k * width + tid]);
    const float whole = top;
    top = top == -INFINITY ? 0.0f : top;
    const float keep = __builtin_amdgcn_exp2f(m - top);
    l *= keep;
    o *= keep;
    for (uint32_t k = 1; k < shares; ++k) {
      const float w = __builtin_amdgcn_exp2f(s_m[k * width + tid] - top);
      l += s_l[k * width + tid] * w;
      o += s_o[k * width + tid] * w;
    }
    m = whole;
  }
  if (quad >= quads) return;
  const bool scaled = KV::kId == LLMHIP_E4M3 && std::is_same_v<Args, AttendArgs>;
  const float vscale = scaled ? a.scale[1][head] : 1.0f, inv = l == 0.0f ? 0.0f : vscale / l;
  Pack<Q, 4> y;
#pragma unroll
  for (int j = 0; j < 4; ++j) y.v[j] = Q::store(o[j] * inv);
  typename Q::Raw* out = static_cast<typename Q::Raw*>(a.out) + (int64_t)cut.request * a.out_stride[0] +
                         query_row(a, a.out_stride, out_token(a), head, qh) + d;
  __builtin_memcpy(out, y.v, sizeof y.v);
  if (a.lse && d == 0u) a.lse[(uint64_t)cut.request * a.q_heads + query_lse(a, head, qh)] = lse_of(m, l);
}

template <class E, bool GROUPED, bool ONCE>
hipError_t launch_attend_group(typename E::Args a, hipStream_t s) {
  constexpr uint32_t kWaves = kWavesOf<E, GROUPED>;
  const AttendSplit split = attend_split(kWaves, E::kTile, a.dim * 2u * E::kElem, a.cus, a.B, a.vheads, a.table_pages * a.page, a.window);
  a.team = split.team;
  a.splits = split.splits;
  a.ranges = split.ranges;
  const uint32_t teams = a.vheads / a.team;
  a.start_words = a.ranges && a.B > 64u ? 16u + (a.B + 1u + 3u) / 4u * 4u : 0u;
  const uint32_t lds = (a.start_words + (a.splits > 1u ? 2u * kWaves * a.part_words : 0u)) * 4u;
  const dim3 grid((a.ranges ? a.ranges : a.B) * teams), threads(a.team * a.splits * 64u);
  if constexpr (E::kBlocks) hipLaunchKernelGGL((block_attend_kernel<E, GROUPED, ONCE>), grid, threads, lds, s, a);
  else hipLaunchKernelGGL((attend_kernel<E, GROUPED, ONCE>), grid, threads, lds, s, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.ranges < 2u) return e;
  const uint32_t quads = a.q_heads * (a.dim / 4u);
  hipLaunchKernelGGL((join_kernel<typename E::Q, typename E::KV, typename E::Args>), dim3((quads + 255u) / 256u, a.ranges - 1u), dim3(256), 0, s, a);
  return hipGetLastError();
}

template <class E, bool ONCE>
hipError_t launch_attend_pages(const typename E::Args& a, hipStream_t s) {
  if constexpr (!E::kWhole) {
    if (a.page % E::kGroup) return launch_attend_group<E, false, ONCE>(a, s);
  }
  return launch_attend_group<E, true, ONCE>(a, s);
}

// Values are read past the caches unless the next call may find them there (the
// card keeps 256 MB: pools of up to 64 MiB each), or the heads beside them on
// their cache lines do. 537 MB 96 us and 102 with plain loads, 2.2 GB of E4M3 346
// and 379; 67 MB of one head 26.4 and 24.9, 205 MB of rows of 32 bytes 89 and 75.
template <class E>
hipError_t launch_attend_engine(const typename E::Args& a, hipStream_t s) {
  if constexpr (E::kDim == 32) {
    return launch_attend_pages<E, false>(a, s);
  } else {
    const uint64_t pool = (uint64_t)a.pages * a.page * a.heads * a.dim * E::kElem;
    if constexpr (E::kBlocks) {
      // (Nor where a cache head has more queries than the matrix cores take at once,
      // whose waves read the same rows. 16 calls of 1 to 256 requests with 20 to 128 queries
      // a cache head, both types of codes, 1 to 12 heads of 64 to 256, pools of 17 to 543
      // MB: 0.94 of the time past the caches in the mean, 0.79 to 1.03; 135 requests of 1656
      // tokens with 20 for each of 8 heads of 112 164 us and 196, one of 131072 with 32
      // for each of 8 heads of 128 82 and 83.)
      const bool once = pool > (64u << 20) && a.blocks == 1u;
      return once ? launch_attend_pages<E, true>(a, s) : launch_attend_pages<E, false>(a, s);
    } else {
      if (a.page % E::kGroup) return launch_attend_group<E, false, true>(a, s);
      return pool > (64u << 20) ? launch_attend_group<E, true, true>(a, s) : launch_attend_group<E, true, false>(a, s);
    }
  }
}

// ENGINE<DIM, FULL>: the smallest DIM that holds head_dim. (Its name is part of
// this function's symbol: each source needs one of its own.)
template <template <int, bool> class ENGINE, class Args = AttendArgs>
hipError_t launch_attend_dims(const Args& a, hipStream_t s) {
  if (a.dim == 64u) return launch_attend_engine<ENGINE<64, true>>(a, s);
  if (a.dim == 128u) return launch_attend_engine<ENGINE<128, true>>(a, s);
  if (a.dim <= 32u) return launch_attend_engine<ENGINE<32, false>>(a, s);
  if (a.dim < 64u) return launch_attend_engine<ENGINE<64, false>>(a, s);
  if (a.dim <= 96u) return launch_attend_engine<ENGINE<96, false>>(a, s);
  if (a.dim < 128u) return launch_attend_engine<ENGINE<128, false>>(a, s);
  if (a.dim <= 192u) return launch_attend_engine<ENGINE<192, false>>(a, s);
  return launch_attend_engine<ENGINE<256, false>>(a, s);
}

}  // namespace llmhip
