// New tokens' keys and values, quantised, into their slots, and their queries
// rotated (llmhip_kv_block_append).
//
// A block's scale needs the largest of its new values before the first code
// can be written. A workgroup finds the blocks that begin among some tokens (their
// slots say so; as many as a block has, 16 to 64) and gives each block and head
// as many neighbouring lanes as hold all of its new values in registers: 8 for a
// decoding request's single row of 128 values, all 256 for 64 of them. The maximum
// goes across those lanes, and codes are written. Of blocks that are larger the
// rows are read again, from the L2. So a value comes from memory once. Cosines and
// sines are computed once for all heads of a workgroup, into LDS. Kept tokens are
// read only where the scale grew. Units are laid out as in the append to a cache
// of values: 2 * VEC values of a row, VEC pairs, or values that are not rotated.
//
// What bounds it: for few tokens the chain slots, rows, maximum, codes (256
// tokens 7.2 us where no block's scale grows); for many the traffic, 368 MB of 16384
// tokens in 78 us, 4.7 TB/s, of which the vector units are busy for 47. A scale that
// grows costs a read and a write of its block's kept codes, 8 at a time by the
// task's lanes one after the other: of 256 single tokens in the middle of their
// blocks of 16 22 us where all grow, 27 where a fifth do. Prompts, whose blocks begin
// in the call but for a few, take the same time either way.
#include <algorithm>

#include "kv_args.h"
#include "kv_block_tasks.h"
#include "kv_turn.h"
#include "kv_types.h"
#include "wave_ops.h"

namespace llmhip {
namespace {

constexpr uint32_t kThreads = kAppendThreads;
constexpr uint32_t kMaxGroup = 64;  // of one of keys or values: a lane's each

template <int VEC>
constexpr uint32_t kHeld = append_held(VEC);

template <int BYTES>
struct Word;
template <> struct Word<1> { using type = uint8_t; };
template <> struct Word<2> { using type = uint16_t; };
template <> struct Word<4> { using type = uint32_t; };
template <> struct Word<8> { using type = uint32_t __attribute__((ext_vector_type(2))); };
template <> struct Word<16> { using type = uint32_t __attribute__((ext_vector_type(4))); };

// Rows of any alignment.
template <class T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const typename T::Raw* p) {
  Pack<T, N> x;
  __builtin_memcpy(&x, p, sizeof x);
  return x;
}
// Past the L2: written once, read by later kernels.
template <class T, int N>
__device__ __forceinline__ void store_once(typename T::Raw* p, const Pack<T, N>& x) {
  using W = typename Word<sizeof(x)>::type;
  typedef W __attribute__((aligned(sizeof(typename T::Raw)))) Placed;
  __builtin_nontemporal_store(__builtin_bit_cast(W, x), reinterpret_cast<Placed*>(p));
}

// A unit's place in a row: first values of its two vectors. They are
// neighbours, or in the two halves of the rotated values, of the ones behind
// them, or of a row that is not rotated, so that neighbouring lanes' accesses
// are neighbours too.
struct Unit {
  uint32_t d0, d1;
  bool turned;
};
template <int VEC, bool NEIGHBOURS>
__device__ __forceinline__ Unit unit_of(uint32_t c, uint32_t dims, uint32_t dim) {
  const bool turned = c * 2u * VEC < dims;
  const uint32_t from = turned ? 0u : dims, apart = turned ? dims / 2u : (dim - dims) / 2u;
  const uint32_t c0 = c - from / (2u * VEC);
  const uint32_t d0 = from + (NEIGHBOURS ? c0 * 2u * VEC : c0 * VEC);
  return {d0, d0 + (NEIGHBOURS ? VEC : apart), turned};
}

// The unit's values as they are stored, of which the first and the second half
// are its two vectors.
template <class X, int VEC, bool NEIGHBOURS>
__device__ __forceinline__ Pack<X, 2 * VEC> get(const typename X::Raw* row, const Unit& u) {
  if constexpr (NEIGHBOURS && VEC > 1) {
    return load_pack<X, 2 * VEC>(row + u.d0);
  } else {
    const Pack<X, VEC> p0 = load_pack<X, VEC>(row + u.d0), p1 = load_pack<X, VEC>(row + u.d1);
    Pack<X, 2 * VEC> x;
    __builtin_memcpy(x.v, &p0, sizeof p0);
    __builtin_memcpy(x.v + VEC, &p1, sizeof p1);
    return x;
  }
}

// Where a token's pair i has its cosine and sine: lanes take VEC neighbouring
// pairs each, two at a time, and what neighbouring lanes read at once is
// neighbouring 16 bytes. (In their order: 16384 tokens 85 us and not 80, a fifth
// of them with bank conflicts.)
template <int VEC>
__device__ __forceinline__ uint32_t turn_at(uint32_t i, uint32_t half) {
  if (VEC < 4) return i;
  const uint32_t c = i / VEC, j = i % VEC;
  return ((j >> 1) * (half / VEC) + c) * 2u + (j & 1u);
}

// In binary32 and rotated; turn: its token's cosines and sines.
template <class X, int VEC, bool NEIGHBOURS>
__device__ __forceinline__ void rotate(float* x, const Pack<X, 2 * VEC>& in, bool turned, uint32_t c, const float2* turn,
                                       uint32_t half) {
#pragma unroll
  for (int j = 0; j < 2 * VEC; ++j) x[j] = X::load(in.v[j]);
  if (turned) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int ia = NEIGHBOURS ? 2 * j : j, ib = NEIGHBOURS ? 2 * j + 1 : VEC + j;
      const float va = x[ia], vb = x[ib];
      const float2 w = turn[turn_at<VEC>(c * VEC + j, half)];
      x[ia] = va * w.x - vb * w.y;
      x[ib] = va * w.y + vb * w.x;
    }
  }
}

// The unit's values times r, rounded, to a row.
template <class T, int VEC, bool NEIGHBOURS>
__device__ __forceinline__ void put(typename T::Raw* row, const Unit& u, const float* x, float r) {
  if constexpr (NEIGHBOURS && VEC > 1) {
    Pack<T, 2 * VEC> p;
#pragma unroll
    for (int j = 0; j < 2 * VEC; ++j) p.v[j] = T::store(x[j] * r);
    store_once<T, 2 * VEC>(row + u.d0, p);
  } else {
    Pack<T, VEC> p0, p1;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      p0.v[j] = T::store(x[j] * r);
      p1.v[j] = T::store(x[VEC + j] * r);
    }
    store_once<T, VEC>(row + u.d0, p0);
    store_once<T, VEC>(row + u.d1, p1);
  }
}

// Codes of numbers that are finite and at most MAX (and 2^-22 of it), two or
// four at a time: whole numbers are the low byte of 1.5 * 2^23 and the number.
__device__ __forceinline__ uint32_t codes4(I8, float x0, float x1, float x2, float x3) {
  constexpr float kMagic = 12582912.0f;
  const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(x1 + kMagic), __float_as_uint(x0 + kMagic), 0x0c0c0400u);
  const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(x3 + kMagic), __float_as_uint(x2 + kMagic), 0x0c0c0400u);
  return lo | hi << 16;
}
__device__ __forceinline__ uint32_t codes4(E4M3, float x0, float x1, float x2, float x3) {
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x2, x3, __builtin_amdgcn_cvt_pk_fp8_f32(x0, x1, 0, false), true);
}
template <class KV, int VEC, bool NEIGHBOURS>
__device__ __forceinline__ void put_finite(typename KV::Raw* row, const Unit& u, const float* x, float r) {
  if constexpr (VEC == 1) {
    put<KV, VEC, NEIGHBOURS>(row, u, x, r);
  } else {
    uint32_t w[(VEC + 1) / 2];
#pragma unroll
    for (int j = 0; j < 2 * VEC; j += 4) w[j / 4] = codes4(KV(), x[j] * r, x[j + 1] * r, x[j + 2] * r, x[j + 3] * r);
    constexpr int kBytes = NEIGHBOURS ? 2 * VEC : VEC;
    Pack<KV, kBytes> p;
    __builtin_memcpy(p.v, w, kBytes);
    store_once<KV, kBytes>(row + u.d0, p);
    if constexpr (!NEIGHBOURS) {
      __builtin_memcpy(p.v, reinterpret_cast<const char*>(w) + VEC, VEC);
      store_once<KV, VEC>(row + u.d1, p);
    }
  }
}

// Magnitudes in an order that has infinities and NaN below all numbers: the
// bits without the sign, plus what makes those of infinity wrap to 0.
template <int N>
__device__ __forceinline__ void range_of(uint32_t& top, uint32_t& low, const float* x) {
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const uint32_t y = (__float_as_uint(x[j]) << 1) + 0x01000000u;
    top = max(top, y);
    low = min(low, y);
  }
}
__device__ __forceinline__ float magnitude(uint32_t top) {
  return top < 0x01000000u ? 0.0f : __uint_as_float((top - 0x01000000u) >> 1);
}

// Cosines and sines of n tokens at these positions. A thread takes every few tokens of
// one pair; while positions go on as tokens do, the next turn is the one before
// and a step's: four products and not two series. The angles' roundings come to
// 2^-53 of the table's whole turn, those of cosines, sines, products and sums to
// 2^-50 a step, of which a table has 31 at most one after the other: 2^-45.
// (positions: in LDS where there are many. Read from memory, one ahead of the
// loop, 16384 tokens take 80 us and not 77.5, 2047 in blocks of 64 17.8 and not 17.2.)
template <int VEC>
__device__ __forceinline__ void fill_turns(float2* turns, const BlockAppendArgs& a, const int32_t* positions, uint32_t n) {
  const uint32_t half = a.by_half.d, first = a.by_half.div(threadIdx.x), pair = threadIdx.x - first * half;
  const uint32_t stride = a.by_half.div(kThreads);
  if (first >= min(stride, n)) return;
  const uint32_t place = turn_at<VEC>(pair, half);
  const double freq = a.freqs[pair];
  Turn step = {1.0, 0.0}, now = {1.0, 0.0};
  int32_t before = 0, next = positions[first];
  // (The first round is the step's own, so that the series are here once. The
  // next position is on its way while a turn is computed.)
#pragma unroll 1
  for (uint32_t i = first + stride < n ? first - stride : first; (int32_t)i < (int32_t)n; i += stride) {
    const bool own = (int32_t)i < 0;
    const int32_t at = own ? (int32_t)stride : next;
    if (!own) next = positions[min(i + stride, n - 1u)];
    if (!own && i != first && (uint32_t)at - (uint32_t)before == stride) {
      now = Turn{now.cos * step.cos - now.sin * step.sin, now.cos * step.sin + now.sin * step.cos};
    } else {
      now = turn_of<true>((double)at * freq);
    }
    if (own) step = now;
    else turns[i * half + place] = {(float)now.cos, (float)now.sin};
    before = at;
  }
}

// New tokens that stand next to each other in one block.
struct Run {
  uint32_t t0, n;        // first token of the batch, and how many
  uint32_t page, token;  // where the first one goes
};

// The keys (KIND 0) or values (KIND 1) of the blocks that begin in a group of
// tokens (or go on there with a token that is no neighbour of the one before).
template <class X, class KV, int VEC, bool NEIGHBOURS>
__device__ __forceinline__ void write_blocks(const BlockAppendArgs& a, float2* turns, uint32_t group, int kind, uint32_t part) {
  constexpr uint32_t kHold = kHeld<VEC>;
  __shared__ Run s_run[kMaxGroup];
  __shared__ uint32_t s_top[kThreads / 64];
  __shared__ int32_t s_position[kMaxTurned];
  const uint32_t tid = threadIdx.x, lane = lane_id(), wave = readlane_u32(tid >> 6, 0);
  const uint32_t begin = group * a.kv_tokens, size = min(a.kv_tokens, a.T - begin), t = begin + lane;

  // The runs, which every wave finds for itself.
  const int64_t slot = lane < size ? a.slots[t] : -1, before = lane < size && t ? a.slots[t - 1u] : -2;
  uint32_t page = 0, token = 0;
  bool bad = false;
  const bool live_slot = a.short_slots ? split_short_slot(slot, a.pages, a.by_page, page, token, bad)
                                       : split_slot(slot, a.pages, a.page, page, token, bad);
  if (bad && part == 0u && kind == 0 && wave == 0u) atomicOr(a.status, LLMHIP_KSTATUS_BAD_INDEX);
  const uint32_t block_size = a.block_scales.by_block.d, in_block = a.block_scales.by_block.mod(token);
  const bool goes_on = live_slot && in_block && before == slot - 1;
  const uint64_t first = __ballot(live_slot && !goes_on), others = __ballot(goes_on);
  const uint32_t runs = (uint32_t)__builtin_popcountll(first);
  if (!runs) return;
  const uint64_t behind = ~(others >> 1 >> lane);  // (the top bit is always set)
  uint32_t n = 1u + (uint32_t)__builtin_ctzll(behind);
  const uint32_t last = 63u - (uint32_t)__builtin_clzll(first);
  if (last + readlane_u32(n, last) == size) {  // the last one may go on behind the group
    const int64_t slot0 = (int64_t)readlane_u64((uint64_t)slot, last);
    const uint32_t most = min(block_size - readlane_u32(in_block, last), a.T - begin - last);
    uint32_t has = size - last;
    while (has < most) {
      const uint32_t i = has + lane;
      const uint64_t other = ~__ballot(i < most && a.slots[begin + last + min(i, most - 1u)] == slot0 + i);
      has += other ? (uint32_t)__builtin_ctzll(other) : 64u;
      if (other) break;
    }
    n = lane == last ? has : n;
  }
  const bool leads = first >> lane & 1u;
  uint32_t most_tokens = leads ? n : 0u;
#pragma unroll
  for (uint32_t off = 1; off < kMaxGroup; off *= 2u) most_tokens = max(most_tokens, (uint32_t)__shfl_xor((int)most_tokens, (int)off, 64));
  most_tokens = readlane_u32(most_tokens, 0);
  if (wave == 0u && leads) s_run[lanes_below(first)] = Run{t, n, page, token};
  __syncthreads();

  // A block's head is a task of `lanes` lanes.
  const uint32_t row = a.by_row.d, dims = kind ? 0u : a.dims, half = dims / 2u;
  const uint32_t longest = most_tokens * row, share = max((longest + kHold - 1u) / kHold, min(row, longest));
  const uint32_t log_lanes = share >= kThreads ? 8u : share <= 1u ? 0u : 32u - (uint32_t)__builtin_clz(share - 1u);
  const uint32_t lanes = 1u << log_lanes, at_once = kThreads >> log_lanes, tasks = runs * a.heads;
  const uint32_t step = lanes * kHold, steps = (longest + step - 1u) / step;  // units at a time; more than one: all lanes' task
  uint32_t turns_from = 0u, turns_to = 0u;  // tokens whose cosines and sines are there
  const auto run_of = [&](uint32_t task) { return a.by_heads.div(task); };
  for (uint32_t turn = part, task0 = turn * at_once, stop; task0 < tasks;
       task0 = stop < min((turn + 1u) * at_once, tasks) ? stop : (turn += a.kv_parts) * at_once) {
    // Tasks task0 .. stop, whose runs' tokens fit the table of cosines and sines.
    stop = min((turn + 1u) * at_once, tasks);
    const uint32_t run0 = run_of(task0), from = s_run[run0].t0;
    uint32_t run1 = run_of(stop - 1u), upto = s_run[run1].t0 + s_run[run1].n;
    while (half && steps == 1u && upto - from > a.turn_tokens && run1 > run0) {
      stop = run1 * a.heads;
      --run1;
      upto = s_run[run1].t0 + s_run[run1].n;
    }
    const uint32_t task = task0 + (tid >> log_lanes), me = tid & (lanes - 1u);
    const bool live = task < stop;
    const uint32_t mine = min(task, stop - 1u), r = run_of(mine), head = mine - r * a.heads;
    const uint32_t units = live ? s_run[r].n * row : 0u, place = a.block_scales.by_block.mod(s_run[r].token);

    // (Again where they are needed: registers are what limits the workgroups of a compute unit.)
    const auto row_out = [&] {
      const Run to = s_run[r];
      return static_cast<typename KV::Raw*>(a.pool[kind]) + (int64_t)to.page * a.pool_stride[kind][0] +
             (int64_t)to.token * a.pool_stride[kind][1] + (int64_t)head * a.pool_stride[kind][2];
    };
    const auto scale_at = [&] {
      const Run to = s_run[r];
      return a.block_scales.scale[kind] + (int64_t)to.page * a.block_scales.stride[kind][0] +
             (int64_t)a.block_scales.by_block.div(to.token) * a.block_scales.stride[kind][1] +
             (int64_t)head * a.block_scales.stride[kind][2];
    };
    const float old = live && place ? *scale_at() : 0.0f;

    // The task's units in steps of as many as its lanes hold: read and looked at,
    // then written; of more than one step all are read again.
    float x[kHold][2 * VEC];
    uint32_t top = 0u, low = ~0u;
    float by = 1.0f;
#pragma unroll 1
    for (uint32_t p = 0; p < 2u * steps; ++p) {
      const bool writes = p >= steps;
      const uint32_t first_unit = (writes ? p - steps : p) * step + me;
      if (!writes || steps > 1u) {
        Pack<X, 2 * VEC> raw[kHold];
        const uint32_t t0 = s_run[r].t0;
        const typename X::Raw* in = static_cast<const typename X::Raw*>(a.x[1 + kind]) + (int64_t)t0 * a.x_stride[1 + kind][0] +
                                    (int64_t)head * a.x_stride[1 + kind][1];
#pragma unroll
        for (uint32_t k = 0; k < kHold; ++k) {
          const uint32_t u = first_unit + k * lanes, i = a.by_row.div(u);
          raw[k] = Pack<X, 2 * VEC>{};
          if (u < units)
            raw[k] = get<X, VEC, NEIGHBOURS>(in + (int64_t)i * a.x_stride[1 + kind][0], unit_of<VEC, NEIGHBOURS>(u - i * row, dims, a.dim));
        }
        // Cosines and sines of the step's tokens, from turned_from on.
        uint32_t turned_from = from;
        if (half) {
          uint32_t to = upto;
          if (steps > 1u) {
            const uint32_t unit0 = first_unit - me;
            turned_from += a.by_row.div(unit0);
            to = min(upto, from + a.by_row.div(unit0 + step - 1u) + 1u);
          }
          if (turned_from != turns_from || to != turns_to) {
            const uint32_t tokens = to > turned_from ? to - turned_from : 0u;  // (a shorter run has none in the last steps)
            for (uint32_t i = tid; i < tokens; i += kThreads) s_position[i] = a.positions[turned_from + i];
            __syncthreads();  // (and the turns before are used)
            fill_turns<VEC>(turns, a, s_position, tokens);
            __syncthreads();
            turns_from = turned_from;
            turns_to = to;
          }
        }
#pragma unroll
        for (uint32_t k = 0; k < kHold; ++k) {
          const uint32_t u = first_unit + k * lanes, i = a.by_row.div(u), c = u - i * row;
          rotate<X, VEC, NEIGHBOURS>(x[k], raw[k], u < units && c * 2u * VEC < dims, c, turns + (t0 + i - turned_from) * half,
                                     half);
          range_of<2 * VEC>(top, low, x[k]);
        }
      }
      if (p + 1u == steps) {
        for (uint32_t off = 1; off < min(lanes, 64u); off *= 2u) top = max(top, (uint32_t)__shfl_xor((int)top, (int)off, 64));
        if (lanes > 64u) {
          __syncthreads();
          if (lane == 0u) s_top[wave] = top;
          __syncthreads();
          for (uint32_t w = 0; w < lanes / 64u; ++w) top = max(top, s_top[(wave & ~(lanes / 64u - 1u)) + w]);
        }
        float s = magnitude(top) / KV::kMax;
        s = s < 0x1p-126f ? 0.0f : s;
        s = old > s ? old : s;
        by = s > 0.0f ? 1.0f / s : 1.0f;  // (1: all finite values are so small that they round to 0)
        if (live && me == 0u && !(place && s == old)) *scale_at() = s;
        if (live && place && s > old) {  // kept tokens: 8 codes at a time
          const float f = old / s;
          const uint32_t eights = a.dim / 8u;
          typename KV::Raw* kept = row_out() - (int64_t)place * a.pool_stride[kind][1];
          for (uint32_t u = me; u < place * eights; u += lanes) {
            const uint32_t i = u / eights;
            typename KV::Raw* c = kept + (int64_t)i * a.pool_stride[kind][1] + (u - i * eights) * 8u;
            Pack<KV, 8> codes = *reinterpret_cast<const Pack<KV, 8>*>(c);
#pragma unroll
            for (int j = 0; j < 8; ++j) codes.v[j] = KV::store(KV::load(codes.v[j]) * f);
            *reinterpret_cast<Pack<KV, 8>*>(c) = codes;
          }
        }
      }
      if (writes) {
        const bool odd = __any(low < 0x01000000u);
        typename KV::Raw* out = row_out();
#pragma unroll
        for (uint32_t k = 0; k < kHold; ++k) {
          const uint32_t u = first_unit + k * lanes, i = a.by_row.div(u);
          if (u >= units) continue;
          const Unit at = unit_of<VEC, NEIGHBOURS>(u - i * row, dims, a.dim);
          typename KV::Raw* to = out + (int64_t)i * a.pool_stride[kind][1];
          if (__builtin_expect(odd, 0)) put<KV, VEC, NEIGHBOURS>(to, at, x[k], by);
          else put_finite<KV, VEC, NEIGHBOURS>(to, at, x[k], by);
        }
      }
    }
  }
}

template <class X, class KV, int VEC, bool NEIGHBOURS>
__global__ __launch_bounds__(kThreads, 4) void block_append_kernel(BlockAppendArgs a) {
  extern __shared__ float2 s_turn[];
  const uint32_t tid = threadIdx.x;
  // (Keys and values first: spread among the queries' workgroups they end later,
  // 16384 tokens 95 us, not 90.)
  const uint32_t kv = a.kv_groups * 2u * a.kv_parts;
  if (blockIdx.x < kv) {
    const uint32_t group = blockIdx.x / (2u * a.kv_parts), part = blockIdx.x - group * 2u * a.kv_parts;
    write_blocks<X, KV, VEC, NEIGHBOURS>(a, s_turn, group, part & 1u, part >> 1);
    return;
  }
  const uint32_t t0 = (blockIdx.x - kv) * a.tokens_per_group, n = min(a.tokens_per_group, a.T - t0);
  const uint32_t half = a.dims / 2u, units = n * a.by_token.d;
  // A thread's first unit is on its way while the cosines and sines are computed.
  const auto unit_at = [&](uint32_t u, uint32_t& t, uint32_t& head, uint32_t& c) {
    t = a.by_token.div(u);
    const uint32_t in_token = u - t * a.by_token.d;
    head = a.by_row.div(in_token);
    c = in_token - head * a.by_row.d;
  };
  const auto row_of = [&](uint32_t t, uint32_t head) {
    return static_cast<const typename X::Raw*>(a.x[0]) + (int64_t)(t0 + t) * a.x_stride[0][0] + (int64_t)head * a.x_stride[0][1];
  };
  uint32_t t, head, c;
  unit_at(min(tid, units - 1u), t, head, c);
  Pack<X, 2 * VEC> in = get<X, VEC, NEIGHBOURS>(row_of(t, head), unit_of<VEC, NEIGHBOURS>(c, a.dims, a.dim));
  if (half) {
    fill_turns<VEC>(s_turn, a, a.positions + t0, n);
    __syncthreads();
  }
#pragma unroll 1
  for (uint32_t u = tid; u < units; u += kThreads) {
    if (u != tid) {
      unit_at(u, t, head, c);
      in = get<X, VEC, NEIGHBOURS>(row_of(t, head), unit_of<VEC, NEIGHBOURS>(c, a.dims, a.dim));
    }
    const Unit at = unit_of<VEC, NEIGHBOURS>(c, a.dims, a.dim);
    float x[2 * VEC];
    rotate<X, VEC, NEIGHBOURS>(x, in, at.turned, c, s_turn + t * half, half);
    put<X, VEC, NEIGHBOURS>(static_cast<typename X::Raw*>(a.out_q) + (int64_t)(t0 + t) * a.oq_stride[0] +
                                (int64_t)head * a.oq_stride[1], at, x, 1.0f);
  }
}

template <class X, class KV, int VEC, bool NEIGHBOURS>
hipError_t launch_vec(BlockAppendArgs a, hipStream_t s) {
  constexpr uint32_t kHold = kHeld<VEC>;
  const uint32_t row = a.dim / (2u * VEC), units = row * a.q_heads, half = a.dims / 2u, block = a.block_scales.by_block.d;
  a.by_row = FastDiv::of(row);
  a.by_token = FastDiv::of(units ? units : 1u);
  a.by_half = FastDiv::of(half ? half : 1u);
  a.by_heads = FastDiv::of(a.heads);
  a.by_page = FastDiv::of(a.page);
  a.short_slots = (uint64_t)a.pages * a.page <= 0x7fffffffu;
  a.tokens_per_group = units ? std::min(std::max(kThreads / units, 1u), kMaxQueryTokens) : 1u;
  // About the tokens of a block, so that a workgroup seldom finds none that begins.
  a.kv_tokens = std::min(std::max(block, 16u), kMaxGroup);
  a.kv_groups = (a.T + a.kv_tokens - 1u) / a.kv_tokens;
  // Workgroups for each group of tokens, keys or values: as many as have tasks
  // when its tokens are blocks of their own, or one block; 1024 in all, as each
  // that finds no task has read the slots for nothing (16384 tokens 90 us, with
  // 8192 workgroups 130).
  const uint32_t longest = std::min(block, a.T), tokens = std::min(a.kv_tokens, a.T);
  const auto parts_of = [&](uint32_t blocks, uint32_t n) {
    uint32_t lanes = 1u;
    while (lanes < kThreads && (lanes * kHold < n * row || lanes < row)) lanes *= 2u;
    return ((uint64_t)blocks * a.heads * lanes + kThreads - 1u) / kThreads;
  };
  const uint64_t parts = std::max(parts_of(tokens, 1u), parts_of(1u, longest));
  a.kv_parts = (uint32_t)std::min<uint64_t>(parts, std::max(1024u / (2u * a.kv_groups), 1u));
  a.turn_tokens = append_turn_tokens(longest, VEC, a.dim);
  const uint32_t lds = half * std::max(a.tokens_per_group, a.turn_tokens) * (uint32_t)sizeof(float2);
  const uint32_t kv = a.kv_groups * 2u * a.kv_parts;
  const dim3 grid(kv + (units ? (a.T + a.tokens_per_group - 1u) / a.tokens_per_group : 0u));
  hipLaunchKernelGGL((block_append_kernel<X, KV, VEC, NEIGHBOURS>), grid, dim3(kThreads), lds, s, a);
  return hipGetLastError();
}

template <class X, class KV>
hipError_t launch(const BlockAppendArgs& a, bool neighbours, uint32_t vec, hipStream_t s) {
  // 16 bytes an access: a vector, or two neighbouring ones.
  constexpr int kWide = 16 / sizeof(typename X::Raw);
  if (neighbours) return vec == kWide / 2 ? launch_vec<X, KV, kWide / 2, true>(a, s) : launch_vec<X, KV, 1, true>(a, s);
  if (vec == kWide) return launch_vec<X, KV, kWide, false>(a, s);
  return vec == kWide / 2 ? launch_vec<X, KV, kWide / 2, false>(a, s) : launch_vec<X, KV, 1, false>(a, s);
}

}  // namespace

hipError_t launch_kv_block_append(const BlockAppendArgs& a, uint32_t dtype, uint32_t kv_dtype, bool neighbours, uint32_t vec,
                                  hipStream_t s) {
  const bool i8 = kv_dtype == LLMHIP_I8;
  switch (dtype) {
    case LLMHIP_F32: return i8 ? launch<F32, I8>(a, neighbours, vec, s) : launch<F32, E4M3>(a, neighbours, vec, s);
    case LLMHIP_BF16: return i8 ? launch<BF16, I8>(a, neighbours, vec, s) : launch<BF16, E4M3>(a, neighbours, vec, s);
    default: return i8 ? launch<F16, I8>(a, neighbours, vec, s) : launch<F16, E4M3>(a, neighbours, vec, s);
  }
}

}  // namespace llmhip
