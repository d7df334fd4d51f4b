// New tokens' keys and values, quantised, into their slots, and their queries
// rotated (llmhip_kv_block_append).
//
// A block's scale needs the largest of its new values before the first code
// can be written. A wave takes one head of one block's new tokens, keys or
// values: it holds what it has read (and turned) in registers while the
// maximum goes across its lanes, then writes codes; of more than it can hold
// it reads the rest again, from the L2. So a value comes from memory once and
// blocks need no workgroup-wide step but the cosines and sines, which all heads
// of a workgroup share in LDS. Kept tokens are read only where the scale grew.
// Units are laid out as in the append to a cache of values: 2 * VEC values of
// a row, VEC pairs, or values that are not rotated.
#include <type_traits>

#include "kv_args.h"
#include "kv_turn.h"
#include "kv_types.h"
#include "wave_ops.h"

namespace llmhip {
namespace {

constexpr uint32_t kMaxWaves = 8;
constexpr uint32_t kMaxTokens = 8;      // of a workgroup of queries
constexpr uint32_t kMaxTurns = 4096;    // cosines and sines in LDS: 32 KiB

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

// The unit's values in binary32; turn: its token's cosines and sines.
template <class X, int VEC, bool NEIGHBOURS>
__device__ __forceinline__ void get(float* x, const typename X::Raw* row, const Unit& u, uint32_t c, const float2* turn) {
  if constexpr (NEIGHBOURS && VEC > 1) {
    const Pack<X, 2 * VEC> in = load_pack<X, 2 * VEC>(row + u.d0);
#pragma unroll
    for (int j = 0; j < 2 * VEC; ++j) x[j] = X::load(in.v[j]);
  } else {
    const Pack<X, VEC> p0 = load_pack<X, VEC>(row + u.d0), p1 = load_pack<X, VEC>(row + u.d1);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      x[j] = X::load(p0.v[j]);
      x[VEC + j] = X::load(p1.v[j]);
    }
  }
  if (u.turned) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int ia = NEIGHBOURS ? 2 * j : j, ib = NEIGHBOURS ? 2 * j + 1 : VEC + j;
      const float va = x[ia], vb = x[ib];
      const float2 w = turn[c * VEC + j];
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

// The largest finite magnitude (fmax drops the NaN that it meets).
template <int N>
__device__ __forceinline__ float largest(float top, const float* x) {
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const float y = __builtin_fabsf(x[j]);
    top = __builtin_fmaxf(top, y == INFINITY ? 0.0f : y);
  }
  return top;
}

__device__ __forceinline__ void fill_turns(float2* turns, const BlockAppendArgs& a, uint32_t t0, uint32_t n) {
  const uint32_t half = a.dims / 2u;
  for (uint32_t i = threadIdx.x; i < n * half; i += blockDim.x) {
    const uint32_t t = i / half;
    turns[i] = cos_sin((double)a.positions[t0 + t] * a.freqs[i - t * half]);
  }
}

// The n new tokens t0 .. of one block, first of them at place `token` of page
// `page`: one head's keys (KIND 0) or values (KIND 1). All waves of the
// workgroup come here together; one that is not `live` has no head.
template <class X, class KV, int VEC, bool NEIGHBOURS>
__device__ __forceinline__ void write_block(const BlockAppendArgs& a, float2* turns, int kind, uint32_t head, bool live,
                                            uint32_t t0, uint32_t n, uint32_t page, uint32_t token) {
  constexpr uint32_t kHeld = VEC == 1 ? 8 : 64 / (2 * VEC);  // units of a lane in registers
  const uint32_t lane = lane_id(), row = a.by_row.d;
  const uint32_t dims = kind ? 0u : a.dims, half = dims / 2u;
  const uint32_t chunk = dims ? a.turn_tokens : n;  // tokens whose cosines and sines are there
  const uint32_t block = a.block_scales.by_block.div(token), place = token - block * a.block_scales.by_block.d;
  const typename X::Raw* in = static_cast<const typename X::Raw*>(a.x[1 + kind]) + (int64_t)t0 * a.x_stride[1 + kind][0] +
                              (int64_t)head * a.x_stride[1 + kind][1];
  typename KV::Raw* out = static_cast<typename KV::Raw*>(a.pool[kind]) + (int64_t)page * a.pool_stride[kind][0] +
                          (int64_t)token * a.pool_stride[kind][1] + (int64_t)head * a.pool_stride[kind][2];
  float* scale = a.block_scales.scale[kind] + (int64_t)page * a.block_scales.stride[kind][0] +
                 (int64_t)block * a.block_scales.stride[kind][1] + (int64_t)head * a.block_scales.stride[kind][2];
  const float old = live && place ? *scale : 0.0f;

  float held[kHeld][2 * VEC], top = 0.0f;
  const auto each = [&](uint32_t u, float* x, uint32_t c0, auto&& use) {
    const uint32_t t = a.by_row.div(u), c = u - t * row;
    const Unit at = unit_of<VEC, NEIGHBOURS>(c, dims, a.dim);
    get<X, VEC, NEIGHBOURS>(x, in + (int64_t)(c0 + t) * a.x_stride[1 + kind][0], at, c, turns + t * half);
    use(at, c0 + t);
  };
  for (uint32_t c0 = 0; c0 < n; c0 += chunk) {
    const uint32_t units = live ? min(chunk, n - c0) * row : 0u;
    if (dims) {
      __syncthreads();  // (the ones before are used)
      fill_turns(turns, a, t0 + c0, min(chunk, n - c0));
      __syncthreads();
    }
    if (n <= chunk) {
#pragma unroll
      for (uint32_t k = 0; k < kHeld; ++k) {
#pragma unroll
        for (int j = 0; j < 2 * VEC; ++j) held[k][j] = 0.0f;
        if (lane + 64u * k < units) each(lane + 64u * k, held[k], c0, [](const Unit&, uint32_t) {});
      }
#pragma unroll
      for (uint32_t k = 0; k < kHeld; ++k) top = largest<2 * VEC>(top, held[k]);
    }
    for (uint32_t u = lane + (n <= chunk ? 64u * kHeld : 0u); u < units; u += 64u) {
      float x[2 * VEC];
      each(u, x, c0, [](const Unit&, uint32_t) {});
      top = largest<2 * VEC>(top, x);
    }
  }
#pragma unroll
  for (uint32_t off = 32; off > 0; off >>= 1) top = __builtin_fmaxf(top, __shfl_xor(top, off, 64));
  float s = top / KV::kMax;
  s = s < 0x1p-126f ? 0.0f : s;
  s = old > s ? old : s;
  const float r = s > 0.0f ? 1.0f / s : 1.0f;  // (1: all finite values are so small that they round to 0)
  if (live && lane == 0u && !(s == old && place)) *scale = s;
  if (live && place && s > old) {  // kept tokens: 8 codes at a time
    const float f = old / s;
    const uint32_t eights = a.dim / 8u;
    typename KV::Raw* first = out - (int64_t)place * a.pool_stride[kind][1];
    for (uint32_t u = lane; u < place * eights; u += 64u) {
      const uint32_t t = u / eights;
      typename KV::Raw* p = first + (int64_t)t * a.pool_stride[kind][1] + (u - t * eights) * 8u;
      Pack<KV, 8> x = *reinterpret_cast<const Pack<KV, 8>*>(p);
#pragma unroll
      for (int j = 0; j < 8; ++j) x.v[j] = KV::store(KV::load(x.v[j]) * f);
      *reinterpret_cast<Pack<KV, 8>*>(p) = x;
    }
  }
  for (uint32_t c0 = 0; c0 < n; c0 += chunk) {
    const uint32_t units = live ? min(chunk, n - c0) * row : 0u;
    if (n <= chunk) {
#pragma unroll
      for (uint32_t k = 0; k < kHeld; ++k) {
        const uint32_t u = lane + 64u * k, t = a.by_row.div(u);
        if (u < units)
          put<KV, VEC, NEIGHBOURS>(out + (int64_t)t * a.pool_stride[kind][1], unit_of<VEC, NEIGHBOURS>(u - t * row, dims, a.dim), held[k], r);
      }
    } else if (dims) {
      __syncthreads();
      fill_turns(turns, a, t0 + c0, min(chunk, n - c0));
      __syncthreads();
    }
    for (uint32_t u = lane + (n <= chunk ? 64u * kHeld : 0u); u < units; u += 64u) {
      float x[2 * VEC];
      each(u, x, c0, [&](const Unit& at, uint32_t t) {
        put<KV, VEC, NEIGHBOURS>(out + (int64_t)t * a.pool_stride[kind][1], at, x, r);
      });
    }
  }
}

template <class X, class KV, int VEC, bool NEIGHBOURS>
__global__ __launch_bounds__(kMaxWaves * 64) void block_append_kernel(BlockAppendArgs a) {
  extern __shared__ float2 s_turn[];
  const uint32_t tid = threadIdx.x, lane = lane_id(), wave = readlane_u32(tid >> 6, 0);
  if (blockIdx.x < a.kv_groups * a.kv_parts) {
    // Keys or values of kv_waves heads, of the blocks that begin in a group of
    // tokens (or go on there with a token that is no neighbour of the last).
    const uint32_t group = blockIdx.x / a.kv_parts, part = blockIdx.x - group * a.kv_parts;
    const int kind = part >= a.kv_parts / 2u;
    const uint32_t head = (part - kind * (a.kv_parts / 2u)) * a.kv_waves + wave;
    const uint32_t t = group * a.kv_tokens + lane;
    const int64_t slot = lane < a.kv_tokens && t < a.T ? a.slots[t] : -1;
    uint32_t page = 0, token = 0;
    bool bad = false, first = split_slot(slot, a.pages, a.page, page, token, bad);
    if (bad && part == 0u && wave == 0u) atomicOr(a.status, LLMHIP_KSTATUS_BAD_INDEX);
    const uint32_t place = a.block_scales.by_block.mod(token);
    if (first && place && t) first = a.slots[t - 1u] != slot - 1;
    for (uint64_t runs = __ballot(first); runs; runs &= runs - 1u) {
      const uint32_t at = (uint32_t)__builtin_ctzll(runs);
      const uint32_t t0 = readlane_u32(t, at);
      const int64_t slot0 = (int64_t)readlane_u64((uint64_t)slot, at);
      const uint32_t most = min(a.block_scales.by_block.d - readlane_u32(place, at), a.T - t0);
      uint32_t n = 0;
      while (n < most) {
        const uint32_t i = n + lane;
        const uint64_t other = ~__ballot(i < most && a.slots[t0 + i] == slot0 + i);
        n += other ? (uint32_t)__builtin_ctzll(other) : 64u;
        if (other) break;
      }
      write_block<X, KV, VEC, NEIGHBOURS>(a, s_turn, kind, min(head, a.heads - 1u), head < a.heads, t0, n, readlane_u32(page, at),
                                          readlane_u32(token, at));
    }
    return;
  }
  const uint32_t t0 = (blockIdx.x - a.kv_groups * a.kv_parts) * a.tokens_per_group, n = min(a.tokens_per_group, a.T - t0);
  if (a.dims) {
    fill_turns(s_turn, a, t0, n);
    __syncthreads();
  }
  const uint32_t half = a.dims / 2u;
  for (uint32_t u = tid; u < n * a.by_token.d; u += blockDim.x) {
    const uint32_t t = a.by_token.div(u), in_token = u - t * a.by_token.d;
    const uint32_t head = a.by_row.div(in_token), c = in_token - head * a.by_row.d;
    const Unit at = unit_of<VEC, NEIGHBOURS>(c, a.dims, a.dim);
    float x[2 * VEC];
    get<X, VEC, NEIGHBOURS>(x, static_cast<const typename X::Raw*>(a.x[0]) + (int64_t)(t0 + t) * a.x_stride[0][0] +
                                   (int64_t)head * a.x_stride[0][1], at, c, s_turn + t * half);
    put<X, VEC, NEIGHBOURS>(static_cast<typename X::Raw*>(a.out_q) + (int64_t)(t0 + t) * a.oq_stride[0] +
                                (int64_t)head * a.oq_stride[1], at, x, 1.0f);
  }
}

template <class X, class KV>
hipError_t launch(BlockAppendArgs a, bool neighbours, uint32_t vec, hipStream_t s) {
  a.kv_waves = min(a.heads, kMaxWaves);
  const uint32_t threads = a.kv_waves * 64u, row = a.dim / (2u * vec), units = row * a.q_heads;
  a.by_row = FastDiv::of(row);
  a.by_token = FastDiv::of(units ? units : 1u);
  // A token of a group where few are (a decode step's are blocks of their
  // own), up to 16, the more of which are one block's, of prompts.
  a.kv_tokens = min(max(a.T / 1024u, 1u), 16u);
  a.kv_groups = (a.T + a.kv_tokens - 1u) / a.kv_tokens;
  a.kv_parts = 2u * ((a.heads + a.kv_waves - 1u) / a.kv_waves);
  a.tokens_per_group = units ? min(max(threads / units, 1u), kMaxTokens) : 1u;
  const uint32_t half = a.dims / 2u;
  a.turn_tokens = half ? min(a.block_scales.by_block.d, kMaxTurns / half) : 1u;
  const uint32_t lds = half * max(a.turn_tokens, a.tokens_per_group) * (uint32_t)sizeof(float2);
  const dim3 grid(a.kv_groups * a.kv_parts + (units ? (a.T + a.tokens_per_group - 1u) / a.tokens_per_group : 0u));
  const auto go = [&](auto v, auto n) {
    constexpr int VEC = decltype(v)::value;
    hipLaunchKernelGGL((block_append_kernel<X, KV, VEC, decltype(n)::value>), grid, dim3(threads), lds, s, a);
  };
  using std::integral_constant;
  // 16 bytes an access: a vector, or two neighbouring ones.
  constexpr int kWide = 16 / sizeof(typename X::Raw);
  if (neighbours) {
    if (vec == kWide / 2) go(integral_constant<int, kWide / 2>{}, std::true_type{});
    else go(integral_constant<int, 1>{}, std::true_type{});
  } else if (vec == kWide) {
    go(integral_constant<int, kWide>{}, std::false_type{});
  } else if (vec == kWide / 2) {
    go(integral_constant<int, kWide / 2>{}, std::false_type{});
  } else {
    go(integral_constant<int, 1>{}, std::false_type{});
  }
  return hipGetLastError();
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
