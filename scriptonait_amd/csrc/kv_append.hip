// New tokens' keys and values into their slots and their queries rotated
// (llmhip_kv_append).
//
// A unit is 2 * VEC values of one head row: VEC pairs, or values that are
// not rotated. A workgroup takes a few tokens. It first computes their
// cosines and sines, once for all heads, into LDS: the angle is reduced to
// [-pi/4, pi/4] in binary64 and both series are summed there, so a far
// position is as exact as a near one. What bounds it is the traffic of the
// rows: 403 MB of 16384 tokens in 69 us, 5.8 TB/s; for few tokens latency.
#include <type_traits>

#include "kv_args.h"
#include "kv_types.h"

namespace llmhip {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kMaxTokens = 8;

// cos and sin of x: x - k pi/2 with pi/2 in two parts (k < 2^31 keeps the
// rest's error below 2^-70), then the Taylor sums. At pi/4 the first left
// out terms are 4e-14 (sin, x^15 / 15!) and 1e-12 (cos, x^14 / 14!), far
// below half a step of binary32.
__device__ __forceinline__ float2 cos_sin(double x) {
  const double k = rint(x * 0.63661977236758134308);
  double r = __builtin_fma(-k, 1.57079632679489661923, x);
  r = __builtin_fma(-k, 6.123233995736766036e-17, r);
  const double z = r * r;
  double s = 1.0 / 6227020800.0, c = 1.0 / 479001600.0;
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
  return {(float)(quarter == 1 || quarter == 2 ? -cc : cc), (float)(quarter >= 2 ? -ss : ss)};
}

// A pack's store past the L2: rows are written once and read by later kernels.
// (16384 tokens of 40 rotated and 8 moved rows of 128 bf16 69 us, with plain
// stores 73; loads past it 67, but an operand that the projections have just
// left in the caches is then read from memory: 4000 tokens of f32 37 us, not 29.)
template <int BYTES>
struct Word;
template <> struct Word<1> { using type = uint8_t; };
template <> struct Word<2> { using type = uint16_t; };
template <> struct Word<4> { using type = uint32_t; };
template <> struct Word<8> { using type = uint32_t __attribute__((ext_vector_type(2))); };
template <> struct Word<16> { using type = uint32_t __attribute__((ext_vector_type(4))); };
template <class P>
__device__ __forceinline__ void store_once(void* p, const P& x) {
  using W = typename Word<sizeof(P)>::type;
  __builtin_nontemporal_store(__builtin_bit_cast(W, x), static_cast<W*>(p));
}

// A unit's values, rounded, to a row.
template <class T, int VEC, bool NEIGHBOURS>
__device__ __forceinline__ void put(typename T::Raw* row, uint32_t d0, uint32_t d1, const float* x) {
  if constexpr (NEIGHBOURS && VEC > 1) {
    Pack<T, 2 * VEC> p;
#pragma unroll
    for (int j = 0; j < 2 * VEC; ++j) p.v[j] = T::store(x[j]);
    store_once(row + d0, p);
  } else {
    Pack<T, VEC> p0, p1;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      p0.v[j] = T::store(x[j]);
      p1.v[j] = T::store(x[VEC + j]);
    }
    store_once(row + d0, p0);
    store_once(row + d1, p1);
  }
}

template <class X, class KV, int VEC, bool NEIGHBOURS>
__global__ __launch_bounds__(kThreads) void append_kernel(AppendArgs a) {
  __shared__ float2 s_turn[kMaxTokens * kMaxHeadDim / 2];
  __shared__ int64_t s_row[2][kMaxTokens];  // each token's place in the pools; -1: none
  const uint32_t tid = threadIdx.x, half = a.dims / 2u;
  const uint32_t t0 = blockIdx.x * a.tokens_per_group, n = min(a.tokens_per_group, a.T - t0);
  bool bad = false;
  if (tid < n) {
    uint32_t p = 0, t = 0;
    const bool live = split_slot(a.slots[t0 + tid], a.pages, a.page, p, t, bad);
    for (uint32_t i = 0; i < 2u; ++i)
      s_row[i][tid] = live ? (int64_t)p * a.pool_stride[i][0] + (int64_t)t * a.pool_stride[i][1] : -1;
  }
  if (bad) atomicOr(a.status, LLMHIP_KSTATUS_BAD_INDEX);
  for (uint32_t i = tid; i < n * half; i += kThreads) {
    const uint32_t t = i / half;
    s_turn[i] = cos_sin((double)a.positions[t0 + t] * a.freqs[i - t * half]);
  }
  __syncthreads();

  const uint32_t units = n * a.by_token.d;
  for (uint32_t u = tid; u < units; u += kThreads) {
    const uint32_t t = a.by_token.div(u), in_token = u - t * a.by_token.d;
    uint32_t head = a.by_row.div(in_token);
    const uint32_t c = in_token - head * a.by_row.d;
    const uint32_t kind = head < a.q_heads ? 0u : head < a.q_heads + a.heads ? 1u : 2u;
    head -= kind == 0u ? 0u : kind == 1u ? a.q_heads : a.q_heads + a.heads;
    if (kind && s_row[kind - 1u][t] < 0) continue;
    // Where the unit's two vectors are. They are neighbours, or in the two
    // halves of the rotated values, of the ones behind them, or of a value's
    // row, so that neighbouring threads' accesses are neighbours too.
    const bool turned = kind < 2u && c * 2u * VEC < a.dims;
    const uint32_t from = kind < 2u && !turned ? a.dims : 0u;
    const uint32_t c0 = c - from / (2u * VEC), apart = kind == 2u ? a.dim / 2u : turned ? half : (a.dim - a.dims) / 2u;
    const uint32_t d0 = from + (NEIGHBOURS ? c0 * 2u * VEC : c0 * VEC), d1 = d0 + (NEIGHBOURS ? VEC : apart);
    const typename X::Raw* row = static_cast<const typename X::Raw*>(a.x[kind]) +
                                 (int64_t)(t0 + t) * a.x_stride[kind][0] + (int64_t)head * a.x_stride[kind][1];
    Pack<X, 2 * VEC> in;
    if constexpr (NEIGHBOURS && VEC > 1) {  // (single values: rows of any alignment)
      in = *reinterpret_cast<const Pack<X, 2 * VEC>*>(row + d0);
    } else {
      const Pack<X, VEC> p0 = *reinterpret_cast<const Pack<X, VEC>*>(row + d0);
      const Pack<X, VEC> p1 = *reinterpret_cast<const Pack<X, VEC>*>(row + d1);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        in.v[j] = p0.v[j];
        in.v[VEC + j] = p1.v[j];
      }
    }
    float x[2 * VEC];
#pragma unroll
    for (int j = 0; j < 2 * VEC; ++j) x[j] = X::load(in.v[j]);
    if (turned) {
      const float2* turn = s_turn + t * half + c * VEC;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int ia = NEIGHBOURS ? 2 * j : j, ib = NEIGHBOURS ? 2 * j + 1 : VEC + j;
        const float va = x[ia], vb = x[ib];
        const float2 w = turn[j];
        x[ia] = va * w.x - vb * w.y;
        x[ib] = va * w.y + vb * w.x;
      }
    }
    if (kind == 0u) {
      put<X, VEC, NEIGHBOURS>(static_cast<typename X::Raw*>(a.out_q) + (int64_t)(t0 + t) * a.oq_stride[0] +
                                  (int64_t)head * a.oq_stride[1],
                              d0, d1, x);
    } else {
      if constexpr (KV::kId == LLMHIP_E4M3) {
        const float scale = a.scale[kind - 1u][head];
#pragma unroll
        for (int j = 0; j < 2 * VEC; ++j) x[j] = x[j] / scale;
      }
      put<KV, VEC, NEIGHBOURS>(static_cast<typename KV::Raw*>(a.pool[kind - 1u]) + s_row[kind - 1u][t] +
                                   (int64_t)head * a.pool_stride[kind - 1u][2],
                               d0, d1, x);
    }
  }
}

template <class X, class KV>
hipError_t launch(AppendArgs a, bool neighbours, uint32_t vec, hipStream_t s) {
  const uint32_t row = a.dim / (2u * vec), units = row * (a.q_heads + 2u * a.heads);
  a.by_row = FastDiv::of(row);
  a.by_token = FastDiv::of(units);
  // One token, or as many as give every thread a unit. (256 tokens of 384
  // units 4.4 us, two of them a workgroup 5.0, four 6.8; 16384 69, 72, 74.)
  a.tokens_per_group = min(max(kThreads / units, 1u), kMaxTokens);
  const dim3 grid((a.T + a.tokens_per_group - 1u) / a.tokens_per_group);
  const auto go = [&](auto v, auto n) {
    constexpr int VEC = decltype(v)::value;
    hipLaunchKernelGGL((append_kernel<X, KV, VEC, decltype(n)::value>), grid, dim3(kThreads), 0, s, a);
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

hipError_t launch_kv_append(const AppendArgs& a, uint32_t dtype, uint32_t kv_dtype, bool neighbours, uint32_t vec,
                            hipStream_t s) {
  const bool e4m3 = kv_dtype == LLMHIP_E4M3;
  switch (dtype) {
    case LLMHIP_F32: return e4m3 ? launch<F32, E4M3>(a, neighbours, vec, s) : launch<F32, F32>(a, neighbours, vec, s);
    case LLMHIP_BF16: return e4m3 ? launch<BF16, E4M3>(a, neighbours, vec, s) : launch<BF16, BF16>(a, neighbours, vec, s);
    default: return e4m3 ? launch<F16, E4M3>(a, neighbours, vec, s) : launch<F16, F16>(a, neighbours, vec, s);
  }
}

}  // namespace llmhip
