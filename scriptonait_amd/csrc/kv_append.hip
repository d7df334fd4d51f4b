// New tokens' keys and values into their slots and their queries rotated
// (llmhip_kv_append).
//
// A unit is 2 * VEC values of one head row: VEC pairs, or values behind the
// rotated ones. A workgroup takes a few tokens. It first computes their
// cosines and sines, once for all heads, into LDS: the angle is reduced to
// [-pi/4, pi/4] in binary64 and both series are summed there, so a far
// position is as exact as a near one.
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
    // The unit's pairs: value j of the first vector with value j of the second
    // one, or neighbours within the two.
    const bool turned = c * 2u * VEC < a.dims;
    const uint32_t d0 = NEIGHBOURS || !turned ? c * 2u * VEC : c * VEC;
    const uint32_t d1 = NEIGHBOURS || !turned ? d0 + VEC : d0 + half;
    const uint32_t kind = head < a.q_heads ? 0u : head < a.q_heads + a.heads ? 1u : 2u;
    head -= kind == 0u ? 0u : kind == 1u ? a.q_heads : a.q_heads + a.heads;
    if (kind && s_row[kind - 1u][t] < 0) continue;
    const typename X::Raw* row = static_cast<const typename X::Raw*>(a.x[kind]) +
                                 (int64_t)(t0 + t) * a.x_stride[kind][0] + (int64_t)head * a.x_stride[kind][1];
    const Pack<X, VEC> p0 = *reinterpret_cast<const Pack<X, VEC>*>(row + d0);
    const Pack<X, VEC> p1 = *reinterpret_cast<const Pack<X, VEC>*>(row + d1);
    float x[2 * VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      x[j] = X::load(p0.v[j]);
      x[VEC + j] = X::load(p1.v[j]);
    }
    if (kind < 2u && turned) {
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
      typename X::Raw* out = static_cast<typename X::Raw*>(a.out_q) + (int64_t)(t0 + t) * a.oq_stride[0] +
                             (int64_t)head * a.oq_stride[1];
      Pack<X, VEC> o0, o1;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        o0.v[j] = X::store(x[j]);
        o1.v[j] = X::store(x[VEC + j]);
      }
      *reinterpret_cast<Pack<X, VEC>*>(out + d0) = o0;
      *reinterpret_cast<Pack<X, VEC>*>(out + d1) = o1;
    } else {
      typename KV::Raw* out = static_cast<typename KV::Raw*>(a.pool[kind - 1u]) + s_row[kind - 1u][t] +
                              (int64_t)head * a.pool_stride[kind - 1u][2];
      if constexpr (KV::kId == LLMHIP_E4M3) {
        const float scale = a.scale[kind - 1u][head];
#pragma unroll
        for (int j = 0; j < 2 * VEC; ++j) x[j] = x[j] / scale;
      }
      Pack<KV, VEC> o0, o1;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        o0.v[j] = KV::store(x[j]);
        o1.v[j] = KV::store(x[VEC + j]);
      }
      *reinterpret_cast<Pack<KV, VEC>*>(out + d0) = o0;
      *reinterpret_cast<Pack<KV, VEC>*>(out + d1) = o1;
    }
  }
}

template <class X, class KV>
hipError_t launch(AppendArgs a, bool neighbours, uint32_t vec, hipStream_t s) {
  a.tokens_per_group = 2;
  const dim3 grid((a.T + a.tokens_per_group - 1u) / a.tokens_per_group);
  const uint32_t row = a.dim / (2u * vec);
  a.by_row = FastDiv::of(row);
  a.by_token = FastDiv::of(row * (a.q_heads + 2u * a.heads));
  const auto go = [&](auto v) {
    constexpr int VEC = decltype(v)::value;
    if (neighbours) hipLaunchKernelGGL((append_kernel<X, KV, VEC, true>), grid, dim3(kThreads), 0, s, a);
    else hipLaunchKernelGGL((append_kernel<X, KV, VEC, false>), grid, dim3(kThreads), 0, s, a);
  };
  if (vec == 8u) go(std::integral_constant<int, 8>{});
  else if (vec == 4u) go(std::integral_constant<int, 4>{});
  else go(std::integral_constant<int, 1>{});
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
