// Attention of one new token over its request's pages (llmhip_kv_attend).
//
// One wave for each request and query head, 64 tokens a step: each lane
// forms one token's score, the wave moves the running maximum m and sum l,
// and each lane then adds the step's rows to its own values of the output,
//   o' = o exp(m - m') + sum exp(s_t - m') v_t.
#include "kv_args.h"
#include "kv_types.h"
#include "wave_ops.h"

namespace llmhip {
namespace {

__device__ __forceinline__ float wave_max_f32(float x) {
#pragma unroll
  for (uint32_t off = 32; off; off >>= 1) x = fmaxf(x, __shfl_xor(x, off, 64));
  return x;
}
__device__ __forceinline__ float wave_sum_f32(float x) {
#pragma unroll
  for (uint32_t off = 32; off; off >>= 1) x += __shfl_xor(x, off, 64);
  return x;
}

template <class Q, class KV>
__global__ __launch_bounds__(64) void attend_kernel(AttendArgs a) {
  __shared__ float s_q[kMaxHeadDim];
  __shared__ float s_p[64];
  __shared__ int64_t s_row[64];
  const uint32_t lane = lane_id(), b = blockIdx.y, hq = blockIdx.x, h = hq / (a.q_heads / a.heads);
  const typename Q::Raw* q = static_cast<const typename Q::Raw*>(a.q) + (int64_t)b * a.q_stride[0] + (int64_t)hq * a.q_stride[1];
  for (uint32_t d = lane; d < a.dim; d += 64u) s_q[d] = Q::load(q[d]);
  __syncthreads();
  bool bad = false;
  const uint32_t len = clamp_len(a.lens[b], a.table_pages * a.page, bad);
  const float scale = a.score_scale * (KV::kId == LLMHIP_E4M3 ? a.scale[0][h] : 1.0f);
  const typename KV::Raw* kp = static_cast<const typename KV::Raw*>(a.pool[0]) + (int64_t)h * a.pool_stride[0][2];
  const typename KV::Raw* vp = static_cast<const typename KV::Raw*>(a.pool[1]) + (int64_t)h * a.pool_stride[1][2];
  float m = -INFINITY, l = 0.0f, o[kMaxHeadDim / 64] = {};
  for (uint32_t t0 = window_start(len, a.window); t0 < len; t0 += 64u) {
    const uint32_t t = t0 + lane;
    float s = -INFINITY;
    int64_t vrow = -1;
    if (t < len) {
      const uint32_t p = a.by_page.div(t), in_page = t - p * a.page;
      const uint32_t id = (uint32_t)a.table[(uint64_t)b * a.table_ld + p];
      if (id < a.pages) {
        const typename KV::Raw* k = kp + (int64_t)id * a.pool_stride[0][0] + (int64_t)in_page * a.pool_stride[0][1];
        vrow = (int64_t)id * a.pool_stride[1][0] + (int64_t)in_page * a.pool_stride[1][1];
        float dot = 0.0f;
        for (uint32_t d = 0; d < a.dim; ++d) dot = __builtin_fmaf(s_q[d], KV::load(k[d]), dot);
        s = dot * scale;
      } else {
        bad = true;
      }
    }
    const float top = fmaxf(m, wave_max_f32(s)), ref = top == -INFINITY ? 0.0f : top;
    const float p = vrow < 0 ? 0.0f : expf(s - ref), keep = expf(m - ref);
    l = l * keep + wave_sum_f32(p);
    m = top;
    __syncthreads();
    s_p[lane] = p;
    s_row[lane] = vrow;
    __syncthreads();
#pragma unroll
    for (uint32_t c = 0; c < kMaxHeadDim / 64u; ++c) {
      const uint32_t d = c * 64u + lane;
      if (d >= a.dim) break;
      float sum = o[c] * keep;
      for (uint32_t i = 0; i < 64u; ++i)
        if (s_row[i] >= 0) sum = __builtin_fmaf(s_p[i], KV::load(vp[s_row[i] + d]), sum);
      o[c] = sum;
    }
  }
  const float vscale = KV::kId == LLMHIP_E4M3 ? a.scale[1][h] : 1.0f, inv = l == 0.0f ? 0.0f : vscale / l;
  typename Q::Raw* out = static_cast<typename Q::Raw*>(a.out) + (int64_t)b * a.out_stride[0] + (int64_t)hq * a.out_stride[1];
#pragma unroll
  for (uint32_t c = 0; c < kMaxHeadDim / 64u; ++c)
    if (c * 64u + lane < a.dim) out[c * 64u + lane] = Q::store(o[c] * inv);
  if (a.lse && lane == 0u) a.lse[(uint64_t)b * a.q_heads + hq] = m + logf(l);
  if (bad) atomicOr(a.status, LLMHIP_KSTATUS_BAD_INDEX);
}

template <class Q, class KV>
hipError_t launch(const AttendArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((attend_kernel<Q, KV>), dim3(a.q_heads, a.B), dim3(64), 0, s, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_kv_attend(const AttendArgs& a, uint32_t dtype, uint32_t kv_dtype, hipStream_t s) {
  switch (dtype) {
    case LLMHIP_F32: return launch<F32, F32>(a, s);
    case LLMHIP_BF16: return kv_dtype == LLMHIP_E4M3 ? launch<BF16, E4M3>(a, s) : launch<BF16, BF16>(a, s);
    default: return kv_dtype == LLMHIP_E4M3 ? launch<F16, E4M3>(a, s) : launch<F16, F16>(a, s);
  }
}

}  // namespace llmhip
