// Tokens' keys and values out of a cache of codes (llmhip_kv_block_read).
//
// A unit is 16 bytes of one head row that is read, key or value: a load of its 4
// or 8 codes, one scale that the row's other lanes read too, and a store past the
// L2, whole lines of neighbouring lanes. A thread has up to 4 units' loads on
// their way. What bounds it is the traffic: 65536 tokens of 8 heads of 128 as
// bfloat16 70 us, 5.8 TB/s (one unit a thread and stores through the L2: 106).
#include <algorithm>

#include "kv_args.h"
#include "kv_types.h"

namespace llmhip {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kMaxTokens = 64;

// Values of a unit.
template <class X>
constexpr int kValues = 16 / sizeof(typename X::Raw);

template <class X, class KV, uint32_t UNITS>
__global__ __launch_bounds__(kThreads) void block_read_kernel(BlockReadArgs a) {
  __shared__ uint32_t s_page[kMaxTokens], s_token[kMaxTokens];
  const uint32_t tid = threadIdx.x, t0 = blockIdx.x * a.tokens_per_group, n = min(a.tokens_per_group, a.T - t0);
  if (tid < n) {
    uint32_t p = 0, t = 0;
    bool bad = false;
    const int64_t slot = a.slots[t0 + tid];
    const bool live = a.short_slots ? split_short_slot(slot, a.pages, a.by_page, p, t, bad) : split_slot(slot, a.pages, a.page, p, t, bad);
    if (bad) atomicOr(a.status, LLMHIP_KSTATUS_BAD_INDEX);
    s_page[tid] = live ? p : 0xffffffffu;
    s_token[tid] = t;
  }
  __syncthreads();
  for (uint32_t u0 = tid; u0 < n * a.by_token.d; u0 += UNITS * kThreads) {
    Pack<KV, kValues<X>> in[UNITS];
    float scale[UNITS];
    typename X::Raw* to[UNITS];
#pragma unroll
    for (uint32_t k = 0; k < UNITS; ++k) {
      const uint32_t u = min(u0 + k * kThreads, n * a.by_token.d - 1u);
      const uint32_t t = a.by_token.div(u), in_token = u - t * a.by_token.d, page = s_page[t], token = s_token[t];
      uint32_t head = a.by_row.div(in_token);
      const uint32_t d = (in_token - head * a.by_row.d) * kValues<X>;
      const uint32_t kind = head >= a.heads || !a.out[0] ? 1u : 0u;
      head -= head >= a.heads ? a.heads : 0u;
      in[k] = Pack<KV, kValues<X>>{};
      scale[k] = 0.0f;
      if (page != 0xffffffffu) {
        in[k] = *reinterpret_cast<const Pack<KV, kValues<X>>*>(static_cast<const typename KV::Raw*>(a.pool[kind]) +
                                                               (int64_t)page * a.pool_stride[kind][0] +
                                                               (int64_t)token * a.pool_stride[kind][1] +
                                                               (int64_t)head * a.pool_stride[kind][2] + d);
        scale[k] = a.block_scales.scale[kind][(int64_t)page * a.block_scales.stride[kind][0] +
                                              (int64_t)a.block_scales.by_block.div(token) * a.block_scales.stride[kind][1] +
                                              (int64_t)head * a.block_scales.stride[kind][2]];
      }
      to[k] = static_cast<typename X::Raw*>(a.out[kind]) + (int64_t)(t0 + t) * a.out_stride[kind][0] +
              (int64_t)head * a.out_stride[kind][1] + d;
    }
#pragma unroll
    for (uint32_t k = 0; k < UNITS; ++k) {
      if (k && u0 + k * kThreads >= n * a.by_token.d) continue;
      Pack<X, kValues<X>> x;
#pragma unroll
      for (int j = 0; j < kValues<X>; ++j) {
        float y = KV::load(in[k].v[j]) * scale[k];
        asm("" : "+v"(y));  // the product in binary32 for every type (else one instruction rounds it to float16)
        x.v[j] = X::store(y);
      }
      using W = uint32_t __attribute__((ext_vector_type(4)));
      typedef W __attribute__((aligned(2))) Placed;  // rows of any alignment
      __builtin_nontemporal_store(__builtin_bit_cast(W, x), reinterpret_cast<Placed*>(to[k]));
    }
  }
}

template <class X, class KV>
hipError_t launch(BlockReadArgs a, hipStream_t s) {
  const uint32_t row = a.dim / kValues<X>, units = row * a.heads * ((a.out[0] != nullptr) + (a.out[1] != nullptr));
  a.by_row = FastDiv::of(row);
  a.by_token = FastDiv::of(units);
  a.by_page = FastDiv::of(a.page);
  a.short_slots = (uint64_t)a.pages * a.page <= 0x7fffffffu;
  // One unit a thread where few workgroups are, else four.
  const bool many = (uint64_t)a.T * units >= 4096u * kThreads;
  a.tokens_per_group = std::min(std::max((many ? 4u : 1u) * kThreads / units, 1u), kMaxTokens);
  const dim3 grid((a.T + a.tokens_per_group - 1u) / a.tokens_per_group);
  if (many) hipLaunchKernelGGL((block_read_kernel<X, KV, 4>), grid, dim3(kThreads), 0, s, a);
  else hipLaunchKernelGGL((block_read_kernel<X, KV, 1>), grid, dim3(kThreads), 0, s, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_kv_block_read(const BlockReadArgs& a, uint32_t dtype, uint32_t kv_dtype, hipStream_t s) {
  const bool i8 = kv_dtype == LLMHIP_I8;
  switch (dtype) {
    case LLMHIP_F32: return i8 ? launch<F32, I8>(a, s) : launch<F32, E4M3>(a, s);
    case LLMHIP_BF16: return i8 ? launch<BF16, I8>(a, s) : launch<BF16, E4M3>(a, s);
    default: return i8 ? launch<F16, I8>(a, s) : launch<F16, E4M3>(a, s);
  }
}

}  // namespace llmhip
