// Pages, slots and positions for the tokens of the next step
// (llmhip_kv_plan).
//
// Requests are served in order, so what request r gets follows from sums
// over the requests before it: of their tokens, of the pages that they need
// and of the pages that they give back. Every workgroup forms the three
// prefix sums, 1024 requests at a time, in 64 bits, rather than waiting for one
// that does; each then takes a part of the tokens, which find their request
// by bisection of the sums in LDS, and of the released requests. Nothing that
// one workgroup writes is read by another: a new page's id comes from the
// ring, not from the table, and ids go back to the ring behind the free ones.
// What bounds it is latency: two rounds of dependent reads and three
// barriers for each 1024 requests.
#include "kv_args.h"
#include "wave_ops.h"

namespace llmhip {
namespace {

template <int CTRL, int ROW_MASK = 0xf>
__device__ __forceinline__ uint64_t dpp0_u64(uint64_t x) {
  return ((uint64_t)dpp0<CTRL, ROW_MASK>((uint32_t)(x >> 32)) << 32) | dpp0<CTRL, ROW_MASK>((uint32_t)x);
}

// wave_incl_scan in 64 bits.
__device__ __forceinline__ uint64_t wave_incl_scan_u64(uint64_t x) {
  x += dpp0_u64<0x111>(x);
  x += dpp0_u64<0x112>(x);
  x += dpp0_u64<0x114>(x);
  x += dpp0_u64<0x118>(x);
  x += dpp0_u64<0x142, 0xa>(x);
  x += dpp0_u64<0x143, 0xc>(x);
  return x;
}

// Inclusive prefix sums over the workgroup's threads of two values at once,
// and their totals. `waves`: LDS that nothing else uses until the next barrier.
template <uint32_t WAVES>
__device__ __forceinline__ void group_scan(uint64_t& x, uint64_t& y, uint64_t (*waves)[WAVES], uint64_t& x_total, uint64_t& y_total) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  x = wave_incl_scan_u64(x);
  y = wave_incl_scan_u64(y);
  if (lane == 63u) {
    waves[0][wave] = x;
    waves[1][wave] = y;
  }
  __syncthreads();
  const uint64_t xs = wave_incl_scan_u64(lane < WAVES ? waves[0][lane] : 0u);
  const uint64_t ys = wave_incl_scan_u64(lane < WAVES ? waves[1][lane] : 0u);
  x_total = readlane_u64(xs, WAVES - 1u);
  y_total = readlane_u64(ys, WAVES - 1u);
  x += wave ? readlane_u64(xs, wave - 1u) : 0u;
  y += wave ? readlane_u64(ys, wave - 1u) : 0u;
}

// A place in a ring; at most one turn past it unless the pool's state is wrong.
__device__ __forceinline__ uint32_t in_ring(uint64_t x, uint32_t pages) {
  if (x < pages) return (uint32_t)x;
  x -= pages;
  return (uint32_t)(x < pages ? x : x % pages);
}

template <uint32_t kThreads>
__global__ __launch_bounds__(kThreads) void plan_kernel(PlanArgs a) {
  constexpr uint32_t kWaves = kThreads / 64u;
  __shared__ uint64_t s_waves[2][2][kWaves];
  __shared__ uint32_t s_end[kThreads];    // tokens asked for up to and with each request, at most T + 1
  __shared__ uint32_t s_begin[kThreads];  // and before it
  __shared__ uint32_t s_base[kThreads];   // its tokens before this call
  __shared__ uint32_t s_first[kThreads];  // where its new pages start in the ring
  __shared__ uint32_t s_took[kThreads];   // how many they are
  __shared__ uint32_t s_back[kThreads];   // pages that it gives back
  __shared__ uint32_t s_put[kThreads];    // where they go in the ring
  __shared__ uint32_t s_ok[kThreads];
  __shared__ unsigned long long s_taken;  // pages handed out
  const uint32_t tid = threadIdx.x;
  const uint64_t cap = (uint64_t)a.table_pages * a.page;
  const uint32_t most = cap > 0x7fffffffu ? 0x7fffffffu : (uint32_t)cap;
  bool bad = false;
  uint32_t head = (uint32_t)a.free_state[0], count = (uint32_t)a.free_state[1];
  if (head >= a.pages || count > a.pages) {
    bad = true;
    head = 0u;
    count = 0u;
  }
  uint64_t asked = 0, needed = 0, returned = 0;
  if (tid == 0u) s_taken = 0ull;
  const bool sums = a.requests && blockIdx.x == 0u;  // this workgroup writes what is one value a request
  if (sums && tid == 0u) a.start[0] = 0;
  for (uint32_t r0 = 0; r0 < a.R; r0 += kThreads) {
    const uint32_t r = r0 + tid, m = min(kThreads, a.R - r0);
    uint32_t base = 0, back = 0;
    uint64_t n = 0;
    if (r < a.R) {
      const uint32_t len = clamp_len(a.lens[r], most, bad);
      const bool gone = a.release && a.release[r] != 0;
      base = gone ? 0u : len;
      back = gone ? a.by_page.div(len + a.page - 1u) : 0u;
      if (a.new_tokens) {
        const int32_t want = a.new_tokens[r];
        bad = bad || want < 0;
        n = want < 0 ? 0u : (uint32_t)want;
      } else {
        n = gone ? 0u : 1u;
      }
    }
    uint64_t n_sum, need_sum, back_sum, unused, end = n, put = back, none = 0u;
    group_scan<kWaves>(end, put, s_waves[0], n_sum, back_sum);
    end += asked;
    put += returned - back;
    const bool fits = r < a.R && base + n <= cap && end <= a.T;
    const uint32_t have = a.by_page.div(base + a.page - 1u);
    const uint32_t need = fits ? a.by_page.div(base + (uint32_t)n + a.page - 1u) - have : 0u;
    uint64_t upto = need;
    group_scan<kWaves>(upto, none, s_waves[1], need_sum, unused);
    upto += needed;
    const bool ok = fits && (need == 0u || upto <= count);
    s_end[tid] = (uint32_t)min(end, (uint64_t)a.T + 1u);
    s_begin[tid] = (uint32_t)min(end - n, (uint64_t)a.T + 1u);
    s_base[tid] = base;
    s_first[tid] = in_ring(head + (upto - need), a.pages);
    s_took[tid] = ok ? need : 0u;
    s_back[tid] = back;
    s_put[tid] = in_ring((uint64_t)head + count + put, a.pages);
    s_ok[tid] = ok;
    if (sums && r < a.R) {
      a.out_lens[r] = (int32_t)(base + (ok ? (uint32_t)n : 0u));
      a.granted[r] = ok ? (int32_t)n : 0;
      a.start[r + 1u] = (int32_t)min(end, (uint64_t)0x7fffffffu);
    }
    __syncthreads();

    // Released pages. A request that is released and prompted anew gets its
    // new pages here as well, each place read before it is written.
    if (a.release && a.requests) {
      for (uint32_t i = blockIdx.x * kWaves + (tid >> 6); i < m; i += gridDim.x * kWaves) {
        const uint32_t back_i = s_back[i], fresh = back_i ? s_took[i] : 0u;
        int32_t* row = a.table + (uint64_t)(r0 + i) * a.table_ld;
        for (uint32_t p = tid & 63u; p < max(back_i, fresh); p += 64u) {
          if (p < back_i) {
            const int32_t id = row[p];
            bad = bad || (uint32_t)id >= a.pages;
            a.ring[in_ring((uint64_t)s_put[i] + p, a.pages)] = id;
          }
          if (p < fresh) row[p] = a.ring[in_ring((uint64_t)s_first[i] + p, a.pages)];
        }
      }
    }

    const uint32_t lo = (uint32_t)min(asked, (uint64_t)a.T), hi = (uint32_t)min(asked + n_sum, (uint64_t)a.T);
    for (uint32_t t = lo + blockIdx.x * kThreads + tid; a.tokens && t < hi; t += gridDim.x * kThreads) {
      uint32_t i = 0, above = m;  // the first request whose sum passes t
      while (i < above) {
        const uint32_t mid = (i + above) >> 1;
        if (s_end[mid] > t) above = mid;
        else i = mid + 1u;
      }
      int64_t slot = -1;
      uint32_t pos = 0;
      if (s_ok[i]) {
        pos = s_base[i] + (t - s_begin[i]);
        const uint32_t p = a.by_page.div(pos), have_i = a.by_page.div(s_base[i] + a.page - 1u);
        int32_t* entry = a.table + (uint64_t)(r0 + i) * a.table_ld + p;
        int32_t id;
        if (p >= have_i) {
          id = a.ring[in_ring((uint64_t)s_first[i] + (p - have_i), a.pages)];
          if (pos == p * a.page && !s_back[i]) *entry = id;  // a page's first token enters it
        } else {
          id = *entry;
        }
        if ((uint32_t)id < a.pages) slot = (int64_t)id * a.page + (pos - p * a.page);
        else bad = true;
      }
      a.slots[t] = slot;
      a.positions[t] = (int32_t)pos;
    }
    // The requests that got pages are the first of those that need some, so
    // the largest of their sums is what the chunk took: the last one's.
    const uint64_t got = __ballot(ok && need);
    if (sums && got) {
      const uint64_t mine = readlane_u64(upto, 63u - (uint32_t)__builtin_clzll(got));
      if ((tid & 63u) == 0u) atomicMax(&s_taken, (unsigned long long)mine);
    }
    asked += n_sum;
    needed += need_sum;
    returned += back_sum;
    __syncthreads();
  }

  for (uint32_t t = (uint32_t)min(asked, (uint64_t)a.T) + blockIdx.x * kThreads + tid; a.tokens && t < a.T;
       t += gridDim.x * kThreads) {
    a.slots[t] = -1;
    a.positions[t] = 0;
  }
  if (sums && tid == 0u) {
    const uint64_t taken = s_taken;
    const uint64_t left = count - taken + returned;
    bad = bad || left > a.pages;  // pages came back that were free already
    a.out_free_state[0] = (int32_t)in_ring(head + taken, a.pages);
    a.out_free_state[1] = (int32_t)min(left, (uint64_t)a.pages);
  }
  if (__any(bad) && (tid & 63u) == 0u) atomicOr(a.status, LLMHIP_KSTATUS_BAD_INDEX);
}

}  // namespace

namespace {

template <uint32_t THREADS>
hipError_t launch(PlanArgs a, hipStream_t s) {
  // A thread for each token, a wave for each 8 requests (few are released).
  const uint32_t groups = min(max(max((a.T + THREADS - 1u) / THREADS, (a.R + THREADS / 8u - 1u) / (THREADS / 8u)), 1u), 256u);
  a.tokens = a.requests = true;
  if (groups > 1u && (a.lens == a.out_lens || a.free_state == a.out_free_state)) {
    // What every workgroup reads is to change in place: the tokens first.
    a.requests = false;
    hipLaunchKernelGGL(plan_kernel<THREADS>, dim3(groups), dim3(THREADS), 0, s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    a.tokens = false;
    a.requests = true;
    hipLaunchKernelGGL(plan_kernel<THREADS>, dim3(1), dim3(THREADS), 0, s, a);
  } else {
    hipLaunchKernelGGL(plan_kernel<THREADS>, dim3(groups), dim3(THREADS), 0, s, a);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_kv_plan(const PlanArgs& a, hipStream_t s) {
  return a.R <= 256u ? launch<256>(a, s) : launch<1024>(a, s);
}

}  // namespace llmhip
