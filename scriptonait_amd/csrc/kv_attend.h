// Attention of one new token over its request's pages (llmhip_kv_attend).
//
// With s_t the scores in base-2 exponents and m a reference that no score
// passes by more than 8, a run of tokens is held as
//   m,  l = sum 2^(s_t - m),  o = sum 2^(s_t - m) v_t,
// runs are joined by l = sum_k l_k 2^(m_k - M), o likewise, and the answer
// is o / l. m moves only when a score passes it by more than 8: the
// numerators then stay below 2^8 and the largest is at least 1, and most
// tiles neither compare across lanes nor scale o.
//
// The work is every request's tiles of tokens in one line, cut into equal
// ranges, so ragged lengths share the card evenly and one long request uses
// all of it. A workgroup takes one range of one cache head, its waves equal
// parts of it. A request's run inside one wave goes straight to the output;
// runs that waves of a group share are joined in LDS, and what a group
// leaves of a request that goes on elsewhere goes to the workspace, for
// join_kernel. What bounds it is reading the cache once.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv_args.h"
#include "kv_engines.h"
#include "wave_ops.h"

namespace llmhip {

constexpr uint32_t kAttendWaves = 4, kAttendThreads = kAttendWaves * 64;
constexpr float kLazyBits = 8.0f;
constexpr float kLn2 = 0.693147180559945309f, kLog2e = 1.44269504088896341f;
constexpr uint32_t kNoId = 0xffffffffu;

// A request's tiles: tile_first .. tile_first + count, the first one holding
// its window's first token.
__device__ __forceinline__ uint32_t tiles_of(uint32_t len, uint32_t window, uint32_t tile, uint32_t& first) {
  first = window_start(len, window) / tile;
  return len ? (len + tile - 1u) / tile - first : 0u;
}

// Inclusive prefix sum over the workgroup's threads, and the total. `waves`:
// kAttendWaves words of LDS.
__device__ __forceinline__ uint32_t group_scan(uint32_t x, uint32_t* waves, uint32_t& total) {
  const uint32_t lane = lane_id(), wave = threadIdx.x >> 6;
  x = wave_incl_scan(x);
  if (lane == 63u) waves[wave] = x;
  __syncthreads();
  total = 0u;
  uint32_t before = 0u;
#pragma unroll
  for (uint32_t w = 0; w < kAttendWaves; ++w) {
    before += w < wave ? waves[w] : 0u;
    total += waves[w];
  }
  __syncthreads();
  return x + before;
}

template <class E, bool GROUPED>
struct Run {
  static constexpr int kIds = GROUPED ? 1 : E::kGroup;       // page ids of the lane's V tokens
  static constexpr int kKIds = GROUPED ? 1 : E::kProducts;   // and of its K tokens
  const AttendArgs& a;
  const int32_t* row;   // the request's table
  const char* base[2];  // the pools at the cache head
  uint32_t g, c, lo, hi;  // the lane, and the tokens that are seen
  float scale;            // of a score, in base-2 exponents
  E e;
  float ref, limit, sum;  // m (0 before the first finite score), m + 8, the lane's part of l
  bool bad = false;
  struct Ids {
    uint32_t k[kKIds], v[kIds];
  };

  __device__ __forceinline__ Run(const AttendArgs& args) : a(args) {}

  // First of the lane's tokens in a tile: V's group, and K's in product p.
  __device__ __forceinline__ uint32_t v_token(uint32_t t0) const { return t0 + E::kGroup * g; }
  __device__ __forceinline__ uint32_t k_token(uint32_t t0, uint32_t p) const {
    return t0 + E::kGroup * (c >> 2) + 4u * p + (c & 3u);
  }

  __device__ __forceinline__ uint32_t page_id(uint32_t t, uint32_t width) const {
    return t < hi && t + width > lo ? (uint32_t)row[a.by_page.div(t)] : kNoId;
  }
  __device__ __forceinline__ Ids fetch_ids(uint32_t t0) const {
    Ids x;
    if constexpr (GROUPED) {
      x.k[0] = page_id(t0 + E::kGroup * (c >> 2), E::kGroup);
      x.v[0] = page_id(v_token(t0), E::kGroup);
    } else {
#pragma unroll
      for (int p = 0; p < kKIds; ++p) x.k[p] = page_id(k_token(t0, p), 1u);
#pragma unroll
      for (int i = 0; i < kIds; ++i) x.v[i] = page_id(v_token(t0) + i, 1u);
    }
    return x;
  }

  // Where token t of page id starts; a token that is not seen leads to the
  // pool's first page.
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
      for (int i = 0; i < E::kGroup; ++i) e.load_v(i, p + i * step, c, a.dim);
    } else {
#pragma unroll
      for (int i = 0; i < E::kGroup; ++i) e.load_v(i, token_row(1, x.v[i], a.by_page.mod(t + i)), c, a.dim);
    }
  }
  // Which of the lane's tokens are seen, as bits; kAll in every lane of most tiles.
  static constexpr uint32_t kAll = (1u << E::kGroup) - 1u;
  __device__ __forceinline__ uint32_t seen_of(uint32_t t0, const Ids& x) {
    bool outside = t0 < lo || t0 + E::kTile > hi;
#pragma unroll
    for (int i = 0; i < kIds; ++i) outside = outside || x.v[i] >= a.pages;
    if (!__any(outside)) return kAll;
    uint32_t seen = 0u;
#pragma unroll
    for (int i = 0; i < E::kGroup; ++i) {
      const uint32_t t = v_token(t0) + i, id = x.v[GROUPED ? 0 : i];
      const bool in = t >= lo && t < hi;
      bad = bad || (in && id >= a.pages);
      seen |= in && id < a.pages ? 1u << i : 0u;
    }
    return seen;
  }

  // Tiles first .. last of the request. A tile's keys are loaded when the
  // tile before has used its own, its values likewise, and its page ids two
  // tiles ahead, so that no wait for one of them includes a younger load.
  __device__ __forceinline__ void tiles(uint32_t first, uint32_t last) {
    ref = 0.0f;
    limit = -INFINITY;
    sum = 0.0f;
    e.clear();
    Ids next = fetch_ids(first * E::kTile);
    load_keys(first * E::kTile, next);
    load_values(first * E::kTile, next);
    uint32_t seen = seen_of(first * E::kTile, next);
    if (first + 1u < last) next = fetch_ids((first + 1u) * E::kTile);
    for (uint32_t tile = first; tile < last; ++tile) {
      const uint32_t t1 = (tile + 1u) * E::kTile;
      const bool more = tile + 1u < last;
      Ids after = next;
      if (tile + 2u < last) after = fetch_ids(t1 + E::kTile);
      float s[E::kGroup];
      e.scores(s, g, a.dim);
      if (more) load_keys(t1, next);
#pragma unroll
      for (int i = 0; i < E::kGroup; ++i) s[i] *= scale;
      if (__any(seen != kAll)) {
#pragma unroll
        for (int i = 0; i < E::kGroup; ++i) {
          if (!(seen >> i & 1u)) {
            s[i] = -INFINITY;
            e.drop_v(i);
          }
        }
      }
      float top = s[0];
#pragma unroll
      for (int i = 1; i < E::kGroup; ++i) top = fmaxf(top, s[i]);
      if (__any(top > limit)) raise(top);
#pragma unroll
      for (int i = 0; i < E::kGroup; ++i) {
        s[i] = __builtin_amdgcn_exp2f(s[i] - ref);
        sum += s[i];
      }
      e.accumulate(s);
      if (more) {
        load_values(t1, next);
        seen = seen_of(t1, next);
      }
      next = after;
    }
  }

  // Moves the reference of each query head to its largest score.
  __device__ __forceinline__ void raise(float top) {
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const bool fresh = limit == -INFINITY, up = top > (fresh ? -INFINITY : ref);
    const float next = up ? top : ref;
    const float keep = fresh || !up ? 1.0f : __builtin_amdgcn_exp2f(ref - next);
    ref = next;
    limit = up || !fresh ? next + kLazyBits : -INFINITY;
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

// Words of a partial answer: o of every query head, then m, then l.
__host__ __device__ __forceinline__ uint32_t partial_words(uint32_t group, uint32_t dim) { return group * (dim + 2u); }

template <class E, bool GROUPED>
__global__ __launch_bounds__(kAttendThreads) void attend_kernel(AttendArgs a) {
  extern __shared__ uint32_t s_mem[];
  __shared__ uint32_t s_waves[kAttendWaves];
  __shared__ int32_t s_slot[2 * kAttendWaves];  // the request of each partial answer, or -1
  uint32_t* s_start = s_mem;                    // split: where each request's tiles begin
  float* s_part = reinterpret_cast<float*>(s_mem + a.start_words);

  const uint32_t tid = threadIdx.x, lane = lane_id(), wave = readlane_u32(tid >> 6, 0);
  const uint32_t vhead = blockIdx.x % a.vheads, range = blockIdx.x / a.vheads;
  const uint32_t head = vhead / a.blocks, q0 = vhead % a.blocks * 16u;  // first query head inside the group
  const uint32_t group = min(16u, a.group - q0);
  const uint32_t most = a.table_pages * a.page;
  bool bad = false;

  // The range of tiles: [begin, end) of the line of all tiles (split), or
  // one request's.
  uint32_t begin, end, b = 0;
  if (a.ranges) {
    uint32_t total = 0;
    for (uint32_t r0 = 0; r0 < a.B; r0 += kAttendThreads) {
      const uint32_t r = r0 + tid;
      uint32_t first, n = 0, sum;
      if (r < a.B) n = tiles_of(clamp_len(a.lens[r], most, bad), a.window, E::kTile, first);
      const uint32_t upto = total + group_scan(n, s_waves, sum);
      if (r < a.B) s_start[r] = upto - n;
      total += sum;
    }
    if (tid == 0u) s_start[a.B] = total;
    __syncthreads();
    const uint32_t quota = max((total + a.ranges - 1u) / a.ranges, kAttendWaves);
    if (blockIdx.x == 0u)
      for (uint32_t r = tid; r <= a.B; r += kAttendThreads) reinterpret_cast<uint32_t*>(a.workspace)[r] = s_start[r];
    begin = min(range * quota, total);
    end = min(begin + quota, total);
  } else {
    uint32_t first;
    b = range;
    begin = 0u;
    end = tiles_of(clamp_len(a.lens[b], most, bad), a.window, E::kTile, first);
  }
  if (tid < 2u * kAttendWaves) s_slot[tid] = -1;
  __syncthreads();
  if (bad && vhead == 0u && (range == 0u || !a.ranges)) atomicOr(a.status, LLMHIP_KSTATUS_BAD_INDEX);
  bad = false;

  Run<E, GROUPED> run(a);
  run.g = lane >> 4;
  run.c = lane & 15u;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    run.base[i] = static_cast<const char*>(a.pool[i]) + (int64_t)head * a.pool_stride[i][2] * E::kElem;
  const bool e4m3 = E::KV::kId == LLMHIP_E4M3;
  run.scale = a.score_scale * kLog2e * (e4m3 ? a.scale[0][head] : 1.0f);
  const float vscale = e4m3 ? a.scale[1][head] : 1.0f;
  const uint32_t qhead = head * a.group + q0;  // of the output
  const uint32_t words = partial_words(group, a.dim);

  uint32_t tile = begin + (end - begin) * wave / kAttendWaves;
  const uint32_t stop = begin + (end - begin) * (wave + 1u) / kAttendWaves;
  if (a.ranges && tile < stop) {
    uint32_t i = 0, above = a.B;  // the last request that begins at or before the tile
    while (above - i > 1u) {
      const uint32_t mid = (i + above) >> 1;
      if (s_start[mid] <= tile) i = mid;
      else above = mid;
    }
    b = readlane_u32(i, 0);
  }
  bool first_run = true;
  while (tile < stop) {
    uint32_t from = 0u, to = end;
    if (a.ranges) {
      from = s_start[b];
      to = s_start[b + 1u];
      if (to <= tile) {  // an empty request
        ++b;
        continue;
      }
    }
    uint32_t zero_tile;
    bool clamped = false;
    const uint32_t len = clamp_len(a.lens[b], most, clamped);
    tiles_of(len, a.window, E::kTile, zero_tile);
    const uint32_t last = min(stop, to);
    run.row = a.table + (uint64_t)b * a.table_ld;
    run.lo = window_start(len, a.window);
    run.hi = len;
    const typename E::Q::Raw* q = static_cast<const typename E::Q::Raw*>(a.q) + (int64_t)b * a.q_stride[0] +
                                  (int64_t)(qhead + (run.c < group ? run.c : 0u)) * a.q_stride[1];
    run.e.load_q(q, run.g, a.dim, run.c < group, a.wide);
    run.tiles(zero_tile + (tile - from), zero_tile + (last - from));
    const float l = run.total(), m = l == 0.0f ? -INFINITY : run.ref;
    if (tile == from && last == to) {  // all of the request
      const float inv = l == 0.0f ? 0.0f : vscale / l;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t qi = 4u * run.g + i;
        const float scale = __shfl(inv, qi, 64);
        if (qi >= group) continue;
        typename E::Q::Raw* out = static_cast<typename E::Q::Raw*>(a.out) + (int64_t)b * a.out_stride[0] +
                                  (int64_t)(qhead + qi) * a.out_stride[1];
#pragma unroll
        for (uint32_t p = 0; p < E::kPanels; ++p) {
          const uint32_t d = (p * 16u + run.c) * E::kVec;
          if (d >= a.dim) continue;
          Pack<typename E::Q, E::kVec> x;
#pragma unroll
          for (int j = 0; j < E::kVec; ++j) x.v[j] = E::Q::store(run.e.o[p][j][i] * scale);
          if (a.wide) {
            *reinterpret_cast<Pack<typename E::Q, E::kVec>*>(out + d) = x;
          } else {
#pragma unroll
            for (int j = 0; j < E::kVec; ++j) out[d + j] = x.v[j];
          }
        }
      }
      if (a.lse && lane < group) a.lse[(uint64_t)b * a.q_heads + qhead + lane] = lse_of(m, l);
    } else {
      const uint32_t slot = 2u * wave + (first_run ? 0u : 1u);
      float* part = s_part + slot * words;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t qi = 4u * run.g + i;
        if (qi >= group) continue;
#pragma unroll
        for (uint32_t p = 0; p < E::kPanels; ++p) {
          const uint32_t d = (p * 16u + run.c) * E::kVec;
          if (d >= a.dim) continue;
#pragma unroll
          for (int j = 0; j < E::kVec; ++j) part[qi * a.dim + d + j] = run.e.o[p][j][i];
        }
      }
      if (lane < group) {
        part[group * a.dim + lane] = m;
        part[group * (a.dim + 1u) + lane] = l;
      }
      if (lane == 0u) s_slot[slot] = (int32_t)b;
    }
    first_run = false;
    tile = last;
    ++b;
  }
  if (__any(run.bad) && lane == 0u) atomicOr(a.status, LLMHIP_KSTATUS_BAD_INDEX);
  __syncthreads();

  // Join neighbouring partial answers of a request. At most two of the
  // group's requests go on outside its range.
  for (uint32_t i = 0; i < 2u * kAttendWaves;) {
    const int32_t r = s_slot[i];
    if (r < 0) {
      ++i;
      continue;
    }
    uint32_t n = i + 1u;
    while (n < 2u * kAttendWaves && (s_slot[n] == r || s_slot[n] < 0)) ++n;
    const bool before = a.ranges && s_start[r] < begin, after = a.ranges && s_start[r + 1] > end;
    float* to = a.workspace + a.part_offset + ((uint64_t)blockIdx.x * 2u + (before ? 0u : 1u)) * a.part_words;
    for (uint32_t x = tid; x < group * a.dim; x += kAttendThreads) {
      const uint32_t qi = a.by_dim.div(x), d = x - qi * a.dim;
      float m = -INFINITY, l = 0.0f, o = 0.0f;
      for (uint32_t k = i; k < n; ++k)
        if (s_slot[k] >= 0) m = fmaxf(m, s_part[k * words + group * a.dim + qi]);
      const float top = m == -INFINITY ? 0.0f : m;
      for (uint32_t k = i; k < n; ++k) {
        if (s_slot[k] < 0) continue;
        const float* part = s_part + k * words;
        const float w = __builtin_amdgcn_exp2f(part[group * a.dim + qi] - top);
        l += part[group * (a.dim + 1u) + qi] * w;
        o += part[x] * w;
      }
      if (before || after) {
        to[x] = o;
        if (d == 0u) {
          to[group * a.dim + qi] = m;
          to[group * (a.dim + 1u) + qi] = l;
        }
      } else {
        const float inv = l == 0.0f ? 0.0f : vscale / l;
        typename E::Q::Raw* out = static_cast<typename E::Q::Raw*>(a.out) + (int64_t)r * a.out_stride[0] +
                                  (int64_t)(qhead + qi) * a.out_stride[1];
        out[d] = E::Q::store(o * inv);
        if (a.lse && d == 0u) a.lse[(uint64_t)r * a.q_heads + qhead + qi] = lse_of(m, l);
      }
    }
    i = n;
  }
  if (!a.ranges && end == 0u) {  // a request of length 0
    for (uint32_t x = tid; x < group * a.dim; x += kAttendThreads) {
      const uint32_t qi = a.by_dim.div(x), d = x - qi * a.dim;
      static_cast<typename E::Q::Raw*>(a.out)[(int64_t)b * a.out_stride[0] + (int64_t)(qhead + qi) * a.out_stride[1] + d] =
          E::Q::store(0.0f);
      if (a.lse && d == 0u) a.lse[(uint64_t)b * a.q_heads + qhead + qi] = -INFINITY;
    }
  }
}

// The answers of requests that several ranges share, and of empty ones. One
// workgroup for each request and query head; the partial answers are joined
// in the ranges' order.
template <class Q, class KV>
__global__ __launch_bounds__(256) void join_kernel(AttendArgs a) {
  __shared__ float s_weight[kMaxRanges];
  __shared__ float s_wave[2][4];
  __shared__ f32x4 s_sum[256];
  const uint32_t tid = threadIdx.x, lane = lane_id(), wave = tid >> 6, b = blockIdx.y, qh = blockIdx.x;
  const uint32_t* start = reinterpret_cast<const uint32_t*>(a.workspace);
  const uint32_t total = start[a.B], from = start[b], to = start[b + 1u];
  const uint32_t quota = max((total + a.ranges - 1u) / a.ranges, kAttendWaves);
  typename Q::Raw* out = static_cast<typename Q::Raw*>(a.out) + (int64_t)b * a.out_stride[0] + (int64_t)qh * a.out_stride[1];
  if (from == to) {
    if (tid < a.dim) out[tid] = Q::store(0.0f);
    if (a.lse && tid == 0u) a.lse[(uint64_t)b * a.q_heads + qh] = -INFINITY;
    return;
  }
  const uint32_t r0 = from / quota, n = (to - 1u) / quota - r0 + 1u;
  if (n == 1u) return;
  const uint32_t head = qh / a.group, in_group = qh % a.group, vhead = head * a.blocks + in_group / 16u;
  const uint32_t group = min(16u, a.group - in_group / 16u * 16u), qi = in_group % 16u;
  const auto part = [&](uint32_t k) {
    return a.workspace + a.part_offset + (((uint64_t)(r0 + k) * a.vheads + vhead) * 2u + (k ? 0u : 1u)) * a.part_words;
  };
  float m = -INFINITY;
  for (uint32_t k = tid; k < n; k += 256u) m = fmaxf(m, part(k)[group * a.dim + qi]);
#pragma unroll
  for (uint32_t off = 32; off; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
  if (lane == 0u) s_wave[0][wave] = m;
  __syncthreads();
  m = fmaxf(fmaxf(s_wave[0][0], s_wave[0][1]), fmaxf(s_wave[0][2], s_wave[0][3]));
  const float top = m == -INFINITY ? 0.0f : m;
  float l = 0.0f;
  for (uint32_t k = tid; k < n; k += 256u) {
    const float w = __builtin_amdgcn_exp2f(part(k)[group * a.dim + qi] - top);
    s_weight[k] = w;
    l += part(k)[group * (a.dim + 1u) + qi] * w;
  }
#pragma unroll
  for (uint32_t off = 32; off; off >>= 1) l += __shfl_xor(l, off, 64);
  if (lane == 0u) s_wave[1][wave] = l;
  __syncthreads();
  l = (s_wave[1][0] + s_wave[1][1]) + (s_wave[1][2] + s_wave[1][3]);
  // dim / 4 threads take a partial answer's values, the rest others'.
  const uint32_t across = a.dim / 4u, share = 256u / across, mine = tid / across, d = (tid - mine * across) * 4u;
  f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  if (mine < share)
    for (uint32_t k = mine; k < n; k += share)
      o += *reinterpret_cast<const f32x4*>(part(k) + qi * a.dim + d) * s_weight[k];
  s_sum[tid] = o;
  __syncthreads();
  if (mine == 0u) {
    for (uint32_t k = 1; k < share; ++k) o += s_sum[k * across + tid];
    const float vscale = KV::kId == LLMHIP_E4M3 ? a.scale[1][head] : 1.0f, inv = l == 0.0f ? 0.0f : vscale / l;
#pragma unroll
    for (int j = 0; j < 4; ++j) out[d + j] = Q::store(o[j] * inv);
  }
  if (a.lse && tid == 0u) a.lse[(uint64_t)b * a.q_heads + qh] = lse_of(m, l);
}

template <class E>
hipError_t launch_attend_engine(const AttendArgs& a, hipStream_t s) {
  const dim3 grid((a.ranges ? a.ranges : a.B) * a.vheads);
  const uint32_t lds = (a.start_words + 2u * kAttendWaves * partial_words(min(16u, a.group), a.dim)) * 4u;
  if (a.page % E::kGroup == 0u)
    hipLaunchKernelGGL((attend_kernel<E, true>), grid, dim3(kAttendThreads), lds, s, a);
  else
    hipLaunchKernelGGL((attend_kernel<E, false>), grid, dim3(kAttendThreads), lds, s, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !a.ranges) return e;
  hipLaunchKernelGGL((join_kernel<typename E::Q, typename E::KV>), dim3(a.q_heads, a.B), dim3(256), 0, s, a);
  return hipGetLastError();
}

template <template <int, bool> class E>
hipError_t launch_attend_dims(const AttendArgs& a, hipStream_t s) {
  if (a.dim == 64u) return launch_attend_engine<E<64, true>>(a, s);
  if (a.dim == 128u) return launch_attend_engine<E<128, true>>(a, s);
  if (a.dim < 64u) return launch_attend_engine<E<64, false>>(a, s);
  if (a.dim < 128u) return launch_attend_engine<E<128, false>>(a, s);
  return launch_attend_engine<E<256, false>>(a, s);
}

}  // namespace llmhip
