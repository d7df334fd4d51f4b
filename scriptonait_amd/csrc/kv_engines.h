// The tile products of the key-value cache's attention (kv_attend.h): how one
// wave loads a tile of tokens and multiplies it on the matrix cores.
//
// Both products keep every operand where the loads and the first product put
// it, so nothing moves between lanes. Lane = 16 g + c.
//   S = K Q^T: row = token, column = query head. An MFMA's A operand has row
//     c in this lane, its result columns c and rows 4 g + i. Which token a
//     row stands for is free: row 4 x + i of the a-th product is token
//     kGroup x + 4 a + i of the tile, so the results in lane (g, c) are
//     query head c's scores of tokens kGroup g .. kGroup g + kGroup - 1.
//   O = P V: row = query head, column = value. These same registers are the
//     A operand (row c, tokens of group g), and a lane's B operand is column
//     c of the same tokens: it loads kVec neighbouring values of each of its
//     group's tokens, 16 lanes a row, and the j-th product takes the j-th
//     value of each. Result columns are values c kVec + j.
// The dot products' order of d is free too: the chunk that a lane of K
// loads is the chunk that the same lane of Q loads.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "kv_args.h"
#include "kv_types.h"

namespace llmhip {

using f32x4 = float __attribute__((ext_vector_type(4)));
using u32x2 = uint32_t __attribute__((ext_vector_type(2)));
using u32x4 = uint32_t __attribute__((ext_vector_type(4)));
using bf16x2 = __bf16 __attribute__((ext_vector_type(2)));
using bf16x8 = __bf16 __attribute__((ext_vector_type(8)));
using f16x2 = _Float16 __attribute__((ext_vector_type(2)));
using f16x8 = _Float16 __attribute__((ext_vector_type(8)));

template <class T, class F>
__device__ __forceinline__ T bits_as(F x) {
  static_assert(sizeof(T) == sizeof(F), "sizes differ");
  return __builtin_bit_cast(T, x);
}

template <int BYTES>
struct RawOf;
template <>
struct RawOf<2> { using type = uint16_t; };
template <>
struct RawOf<4> { using type = uint32_t; };
template <>
struct RawOf<8> { using type = u32x2; };
template <>
struct RawOf<16> { using type = u32x4; };

// Keys: two neighbouring loads share a cache line, the first level keeps it.
// ALIGN: what the rows are aligned to, which E4M3's are to 8 bytes.
template <class T, int ALIGN = sizeof(T)>
__device__ __forceinline__ T load_key(const char* p) {
  typedef T __attribute__((aligned(ALIGN))) Placed;
  return *reinterpret_cast<const Placed*>(p);
}
// Values: whole lines; ONCE: past the caches' reach before they are read again.
template <class T, bool ONCE>
__device__ __forceinline__ T load_value(const char* p) {
  if constexpr (ONCE) return __builtin_nontemporal_load(reinterpret_cast<const T*>(p));
  else return *reinterpret_cast<const T*>(p);
}

// The 16-bit types' products, 32 deep.
__device__ __forceinline__ f32x4 mfma(BF16, u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(bits_as<bf16x8>(a), bits_as<bf16x8>(b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(F16, u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(bits_as<f16x8>(a), bits_as<f16x8>(b), c, 0, 0, 0);
}
__device__ __forceinline__ uint32_t pack2(BF16, float x, float y) {
  const bf16x2 v = {(__bf16)x, (__bf16)y};
  return bits_as<uint32_t>(v);
}
__device__ __forceinline__ uint32_t pack2(F16, float x, float y) {
  const f16x2 v = {(_Float16)x, (_Float16)y};
  return bits_as<uint32_t>(v);
}
__device__ __forceinline__ void unpack2(BF16, uint32_t v, float& x, float& y) {
  x = __uint_as_float(v << 16);
  y = __uint_as_float(v & 0xffff0000u);
}
__device__ __forceinline__ void unpack2(F16, uint32_t v, float& x, float& y) {
  const f16x2 h = bits_as<f16x2>(v);
  x = (float)h[0];
  y = (float)h[1];
}
// A word with those of its two values that are infinite or NaN replaced by 0.
template <class T>
__device__ __forceinline__ uint32_t finite2(T, uint32_t x) {
  constexpr uint32_t kTop = std::is_same_v<T, BF16> ? 0x7f80u : 0x7c00u;
  const uint32_t low = (x & kTop) == kTop ? 0u : x & 0xffffu;
  return (x >> 16 & kTop) == kTop ? low : low | (x & 0xffff0000u);
}
// Two 8-bit values of a word as 16-bit values, exactly.
template <bool HIGH>
__device__ __forceinline__ uint32_t widen2(E4M3, BF16, uint32_t x) {
  return bits_as<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, HIGH));
}
template <bool HIGH>
__device__ __forceinline__ uint32_t widen2(E4M3, F16, uint32_t x) {
  return bits_as<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, HIGH));
}
// Whole numbers: by way of binary32.
template <bool HIGH>
__device__ __forceinline__ uint32_t widen2(I8, BF16, uint32_t x) {
  return pack2(BF16(), (float)(int8_t)(x >> (HIGH ? 16 : 0)), (float)(int8_t)(x >> (HIGH ? 24 : 8)));
}
// 1024 + (c + 128) is 0x6400 with c + 128 in its low byte.
template <bool HIGH>
__device__ __forceinline__ uint32_t widen2(I8, F16, uint32_t x) {
  const uint32_t y = __builtin_amdgcn_perm(0x64646464u, x ^ 0x80808080u, HIGH ? 0x04030402u : 0x04010400u);
  return bits_as<uint32_t>(bits_as<f16x2>(y) - f16x2{(_Float16)1152.0f, (_Float16)1152.0f});
}

// Queries of a 16-bit type over a cache of that type or of 8 bits. DIM: head_dim
// rounded up to one of 32, 64, 96, 128, 192 and 256; FULL: it is head_dim.
// CHUNK: neighbouring values that a lane loads of a key, 16 in an E4M3 row
// of whole 16s, else 8.
template <class Q_, class KV_, int DIM, bool FULL, int CHUNK>
struct Engine16 {
  using Q = Q_;
  using KV = KV_;
  using Args = AttendArgs;
  static constexpr bool kBlocks = false, kWhole = false;
  static constexpr int kElem = sizeof(typename KV::Raw);
  static constexpr int kDim = DIM;
  static constexpr int kGroup = 8, kTile = 32, kProducts = 2;
  static constexpr int kLoads = (DIM + 4 * CHUNK - 1) / (4 * CHUNK);  // of a lane, for a key
  static constexpr int kDeep = CHUNK / 8;                             // products of a load
  // Values of a token in a lane. A divisor of 8, as head_dim is a multiple of
  // 8: no load or store passes the row's end.
  static constexpr int kVec = DIM == 32 ? 2 : DIM == 64 || (DIM == 192 && kElem == 2) ? 4 : 8;
  static constexpr int kPanels = (DIM + 16 * kVec - 1) / (16 * kVec);
  // The numerators' and values' type in the second product. 8-bit values are
  // exact in either; BF16 numerators have no smallest step to lose.
  using W = std::conditional_t<kElem == 1, BF16, Q>;
  // F16 has: numerators are held 2^kLift times as large, up to 2^15, and what
  // their rounding lost kSpread times as large again.
  static constexpr bool kNarrow = std::is_same_v<W, F16>;
  static constexpr float kLift = kNarrow ? 7.0f : 0.0f;
  static constexpr float kSpread = 4096.0f;
  // Infinite values need passes of their own: 0 times them is NaN, and the
  // second part of a numerator is often 0 or negative.
  static constexpr bool kInfinities = kElem == 2;
  static constexpr bool kNaNs = false;
  using KRaw = typename RawOf<CHUNK * kElem>::type;
  using VRaw = typename RawOf<kVec * kElem>::type;

  u32x4 q[kLoads][kDeep];
  KRaw k[kProducts][kLoads];
  VRaw v[kGroup][kPanels];
  f32x4 o[kPanels][kVec];

  // First value of this lane's chunk in load s, and whether the row has it (a
  // lane without reads the row's start and drops it).
  __device__ __forceinline__ static bool chunk(uint32_t s, uint32_t g, uint32_t dim, uint32_t& d) {
    d = (s * 4u + g) * CHUNK;
    if ((FULL && DIM % (4 * CHUNK) == 0) || d < dim) return true;
    d = 0u;
    return false;
  }

  __device__ __forceinline__ void load_q(const typename Q::Raw* row, uint32_t g, uint32_t dim, bool live) {
#pragma unroll
    for (uint32_t s = 0; s < kLoads; ++s) {
      uint32_t d;
      const bool has = chunk(s, g, dim, d) && live;
#pragma unroll
      for (int h = 0; h < kDeep; ++h) {
        u32x4 x = {0u, 0u, 0u, 0u};
        if (has) __builtin_memcpy(&x, row + d + 8 * h, 16);  // rows of any alignment
        q[s][h] = x;
      }
    }
  }

  __device__ __forceinline__ void load_k(int a, const char* row, uint32_t g, uint32_t dim) {
#pragma unroll
    for (uint32_t s = 0; s < kLoads; ++s) {
      uint32_t d;
      chunk(s, g, dim, d);
      k[a][s] = load_key<KRaw, kElem == 1 ? 8 : sizeof(KRaw)>(row + d * kElem);
    }
  }

  template <bool ONCE>
  __device__ __forceinline__ void load_v(int i, const char* row, uint32_t c, uint32_t dim) {
#pragma unroll
    for (uint32_t p = 0; p < kPanels; ++p) {
      const uint32_t d = (p * 16u + c) * kVec;
      v[i][p] = load_value<VRaw, ONCE>(row + (FULL || d < dim ? d : 0u) * kElem);
    }
  }
  __device__ __forceinline__ void keep_v(int i, bool keep) {
#pragma unroll
    for (int p = 0; p < kPanels; ++p) v[i][p] &= VRaw(keep ? ~0u : 0u);
  }

  // Scores of the lane's tokens.
  __device__ __forceinline__ void scores(float* s, uint32_t g, uint32_t dim) const {
#pragma unroll
    for (int a = 0; a < kProducts; ++a) {
      f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (uint32_t t = 0; t < kLoads; ++t) {
        uint32_t d;
        const uint32_t keep = chunk(t, g, dim, d) ? ~0u : 0u;
#pragma unroll
        for (int h = 0; h < kDeep; ++h) {
          u32x4 y;
          if constexpr (kElem == 1) {
            y[0] = widen2<false>(KV(), Q(), k[a][t][2 * h]);
            y[1] = widen2<true>(KV(), Q(), k[a][t][2 * h]);
            y[2] = widen2<false>(KV(), Q(), k[a][t][2 * h + 1]);
            y[3] = widen2<true>(KV(), Q(), k[a][t][2 * h + 1]);
          } else {
            y = k[a][t];
          }
          if constexpr (!FULL) {
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] &= keep;
          }
          x = mfma(Q(), y, q[t][h], x);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) s[4 * a + i] = x[i];
    }
  }

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int p = 0; p < kPanels; ++p)
#pragma unroll
      for (int j = 0; j < kVec; ++j) o[p][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  // Whether a value that was added is no finite number. All rows of its column
  // are none then, whatever their weights (0 times it is NaN): one is looked at.
  __device__ __forceinline__ bool infinite() const {
    float x = 0.0f, y = 0.0f;
#pragma unroll
    for (int p = 0; p < kPanels; ++p)
#pragma unroll
      for (int j = 0; j < kVec; j += 2) {
        x = __builtin_fmaf(o[p][j][0], 0.0f, x);
        y = __builtin_fmaf(o[p][j + 1][0], 0.0f, y);
      }
    return !(x + y == 0.0f);
  }
  // Of token i's values only those that are finite, or only the others.
  __device__ __forceinline__ void keep_finite(int i, bool finite) {
#pragma unroll
    for (int p = 0; p < kPanels; ++p)
#pragma unroll
      for (int w = 0; w < kVec / 2; ++w) {
        if constexpr (kVec == 2) {
          const uint32_t x = finite2(W(), v[i][p]);
          v[i][p] = finite ? x : v[i][p] ^ x;
        } else if constexpr (kElem == 2) {
          const uint32_t x = finite2(W(), v[i][p][w]);
          v[i][p][w] = finite ? x : v[i][p][w] ^ x;
        }
      }
  }

  // Of token i's values, in E4M3, only those that are numbers; or (mark) 1 in the
  // place of each that is none and 0 for all others.
  __device__ __forceinline__ static uint32_t numbers4(uint32_t x, bool mark) {
    const uint32_t top = ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;  // of bytes whose other bits are all set
    const uint32_t none = top | (top - (top >> 7));
    return mark ? none & 0x38383838u : x & ~none;
  }
  __device__ __forceinline__ void keep_numbers(int i, bool mark) {
#pragma unroll
    for (int p = 0; p < kPanels; ++p) {
      if constexpr (kVec <= 4) {
        v[i][p] = (VRaw)numbers4(v[i][p], mark);
      } else {
#pragma unroll
        for (int w = 0; w < kVec / 4; ++w) v[i][p][w] = numbers4(v[i][p][w], mark);
      }
    }
  }
  // What was marked: no number.
  __device__ __forceinline__ void spoil() {
#pragma unroll
    for (int p = 0; p < kPanels; ++p)
#pragma unroll
      for (int j = 0; j < kVec; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[p][j][r] = o[p][j][r] > 0.0f ? NAN : 0.0f;
  }

  // Word w (values 2 w and 2 w + 1) of token i's values in panel p.
  __device__ __forceinline__ uint32_t word(int i, int p, int w) const {
    uint32_t x;
    if constexpr (kVec * kElem <= 4) x = v[i][p];
    else x = v[i][p][kElem == 1 ? w >> 1 : w];
    if constexpr (kElem == 1) return w & 1 ? widen2<true>(KV(), W(), x) : widen2<false>(KV(), W(), x);
    else return x;
  }

  // Value j of token i's in panel p, of whole numbers.
  __device__ __forceinline__ float whole(int i, int p, int j) const {
    uint32_t x;
    if constexpr (kVec <= 4) x = v[i][p];
    else x = v[i][p][j >> 2];
    return (float)(int8_t)(x >> 8 * (j & 3));
  }

  __device__ __forceinline__ static void add_product(u32x4 hi, u32x4 lo, u32x4 v, f32x4& x) {
    if constexpr (kNarrow) {
      const f32x4 y = mfma(W(), lo, v, f32x4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = __builtin_fmaf(y[i], 1.0f / kSpread, x[i]);
    } else {
      x = mfma(W(), lo, v, x);
    }
    x = mfma(W(), hi, v, x);
  }

  // O += P V. A numerator is held as the sum of two 16-bit values, the
  // second what the first one's rounding lost: the matrix cores have the time
  // (24 products for 16 KiB of cache), and at least 16 bits of it are kept, not 8.
  // BF16 loses 2^-17 of a numerator. F16 loses 2^-23 of it or, as its smallest
  // step is 2^-24, 2^-25 in the second value's scale: 2^-44 of the largest
  // numerator, which is at least 2^kLift. So n tokens are off by at most
  // n 2^-44 max |v|; values without a scale, of a sum that has all
  // numerators, were off by n 2^-25 max |v|.
  __device__ __forceinline__ void accumulate(const float* s) {
    u32x4 hi, lo;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      hi[i] = pack2(W(), s[2 * i], s[2 * i + 1]);
      float x, y;
      unpack2(W(), hi[i], x, y);
      x = s[2 * i] - x;
      y = s[2 * i + 1] - y;
      lo[i] = kNarrow ? pack2(W(), x * kSpread, y * kSpread) : pack2(W(), x, y);
    }
#pragma unroll
    for (int p = 0; p < kPanels; ++p) {
#pragma unroll
      for (int w = 0; w < kVec / 2; ++w) {
        u32x4 even, odd;  // values 2 w and 2 w + 1 of the eight tokens
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (std::is_same_v<KV, I8>) {  // (two tokens' values are rounded into one word: nothing to sort after that)
            even[i] = pack2(W(), whole(2 * i, p, 2 * w), whole(2 * i + 1, p, 2 * w));
            odd[i] = pack2(W(), whole(2 * i, p, 2 * w + 1), whole(2 * i + 1, p, 2 * w + 1));
          } else {
            const uint32_t x = word(2 * i, p, w), y = word(2 * i + 1, p, w);
            even[i] = __builtin_amdgcn_perm(y, x, 0x05040100u);
            odd[i] = __builtin_amdgcn_perm(y, x, 0x07060302u);
          }
        }
        add_product(hi, lo, even, o[p][2 * w]);
        add_product(hi, lo, odd, o[p][2 * w + 1]);
      }
    }
  }
};

// The same over a cache with a scale for each block of tokens and head, which
// Run applies. EACH: blocks are no whole groups of tokens.
template <class Q_, class KV_, int DIM, bool FULL, int CHUNK, bool EACH>
struct BlockEngine : Engine16<Q_, KV_, DIM, FULL, CHUNK> {
  using Args = BlockAttendArgs;
  static constexpr bool kBlocks = true;
  static constexpr bool kEach = EACH;
  static constexpr bool kWhole = !EACH;  // (blocks divide pages)
  static constexpr bool kNaNs = std::is_same_v<KV_, E4M3>;
};

// Queries and cache in binary32: the products are 4 deep, one token of each
// group and one value of each chunk at a time.
template <int DIM, bool FULL>
struct Engine32 {
  using Q = F32;
  using KV = F32;
  using Args = AttendArgs;
  static constexpr bool kBlocks = false, kWhole = false;
  static constexpr int kElem = 4;
  static constexpr int kDim = DIM;
  static constexpr int kGroup = 4, kTile = 16, kProducts = 1;
  static constexpr int kSteps = DIM / 16;
  static constexpr float kLift = 0.0f;
  static constexpr bool kInfinities = false, kNaNs = false;
  static constexpr int kVec = DIM % 64 ? 2 : 4, kPanels = DIM / (16 * kVec);
  using VRaw = float __attribute__((ext_vector_type(kVec)));

  f32x4 q[kSteps];
  f32x4 k[kProducts][kSteps];
  VRaw v[kGroup][kPanels];
  f32x4 o[kPanels][kVec];

  __device__ __forceinline__ static bool chunk(uint32_t s, uint32_t g, uint32_t dim, uint32_t& d) {
    d = s * 16u + g * 4u;
    if (FULL || d < dim) return true;
    d = 0u;
    return false;
  }

  __device__ __forceinline__ void load_q(const float* row, uint32_t g, uint32_t dim, bool live) {
#pragma unroll
    for (uint32_t s = 0; s < kSteps; ++s) {
      uint32_t d;
      const bool has = chunk(s, g, dim, d) && live;
      f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
      if (has) __builtin_memcpy(&x, row + d, 16);
      q[s] = x;
    }
  }

  __device__ __forceinline__ void load_k(int a, const char* row, uint32_t g, uint32_t dim) {
#pragma unroll
    for (uint32_t s = 0; s < kSteps; ++s) {
      uint32_t d;
      chunk(s, g, dim, d);
      k[a][s] = load_key<f32x4>(row + d * kElem);
    }
  }

  template <bool ONCE>
  __device__ __forceinline__ void load_v(int i, const char* row, uint32_t c, uint32_t dim) {
#pragma unroll
    for (uint32_t p = 0; p < kPanels; ++p) {
      const uint32_t d = (p * 16u + c) * kVec;
      v[i][p] = load_value<VRaw, ONCE>(row + (FULL || d < dim ? d : 0u) * kElem);
    }
  }
  __device__ __forceinline__ void keep_v(int i, bool keep) {
#pragma unroll
    for (int p = 0; p < kPanels; ++p)
#pragma unroll
      for (int j = 0; j < kVec; ++j) v[i][p][j] = keep ? v[i][p][j] : 0.0f;
  }

  __device__ __forceinline__ void scores(float* s, uint32_t g, uint32_t dim) const {
    // Sums side by side: shorter chains of dependent products, and of
    // roundings (outputs at head size 128 are off by 3.3e-7 of their size, with
    // one sum 7.8e-7). Four; two where the registers are full.
    constexpr int kSums = DIM > 192 ? 2 : 4;
    f32x4 x[kSums];
#pragma unroll
    for (int j = 0; j < kSums; ++j) x[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (uint32_t t = 0; t < kSteps; ++t) {
      uint32_t d;
      const bool has = chunk(t, g, dim, d);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j % kSums] = __builtin_amdgcn_mfma_f32_16x16x4f32(has ? k[0][t][j] : 0.0f, q[t][j], x[j % kSums], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = (x[0][i] + x[1][i]) + (kSums == 4 ? x[kSums - 2][i] + x[kSums - 1][i] : 0.0f);
  }

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int p = 0; p < kPanels; ++p)
#pragma unroll
      for (int j = 0; j < kVec; ++j) o[p][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  __device__ __forceinline__ void accumulate(const float* s) {
#pragma unroll
    for (int i = 0; i < kGroup; ++i)
#pragma unroll
      for (int p = 0; p < kPanels; ++p)
#pragma unroll
        for (int j = 0; j < kVec; ++j)
          o[p][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(s[i], v[i][p][j], o[p][j], 0, 0, 0);
  }
};

}  // namespace llmhip
