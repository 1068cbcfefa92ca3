// Attention on tiles of 32 keys (gfx950, wave64): what the kernels over drafted trees and over pages share.
//
// The query rows that share a key head are the columns of one product, S^T = K Q^T, so
// that a lane of the 16 x 16 result holds four keys of one query: those are the B operand of the
// second product, O^T = V^T P^T, as they stand, when V's rows are read in the same key order.
// Softmax statistics stay in the lanes (max over the four lane groups of a column by two
// exchanges, sums only at the end).
#pragma once

#include <type_traits>

#include "frag.h"

namespace itts {
namespace {

constexpr int kTileKeys = 32;  // keys a wave takes at a time
constexpr int kKeyWaves = 4;   // waves of a block that share a few rows' keys
constexpr int kRowWaves = 4;   // waves of a block with rows of their own over the same keys
constexpr float kLog2e = 1.4426950408889634f;

struct F32 {
  static constexpr int kBytes = 4;
};
struct Bf16 {
  static constexpr int kBytes = 2;
  static constexpr uint32_t kOddBits = 0x7f80u;  // exponent of infinities and NaN
};
struct F16 {
  static constexpr int kBytes = 2;
  static constexpr uint32_t kOddBits = 0x7c00u;
};

// One element at p as a float.
template <class T>
__device__ __forceinline__ float load1(const char *p) {
  if constexpr (T::kBytes == 4) return *reinterpret_cast<const float *>(p);
  else if constexpr (std::is_same_v<T, Bf16>) return bf16_bits_to_float(*reinterpret_cast<const uint16_t *>(p));
  else return half_bits_to_float(*reinterpret_cast<const uint16_t *>(p));
}

// N dwords at p (16-byte aligned where they fill 16 bytes).
template <int N>
__device__ __forceinline__ void load_dwords(const char *p, uint32_t (&o)[N]) {
  if constexpr (N == 2) {
    const u32x2 v = *reinterpret_cast<const u32x2 *>(p);
    o[0] = v[0], o[1] = v[1];
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const u32x4 v = *reinterpret_cast<const u32x4 *>(p + 4 * i);
      o[i] = v[0], o[i + 1] = v[1], o[i + 2] = v[2], o[i + 3] = v[3];
    }
  }
}

// Four values, one rounding to the output's type.
template <class T>
__device__ __forceinline__ void store4(char *p, float a, float b, float c, float d) {
  if constexpr (T::kBytes == 4) {
    *reinterpret_cast<float4 *>(p) = make_float4(a, b, c, d);
  } else if constexpr (std::is_same_v<T, Bf16>) {
    const bf16x2v x = __builtin_convertvector((f32x2e){a, b}, bf16x2v), y = __builtin_convertvector((f32x2e){c, d}, bf16x2v);
    *reinterpret_cast<uint2 *>(p) = make_uint2(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, y));
  } else {
    const f16x2v x = __builtin_convertvector((f32x2e){a, b}, f16x2v), y = __builtin_convertvector((f32x2e){c, d}, f16x2v);
    *reinterpret_cast<uint2 *>(p) = make_uint2(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, y));
  }
}

__device__ __forceinline__ float col_max(float v) {  // over the four lanes of a column
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float col_sum(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

// The pair (a, b) as planes of 16-bit values, the first in the low half: plane 0 holds the leading
// bits (cut, not rounded), the next what is left, so that every plane has its value's sign.  A
// rest of exactly 0 becomes a small number of that sign: 0 times an infinity in the other operand
// would turn what is an infinity into NaN.  A value of 0 stays 0 in every plane: a masked key's finite
// values, however large, must not weigh anything.  bf16: 8 bits a plane, three hold a float.
__device__ __forceinline__ float cut_bits(float v) { return __uint_as_float(__float_as_uint(v) & 0xffff0000u); }
__device__ __forceinline__ uint32_t cut_pair(float a, float b) {
  return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}
__device__ __forceinline__ void cut3(float a, float b, uint32_t (&o)[3]) {
  const float least_a = fminf(fabsf(a), 0x1p-120f), least_b = fminf(fabsf(b), 0x1p-120f);
#pragma unroll
  for (int i = 0; i < 3; i++) {
    o[i] = cut_pair(a, b);
    if (i < 2) {
      a = __builtin_copysignf(fmaxf(fabsf(a - cut_bits(a)), least_a), a);
      b = __builtin_copysignf(fmaxf(fabsf(b - cut_bits(b)), least_b), b);
    }
  }
}
// The same for probabilities (never negative).  bf16: the last rest is raised by 2^-23 of what it is the rest
// of in the subtraction itself; the second of two planes is rounded, 2^-16 of the value at most.  fp16: 11 bits a
// plane, two hold 22, down to its smallest number, 2^-24, which both planes of a positive value are at least: 0 times an
// infinity that is seen would be NaN, however small its weight.  A weight comes out 2^-23 too large at most by that, 2^-33 of
// the largest one as probabilities are held.
typedef unsigned short u16x2e __attribute__((ext_vector_type(2)));
template <class T, int N>
__device__ __forceinline__ void cut_pos(float a, float b, uint32_t (&o)[N]) {
  constexpr float kUp = 1.0f + 0x1p-23f, kLeast = 0x1.01p-118f;  // (more than the 8 bits of one plane)
  if constexpr (std::is_same_v<T, F16>) {
    static_assert(N == 2);
    const auto h = __builtin_amdgcn_cvt_pkrtz(a, b);
    const auto rest = __builtin_amdgcn_cvt_pkrtz(a - (float)h[0], b - (float)h[1]);
    // 1, the bits of 2^-24, where a value is positive: bits of floats as whole numbers, brought down to 16 bits, and no more than 1
    // (a number that the compiler does not know, or it compares the halves one by one).
    uint32_t one = 0x00010001u;
    asm("" : "+s"(one));
    const u16x2e some = __builtin_elementwise_min(
        __builtin_bit_cast(u16x2e, __builtin_amdgcn_cvt_pk_u16(__float_as_uint(a), __float_as_uint(b))), __builtin_bit_cast(u16x2e, one));
    o[0] = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2e, h), some));
    o[1] = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2e, rest), some));
  } else if constexpr (N == 2) {
    o[0] = cut_pair(a, b);
    const f32x2e rest = {__builtin_fmaf(a, kUp, -cut_bits(a)), __builtin_fmaf(b, kUp, -cut_bits(b))};
    o[1] = __builtin_bit_cast(uint32_t, __builtin_convertvector(rest, bf16x2v));
  } else {
    static_assert(N == 3);
    const float rest_a = fmaxf(a - cut_bits(a), fminf(a, kLeast)), rest_b = fmaxf(b - cut_bits(b), fminf(b, kLeast));
    o[0] = cut_pair(a, b), o[1] = cut_pair(rest_a, rest_b);
    o[2] = cut_pair(__builtin_fmaf(rest_a, kUp, -cut_bits(rest_a)), __builtin_fmaf(rest_b, kUp, -cut_bits(rest_b)));
  }
}

template <class T>
__device__ __forceinline__ floatx4 mfma16(const uint32_t *a, const uint32_t *b, floatx4 c) {
  const u32x4 x = {a[0], a[1], a[2], a[3]}, y = {b[0], b[1], b[2], b[3]};
  if constexpr (std::is_same_v<T, Bf16>)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, y), c, 0, 0, 0);
}

// Planes of 16 bits that hold a probability: two under 16-bit queries (16 bits of bf16, 22 of fp16) leave no
// more than the result's own rounding, whichever kernel a launch takes; three under fp32 ones, an fp32's bits.
// (64 bf16 tokens over up to 6,001 rows are 1.7e-3 of their 2-norm off the 64-bit result, as that result rounded to bf16 is; with
// three planes just as much, prompts 557 us -> 739, 4 bits 95 -> 107.)
template <class TQ>
constexpr int kProbPlanes = TQ::kBytes == 4 ? 3 : 2;

// What a wave holds of RT tiles of 16 query rows (lane (c, g): row c of each), and the three steps of
// a tile of keys.  16-bit caches go through the 16-bit matrix instructions: queries in NQ planes (fp32
// ones in three, exactly), probabilities in NP.  fp32 caches take the fp32 ones.
template <int D, class TQ, class TKV, int RT, bool MANY>
struct Rows {
  static constexpr bool kWide = TKV::kBytes == 4;
  static constexpr int NQ = kWide || TQ::kBytes == 2 ? 1 : 3, NP = kProbPlanes<TQ>;
  static constexpr int kV = D / 16 * TKV::kBytes / 4;
  // probabilities are held up to 2^(kLag + kUp): the running maximum moves only when a score passes
  // it by 2^kLag; fp16 planes use their range below 1 too
  static constexpr float kLag = 5.0f, kUp = std::is_same_v<TKV, F16> ? 10.0f : 0.0f;
  uint32_t q[NQ][RT][D / 32][kWide ? 8 : 4];  // elements 32 j + 8 g ..
  float scale;  // what a score is still multiplied by, for powers of two
  floatx4 o[RT][D / 16];
  float m[RT];
  // the probabilities' sums: over this lane's keys, or (MANY) over all keys, by products with ones
  typename std::conditional<MANY, floatx4, float>::type l[RT];

  // at[t]: element 8 g of tile t's row c
  __device__ __forceinline__ void load(const char *const (&at)[RT], float score_scale) {
    uint32_t raw[RT][D / 32][8 * TQ::kBytes / 4];
#pragma unroll
    for (int t = 0; t < RT; t++) {
#pragma unroll
      for (int j = 0; j < D / 32; j++) load_dwords<8 * TQ::kBytes / 4>(at[t] + 32 * j * TQ::kBytes, raw[t][j]);
      m[t] = -INFINITY, l[t] = {};
#pragma unroll
      for (int d = 0; d < D / 16; d++) o[t][d] = floatx4{};
    }
    const float by = score_scale * kLog2e;
    const uint32_t flip = score_scale < 0.0f ? 0x80008000u : 0;
    scale = kWide || NQ == 3 ? 1.0f : fmaxf(fabsf(by), 0x1p-120f);  // (0 times the mask's -inf would be NaN)
#pragma unroll
    for (int t = 0; t < RT; t++)
#pragma unroll
      for (int j = 0; j < D / 32; j++) {
        if constexpr (kWide) {  // fp32 queries carry the scale
#pragma unroll
          for (int e = 0; e < 8; e++) q[0][t][j][e] = __float_as_uint(__uint_as_float(raw[t][j][e]) * by);
        } else if constexpr (NQ == 3) {
#pragma unroll
          for (int e = 0; e < 4; e++) {
            uint32_t w[3];
            cut3(__uint_as_float(raw[t][j][2 * e]) * by, __uint_as_float(raw[t][j][2 * e + 1]) * by, w);
#pragma unroll
            for (int i = 0; i < 3; i++) q[i][t][j][e] = w[i];
          }
        } else {  // 16-bit ones its sign
#pragma unroll
          for (int e = 0; e < 4; e++) q[0][t][j][e] = raw[t][j][e] ^ flip;
        }
      }
  }

  // s[h][t]: keys 16 h + 4 g + r of tile t's row c; k[h]: the keys' elements 32 j + 8 g ..
  template <int N>
  __device__ __forceinline__ void scores(floatx4 (&s)[2][RT], int j, const uint32_t (&k0)[N], const uint32_t (&k1)[N]) const {
    if constexpr (kWide) {
#pragma unroll
      for (int e = 0; e < 8; e++)
#pragma unroll
        for (int t = 0; t < RT; t++) {
          s[0][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k0[e]), __uint_as_float(q[0][t][j][e]), s[0][t], 0, 0, 0);
          s[1][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k1[e]), __uint_as_float(q[0][t][j][e]), s[1][t], 0, 0, 0);
        }
    } else {
#pragma unroll
      for (int i = NQ - 1; i >= 0; i--)
#pragma unroll
        for (int t = 0; t < RT; t++) {
          s[0][t] = mfma16<TKV>(k0, q[i][t][j], s[0][t]);
          s[1][t] = mfma16<TKV>(k1, q[i][t][j], s[1][t]);
        }
    }
  }

  // The running maxima for a tile's scores, and what was summed rescaled where one moves.  At an edge bit
  // 16 h + r of seen[t] says whether key 16 h + 4 g + r counts.
  __device__ __forceinline__ void limit(floatx4 (&s)[2][RT], bool edge, const uint32_t (&seen)[RT]) {
    if (edge) {
#pragma unroll
      for (int t = 0; t < RT; t++)
#pragma unroll
        for (int i = 0; i < 8; i++)
          s[i >> 2][t][i & 3] = seen[t] & 1u << (16 * (i >> 2) + (i & 3)) ? s[i >> 2][t][i & 3] : -INFINITY;
    }
    float top[RT];
    bool grows = false;
#pragma unroll
    for (int t = 0; t < RT; t++) {
      top[t] = s[0][t][0];
#pragma unroll
      for (int i = 1; i < 7; i += 2) top[t] = fmaxf(fmaxf(s[i >> 2][t][i & 3], s[(i + 1) >> 2][t][(i + 1) & 3]), top[t]);
      top[t] = fmaxf(s[1][t][3], top[t]) * scale;
      grows = grows || top[t] > m[t] + kLag;
    }
    if (__ballot(grows)) {
#pragma unroll
      for (int t = 0; t < RT; t++) {
        const float mn = fmaxf(m[t], col_max(top[t]));
        const float f = __builtin_amdgcn_exp2f(m[t] - (mn == -INFINITY ? 0.0f : mn));
        m[t] = mn;
        l[t] *= f;
#pragma unroll
        for (int d = 0; d < D / 16; d++) o[t][d] *= f;
      }
    }
  }

  // Scores to probabilities, and their sums.
  __device__ __forceinline__ void weigh(floatx4 (&s)[2][RT]) {
#pragma unroll
    for (int t = 0; t < RT; t++) {
      const float ms = (m[t] == -INFINITY ? 0.0f : m[t]) - kUp;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i >> 2][t][i & 3], scale, -ms));
        s[i >> 2][t][i & 3] = p;
        if constexpr (!MANY) l[t] += p;
      }
    }
  }

  // Probabilities as the second product's operand: 16-bit planes of a lane's 8 keys.  At an edge masked keys
  // are 0 in all of them.
  struct Probs {
    uint32_t p[kWide ? 1 : RT][NP][4];
  };
  __device__ __forceinline__ void pack(const floatx4 (&s)[2][RT], Probs &x) const {
    if constexpr (!kWide) {
#pragma unroll
      for (int t = 0; t < RT; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float a = s[i >> 1][t][2 * (i & 1)], b = s[i >> 1][t][2 * (i & 1) + 1];
          uint32_t w[NP];
          cut_pos<TKV, NP>(a, b, w);
#pragma unroll
          for (int k = 0; k < NP; k++) x.p[t][k][i] = w[k];
        }
    }
  }

  __device__ __forceinline__ void add_sums(const Probs &x) {
    constexpr uint32_t kOne = std::is_same_v<TKV, Bf16> ? 0x3f803f80u : 0x3c003c00u;
    const uint32_t ones[4] = {kOne, kOne, kOne, kOne};
#pragma unroll
    for (int t = 0; t < RT; t++)
#pragma unroll
      for (int k = NP - 1; k >= 0; k--) l[t] = mfma16<TKV>(ones, x.p[t][k], l[t]);
  }
  // o[.][d0 ..] += P V; vt[d]: the operand of V^T whose row c is element (d0 + d, c) of keys 4 g + r, then
  // of keys 16 + 4 g + r.
  template <int N>
  __device__ __forceinline__ void add(const Probs &x, int d0, const uint32_t (&vt)[N][4]) {
#pragma unroll
    for (int t = 0; t < RT; t++)
#pragma unroll
      for (int k = NP - 1; k >= 0; k--)
#pragma unroll
        for (int d = 0; d < N; d++) o[t][d0 + d] = mfma16<TKV>(vt[d], x.p[t][k], o[t][d0 + d]);
  }
  // The same from rows: v[i], elements D / 16 c .. of key 16 (i / 4) + 4 g + i % 4, in pairs of rows.
  __device__ __forceinline__ void add_rows(const Probs &x, const uint32_t (&v)[8][kV]) {
    uint32_t vt[D / 16][4];
#pragma unroll
    for (int d = 0; d < D / 16; d++)
#pragma unroll
      for (int i = 0; i < 4; i++)
        vt[d][i] = __builtin_amdgcn_perm(v[2 * i + 1][d / 2], v[2 * i][d / 2], d % 2 ? 0x07060302u : 0x05040100u);
    add(x, 0, vt);
  }
  __device__ __forceinline__ void add_wide(const floatx4 (&s)[2][RT], const uint32_t (&v)[8][kV]) {
#pragma unroll
    for (int i = 0; i < 8; i++)
#pragma unroll
      for (int t = 0; t < RT; t++)
#pragma unroll
        for (int d = 0; d < D / 16; d++)
          o[t][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v[i][d]), s[i >> 2][t][i & 3], o[t][d], 0, 0, 0);
  }
};

// Rows of nodes count only where they are seen, and rows past the last one nowhere: 0 times what a
// masked row may hold (infinities, NaN) must stay out of a tile's product, so such values leave it
// and are added at the end, row by row (odd_values).  Returns whether there were any.
template <class T, int N>
__device__ __forceinline__ uint32_t take_odd(uint32_t (&v)[8][N], int key0, int len, int total, int g) {
  uint32_t odd = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const int key = key0 + 16 * (i >> 2) + 4 * g + (i & 3);
    const uint32_t own = key < len ? ~0u : 0, in = key < total ? ~0u : 0;
#pragma unroll
    for (int d = 0; d < N; d++) {
      const uint32_t w = v[i][d];
      uint32_t keep;
      if constexpr (T::kBytes == 4) {
        keep = (w & 0x7f800000u) == 0x7f800000u ? 0 : ~0u;
      } else {
        keep = (w & T::kOddBits) == T::kOddBits ? 0xffff0000u : ~0u;
        keep = (w & T::kOddBits << 16) == T::kOddBits << 16 ? keep & 0xffffu : keep;
      }
      keep |= own;
      odd |= ~keep & in;
      v[i][d] = w & keep & in;
    }
  }
  return odd;
}
// The same where keys 4 g + 2 i, 4 g + 2 i + 1 (i < 2; then 16 more) share dword i.
template <class T, int N>
__device__ __forceinline__ uint32_t take_odd_columns(uint32_t (&v)[N][4], int key0, int len, int total, int g) {
  uint32_t odd = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int key = key0 + 16 * (i >> 1) + 4 * g + 2 * (i & 1);
    const uint32_t own = (key < len ? 0xffffu : 0) | (key + 1 < len ? 0xffff0000u : 0);
    const uint32_t in = (key < total ? 0xffffu : 0) | (key + 1 < total ? 0xffff0000u : 0);
#pragma unroll
    for (int d = 0; d < N; d++) {
      const uint32_t w = v[d][i];
      uint32_t keep = (w & T::kOddBits) == T::kOddBits ? 0xffff0000u : ~0u;
      keep = (w & T::kOddBits << 16) == T::kOddBits << 16 ? keep & 0xffffu : keep;
      keep |= own;
      odd |= ~keep & in;
      v[d][i] = w & keep & in;
    }
  }
  return odd;
}
// A 16-byte piece's half through LDS's transposing load (gfx950), over groups of 16 lanes.
__device__ __forceinline__ u32x2 load_transposed(u32x4 *piece, int half) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  using Lds = __attribute__((address_space(3))) s16x4;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds *)(reinterpret_cast<s16x4 *>(piece) + half)));
}

}  // namespace
}  // namespace itts
