// Rows of keys and values into pages and out of them.
//
// Append.  Token i of sequence b has row r = lengths[b] + i.  With (a, b) a pair of its key's (or query's) elements and t the
// pair's angle at the row's position,
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t),
// the cosines and sines from a table.  A cache of 4 bits takes every 64 elements x as
//   base = min x, scale = (max x - min x) / 15 (to fp32 and to fp16), code = rint((x - base) / scale) in 0 .. 15 (scale 0: 0),
// the quantiser of the decoder's weights.  Rotation and quantiser work in 64 bits, which run at the rate of 32 here:
// codes are those of the definition, also where a value lies next to the border of two.
// 6,582 tokens, 32 heads and 8 key heads of 128, all turned, us a call: into bf16 30.5 (162 MB, 5.3 TB/s: memory), into 4 bits 43.4
// (142 MB): half of it are its waves' 64-bit instructions (two exchanges through LDS a step and canonical operands more: 45).
//
// Gather.  A copy: 147 MB of bf16 rows 21.4 us (6.9 TB/s: caches hold some of them); 4 bits to fp32 values, 186 MB, 25 us (one piece a
// thread: 31).
#include <algorithm>
#include <type_traits>

#include "attn_tiles.h"
#include "pages.h"

namespace itts {
namespace {

struct I4 {};

// Eight elements of 16 bits or 32 at p.
template <class T>
__device__ __forceinline__ void load8(const char *p, float (&x)[8]) {
  uint32_t w[2 * T::kBytes];
  load_dwords<2 * T::kBytes>(p, w);
#pragma unroll
  for (int e = 0; e < 8; e++) {
    if constexpr (T::kBytes == 4) x[e] = __uint_as_float(w[e]);
    else if constexpr (std::is_same_v<T, Bf16>) x[e] = __uint_as_float(e % 2 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
    else x[e] = half_bits_to_float(e % 2 ? w[e / 2] >> 16 : w[e / 2] & 0xffffu);
  }
}
template <class T, class X>
__device__ __forceinline__ void store8(char *p, const X (&x)[8]) {
  store4<T>(p, (float)x[0], (float)x[1], (float)x[2], (float)x[3]);
  store4<T>(p + 4 * T::kBytes, (float)x[4], (float)x[5], (float)x[6], (float)x[7]);
}

// (in one instruction: fmin and fmax have both operands made canonical first)
__device__ __forceinline__ double lesser(double a, double b) {
  double r;
  asm("v_min_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
__device__ __forceinline__ double greater(double a, double b) {
  double r;
  asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
// The other lane's value, a step of 1, 2 or 4 lanes away in a group of 8 (4: mirrored, which does where all lanes of four agree).
template <int STEP>
__device__ __forceinline__ double near_lane(double v) {
  constexpr int kMove = STEP == 1 ? 0xb1 : STEP == 2 ? 0x4e : 0x141;  // quad_perm [1 0 3 2], [2 3 0 1], row_half_mirror
  asm("s_nop 1" : "+v"(v));  // (what the instructions above wrote is read by other lanes two wait states later at the earliest)
  const uint64_t w = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (uint32_t)w, kMove, 0xf, 0xf, true);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (uint32_t)(w >> 32), kMove, 0xf, 0xf, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// A row's lanes (D / 16 of them, 16 elements each in two runs of 8 with numbers run[0], run[1]) to codes and pairs.
template <int D>
__device__ __forceinline__ void store_codes(char *codes, char *pairs, const int (&run)[2], int j, const double (&x)[2][8]) {
  constexpr int kLanes = D / 16, kGroups = D / 64;
  double least[2], most[2];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    double odd = 0.0;  // (of each run by itself: the two may lie in different groups)
    least[i] = most[i] = x[i][0];
#pragma unroll
    for (int e = 0; e < 8; e++) {
      least[i] = lesser(least[i], x[i][e]), most[i] = greater(most[i], x[i][e]);
      odd = __builtin_fma(x[i][e], 0.0, odd);  // NaN for a value that is no finite number
    }
    // (which then makes the range infinite)
    if (odd != 0.0) least[i] = 0.0, most[i] = INFINITY;
  }
  double lo[kGroups], hi[kGroups];
#pragma unroll
  for (int G = 0; G < kGroups; G++) {
    const bool in0 = kGroups == 1 || run[0] >> 3 == G, in1 = kGroups == 1 || run[1] >> 3 == G;
    lo[G] = in0 ? least[0] : INFINITY, hi[G] = in0 ? most[0] : -INFINITY;
    lo[G] = lesser(lo[G], in1 ? least[1] : INFINITY), hi[G] = greater(hi[G], in1 ? most[1] : -INFINITY);
    lo[G] = lesser(lo[G], near_lane<1>(lo[G])), hi[G] = greater(hi[G], near_lane<1>(hi[G]));
    lo[G] = lesser(lo[G], near_lane<2>(lo[G])), hi[G] = greater(hi[G], near_lane<2>(hi[G]));
    if constexpr (kLanes == 8) lo[G] = lesser(lo[G], near_lane<4>(lo[G])), hi[G] = greater(hi[G], near_lane<4>(hi[G]));
  }
  double scale[kGroups], base[kGroups], inverse[kGroups];
#pragma unroll
  for (int G = 0; G < kGroups; G++) {
    // (to 32 bits and from there to 16, as the definition has it: left alone, the compiler makes one rounding of the two)
    float s32 = (float)((hi[G] - lo[G]) / 15.0), b32 = (float)lo[G];
    asm volatile("" : "+v"(s32), "+v"(b32));
    const _Float16 s = (_Float16)s32, b = (_Float16)b32;
    const bool ok = fabsf((float)s) < INFINITY && fabsf((float)b) < INFINITY;
    scale[G] = ok && s != (_Float16)0 ? (double)(float)s : INFINITY, base[G] = ok ? (double)(float)b : 0.0;
    inverse[G] = 1.0 / scale[G];  // (0 where there is no scale, or none that holds: codes of 0)
    const uint32_t pair = (uint32_t)__builtin_bit_cast(uint16_t, s) | (uint32_t)__builtin_bit_cast(uint16_t, b) << 16;
    if (j == 0) *reinterpret_cast<uint32_t *>(pairs + 4 * G) = ok ? pair : 0x7e007e00u;
  }
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const double s = kGroups == 1 || run[i] >> 3 == 0 ? scale[0] : scale[kGroups - 1];
    const double b = kGroups == 1 || run[i] >> 3 == 0 ? base[0] : base[kGroups - 1];
    const double inv = kGroups == 1 || run[i] >> 3 == 0 ? inverse[0] : inverse[kGroups - 1];
    auto code = [](double y) { return (uint32_t)(int)__builtin_amdgcn_fmed3f((float)__builtin_rint(y), 0.0f, 15.0f); };
    uint32_t w = 0;
    bool near = false;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const double y = (x[i][e] - b) * inv;
      near = near || fabs(y - __builtin_rint(y)) > 0.5 - 1e-12;
      w |= code(y) << (4 * e);
    }
    if (near) {  // the product is off by 2^-51 of at most 16: next to a border the quotient itself decides
      w = 0;
#pragma unroll
      for (int e = 0; e < 8; e++) w |= code((x[i][e] - b) / s) << (4 * e);
    }
    *reinterpret_cast<uint32_t *>(codes + 4 * run[i]) = w;
  }
}

// A wave takes pieces of one token, 64 lanes' at a time: D / 16 lanes a row, query heads first, then those of keys and values.
// A lane's 16 elements are two runs of 8 that rotate with each other (halves of the rotated part, or neighbours in pairs), the
// same ones of every row, so that a wave reads the angles once.  The last waves take a sequence each, for its new length.
template <int D, class TX, class TKV>
__global__ __launch_bounds__(256) void append_kernel(PagedAppend a, int pieces, int parts, uint64_t mul) {
  constexpr int kLanes = D / 16;
  const int lane = threadIdx.x & 63;
  const int64_t job = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
  const int64_t jobs = (int64_t)a.tokens * parts;
  const int max_rows = (int)min((int64_t)a.n_table * a.pages.size, (int64_t)kPagesMaxRows);
  if (job >= jobs) {
    const int b = (int)(job - jobs);
    if (b >= a.batch) return;
    const int start = a.starts[b], end = a.starts[b + 1], len = a.lengths[b], n = end - start;
    bool ok = start >= 0 && end >= start && end <= a.tokens && len >= 0 && len <= max_rows - n;
    if (ok && n > 0) {
      ok = owner_of(a.starts, a.batch, a.tokens, start).b == b;
      const int last = page_of(len + n - 1, mul);
      for (int p = page_of(len, mul) + lane; p <= last; p += 64) ok = ok && (uint32_t)a.table[b * a.tab_b + p] < (uint32_t)a.pages.n;
    }
    const bool all = __ballot(!ok) == 0;
    if (lane == 0) a.new_lengths[b] = all ? len + n : -1;
    return;
  }
  const int token = (int)(job / parts), part = (int)(job - (int64_t)token * parts), Hk = a.pages.Hk;
  const int turned = a.rot >> 4;  // lanes of a row that rotate
  const int j = lane % kLanes;
  int run[2];
  if (a.interleaved || j >= turned) run[0] = 2 * j, run[1] = 2 * j + 1;
  else run[0] = j, run[1] = j + turned;

  // A piece's rows: what they are (0 query, 1 key, 2 value, 3 none) and which head.
  auto head_of = [&](int piece, int &own) {
    const int head = (piece * 64 + lane) / kLanes;
    const int kind = head < a.H ? 0 : head < a.H + Hk ? 1 : head < a.H + 2 * Hk ? 2 : 3;
    own = kind == 0 ? head : kind == 1 ? head - a.H : head - a.H - Hk;
    return kind;
  };
  auto load = [&](int piece, float (&raw)[2][8]) {
    int own;
    const int kind = piece < pieces ? head_of(piece, own) : 3;
    if (kind == 3) return;
    const char *from = kind == 0 ? static_cast<const char *>(a.q) + (token * a.q_t + own * a.q_h) * TX::kBytes
                     : kind == 1 ? static_cast<const char *>(a.k) + (token * a.k_t + own * a.k_h) * TX::kBytes
                                 : static_cast<const char *>(a.v) + (token * a.v_t + own * a.v_h) * TX::kBytes;
#pragma unroll
    for (int i = 0; i < 2; i++) load8<TX>(from + 8 * run[i] * TX::kBytes, raw[i]);
  };
  float raw[2][8] = {};
  load(part, raw);  // (on its way before anything is known of the sequence)

  const Owner of = owner_of(a.starts, a.batch, a.tokens, token);
  int row = -1, page = -1, pos = -1;  // row: -2 for a token of a sequence that is refused
  if (of.b >= 0) {
    const int len = uniform_load(a.lengths + of.b);
    row = len >= 0 && len <= max_rows - of.n ? len + token - of.first : -2;
    if (row >= 0) {
      page = uniform_load(a.table + of.b * a.tab_b + page_of(row, mul));
      pos = a.positions ? uniform_load(a.positions + token) : row;
    }
  }
  const bool place = row >= 0 && (uint32_t)page < (uint32_t)a.pages.n, known = (uint32_t)pos < (uint32_t)a.n_positions;
  const int64_t at = place ? row - page_of(row, mul) * a.pages.size : 0;
  float c[8], s[8];
  const bool turns = a.rotation && j < turned;
  if (turns) {
    const float *table = a.rotation + (int64_t)(known ? pos : 0) * a.rot_r;
    load8<F32>(reinterpret_cast<const char *>(table + 8 * j), c);
    load8<F32>(reinterpret_cast<const char *>(table + a.rot / 2 + 8 * j), s);
  }
  for (int piece = part; piece < pieces; piece += parts) {
    int own;
    const int kind = head_of(piece, own);
    double x[2][8];
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int e = 0; e < 8; e++) x[i][e] = raw[i][e];
    load(piece + parts, raw);
    if (kind == 3 || (kind != 0 && !place)) continue;
    if (a.rotation && kind != 2) {
      if (!known) {
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
          for (int e = 0; e < 8; e++) x[i][e] = NAN;
      } else if (turns) {
        if (!a.interleaved) {
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const double u = x[0][e], w = x[1][e];
            x[0][e] = u * c[e] - w * s[e], x[1][e] = w * c[e] + u * s[e];
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const double u = x[e / 4][2 * (e % 4)], w = x[e / 4][2 * (e % 4) + 1];
            x[e / 4][2 * (e % 4)] = u * c[e] - w * s[e], x[e / 4][2 * (e % 4) + 1] = w * c[e] + u * s[e];
          }
        }
      }
    }
    if (kind == 0) {
      char *to = static_cast<char *>(a.q_out) + (token * a.o_t + own * a.o_h) * TX::kBytes;
#pragma unroll
      for (int i = 0; i < 2; i++) {
        if (row < 0) {  // no sequence's token, or one of a refused sequence
#pragma unroll
          for (int e = 0; e < 8; e++) x[i][e] = row == -1 ? 0.0 : NAN;
        }
        store8<TX>(to + 8 * run[i] * TX::kBytes, x[i]);
      }
    } else {
      char *to = kind == 1 ? a.pages.k + page * a.pages.k_p + own * a.pages.k_h + at * a.pages.k_r
                           : a.pages.v + page * a.pages.v_p + own * a.pages.v_h + at * a.pages.v_r;
      if constexpr (std::is_same_v<TKV, I4>) {
        char *pairs = kind == 1 ? a.pages.kp + page * a.pages.kp_p + own * a.pages.kp_h + at * a.pages.kp_r
                                : a.pages.vp + page * a.pages.vp_p + own * a.pages.vp_h + at * a.pages.vp_r;
        store_codes<D>(to, pairs, run, j, x);
      } else {
#pragma unroll
        for (int i = 0; i < 2; i++) store8<TKV>(to + 8 * run[i] * TKV::kBytes, x[i]);
      }
    }
  }
}

// A thread takes kAtOnce pieces of 16 bytes of an output's rows; blocks of a sequence, key head and cache.
constexpr int kAtOnce = 4;
template <int D, class TKV, class TO>
__global__ __launch_bounds__(256) void gather_kernel(PagedGather a, uint64_t mul) {
  constexpr int kPer = 16 / TO::kBytes, kPieces = D / kPer;
  const int b = blockIdx.y, is_v = blockIdx.z & 1, head = blockIdx.z >> 1;
  const int i0 = blockIdx.x * 256 * kAtOnce + threadIdx.x;
  const int len = uniform_load(a.lengths + b);
  const bool bad = len < 0 || len > (int)min((int64_t)a.n_table * a.pages.size, (int64_t)kPagesMaxRows);
  const int rows = bad ? 0 : min(len, a.rows);
  const char *pages = is_v ? a.pages.v + head * a.pages.v_h : a.pages.k + head * a.pages.k_h;
  const int64_t page_step = is_v ? a.pages.v_p : a.pages.k_p, row_step = is_v ? a.pages.v_r : a.pages.k_r;
  const char *all_pairs = is_v ? a.pages.vp + head * a.pages.vp_h : a.pages.kp + head * a.pages.kp_h;
  const int64_t pair_page = is_v ? a.pages.vp_p : a.pages.kp_p, pair_row = is_v ? a.pages.vp_r : a.pages.kp_r;
  int page[kAtOnce], at[kAtOnce];
#pragma unroll
  for (int u = 0; u < kAtOnce; u++) {
    const int row = (i0 + 256 * u) / kPieces, p = row < rows ? page_of(row, mul) : 0;
    page[u] = row < rows ? a.table[b * a.tab_b + p] : -1;
    at[u] = row - p * a.pages.size;
  }
  constexpr bool kCodes = std::is_same_v<TKV, I4>;
  uint32_t w[kAtOnce][kCodes ? 2 : 4];
#pragma unroll
  for (int u = 0; u < kAtOnce; u++) {
    const int run = (i0 + 256 * u) % kPieces;
    if ((uint32_t)page[u] >= (uint32_t)a.pages.n) continue;
    const char *from = pages + page[u] * page_step + at[u] * row_step;
    if constexpr (kCodes) {
      if constexpr (kPer == 8) w[u][0] = *reinterpret_cast<const uint32_t *>(from + 4 * run);
      else w[u][0] = *reinterpret_cast<const uint16_t *>(from + 2 * run);
      w[u][1] = *reinterpret_cast<const uint32_t *>(all_pairs + page[u] * pair_page + at[u] * pair_row + 4 * (run * kPer >> 6));
    } else {
      load_dwords<4>(from + 16 * run, w[u]);
    }
  }
  char *to = static_cast<char *>(is_v ? a.v : a.k) + (is_v ? b * a.v_b + head * a.v_h : b * a.k_b + head * a.k_h) * TO::kBytes;
  const int64_t to_row = is_v ? a.v_r : a.k_r;
#pragma unroll
  for (int u = 0; u < kAtOnce; u++) {
    const int row = (i0 + 256 * u) / kPieces, run = (i0 + 256 * u) % kPieces;
    if (row >= a.rows) return;
    const bool there = (uint32_t)page[u] < (uint32_t)a.pages.n;
    const float rest = bad || row < rows ? NAN : 0.0f;  // of rows that are not there
    char *p = to + (row * to_row + kPer * run) * TO::kBytes;
    if constexpr (kCodes) {
      const float s = half_bits_to_float(w[u][1] & 0xffffu), base = half_bits_to_float(w[u][1] >> 16);
      float x[kPer];
#pragma unroll
      for (int e = 0; e < kPer; e++) x[e] = there ? __builtin_fmaf((float)(w[u][0] >> (4 * e) & 15u), s, base) : rest;
      if constexpr (kPer == 8) store8<TO>(p, x);
      else store4<TO>(p, x[0], x[1], x[2], x[3]);
    } else {
      const uint32_t fill = rest == 0.0f ? 0u : TO::kBytes == 4 ? 0x7fc00000u : std::is_same_v<TO, Bf16> ? 0x7fc07fc0u : 0x7e007e00u;
      *reinterpret_cast<u32x4 *>(p) = there ? u32x4{w[u][0], w[u][1], w[u][2], w[u][3]} : u32x4{fill, fill, fill, fill};
    }
  }
}

template <int D, class TX, class TKV>
hipError_t launch_append(const PagedAppend &a, int n_cu, hipStream_t s) {
  const int pieces = ((a.H + 2 * a.pages.Hk) * (D / 16) + 63) / 64;
  // a piece a wave, until those fill the card
  const int64_t waves = 32ll * n_cu;
  const int parts = (int)std::clamp<int64_t>(waves / std::max(1, a.tokens), 1, pieces);
  const int64_t jobs = (int64_t)a.tokens * parts + a.batch;
  hipLaunchKernelGGL((append_kernel<D, TX, TKV>), dim3((unsigned)((jobs + 3) / 4)), dim3(256), 0, s, a, pieces, parts, page_mul(a.pages.size));
  return hipGetLastError();
}
template <class TX, class TKV>
hipError_t launch_append(const PagedAppend &a, int n_cu, hipStream_t s) {
  return a.pages.D == 64 ? launch_append<64, TX, TKV>(a, n_cu, s) : launch_append<128, TX, TKV>(a, n_cu, s);
}
template <class TKV, class TO>
hipError_t launch_gather(const PagedGather &a, hipStream_t s) {
  const int D = a.pages.D;
  const int pieces = D * TO::kBytes / 16;
  const dim3 grid((unsigned)(((int64_t)a.rows * pieces + 256 * kAtOnce - 1) / (256 * kAtOnce)), a.batch, 2 * a.pages.Hk);
  if (D == 64) hipLaunchKernelGGL((gather_kernel<64, TKV, TO>), grid, dim3(256), 0, s, a, page_mul(a.pages.size));
  else hipLaunchKernelGGL((gather_kernel<128, TKV, TO>), grid, dim3(256), 0, s, a, page_mul(a.pages.size));
  return hipGetLastError();
}

}  // namespace

hipError_t paged_append(const PagedAppend &a, int n_cu, hipStream_t s) {
  if (a.batch <= 0) return hipSuccess;
  const int kv = a.pages.type;
  if (a.type == kOpF32) {
    if (kv == kOpF32) return launch_append<F32, F32>(a, n_cu, s);
    if (kv == kOpBf16) return launch_append<F32, Bf16>(a, n_cu, s);
    if (kv == kOpI4) return launch_append<F32, I4>(a, n_cu, s);
  } else if (a.type == kOpBf16) {
    if (kv == kOpBf16) return launch_append<Bf16, Bf16>(a, n_cu, s);
    if (kv == kOpI4) return launch_append<Bf16, I4>(a, n_cu, s);
  } else if (a.type == kOpF16) {
    if (kv == kOpF16) return launch_append<F16, F16>(a, n_cu, s);
    if (kv == kOpI4) return launch_append<F16, I4>(a, n_cu, s);
  }
  return hipErrorInvalidValue;
}

hipError_t paged_gather(const PagedGather &a, hipStream_t s) {
  if (a.batch <= 0 || a.rows <= 0) return hipSuccess;
  const int kv = a.pages.type;
  if (kv == kOpF32 && a.type == kOpF32) return launch_gather<F32, F32>(a, s);
  if (kv == kOpBf16 && a.type == kOpBf16) return launch_gather<Bf16, Bf16>(a, s);
  if (kv == kOpF16 && a.type == kOpF16) return launch_gather<F16, F16>(a, s);
  if (kv == kOpI4 && a.type == kOpF32) return launch_gather<I4, F32>(a, s);
  if (kv == kOpI4 && a.type == kOpBf16) return launch_gather<I4, Bf16>(a, s);
  if (kv == kOpI4 && a.type == kOpF16) return launch_gather<I4, F16>(a, s);
  return hipErrorInvalidValue;
}

}  // namespace itts
