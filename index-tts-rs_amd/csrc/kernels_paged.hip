// Attention over paged caches: the tokens of ragged sequences (single ones, pieces of prompts) over their sequences' rows.
//
// The n tokens of sequence b are its last ones: token i has position P = lengths[b] - n + i and sees the rows t <= P, with a
// window W the rows t > P - W and t < S (the first ones, which stay in sight) alone:
//   o_i = sum_t p_it v_t / sum_t p_it,   p_it = exp(scale q_i . k_t - m_i).
// The rows (token, head of the group) that share a key head are the columns of the products (attn_tiles.h); row r is head
// r % group of token r / group.  Keys go by in tiles of 32; pages are multiples of 16 rows, so that each half of a tile lies in
// one page, whose number comes through the scalar cache a tile ahead of its rows.
#include <algorithm>
#include <cmath>
#include <numeric>
#include <type_traits>

#include "attn_tiles.h"
#include "pages.h"

namespace itts {
namespace {

// A cache of 4 bits.
struct I4 {};

// A launch: blocks of kTileRows rows of a sequence and key head, each with all keys that they see (parts 0) or with a share
// of them and results of its own (o [Hk][parts][rows][D], then (max, sum) [Hk][parts][rows], then (first block, blocks of a
// row tile) [batch]) that a second kernel joins.
struct Args {
  PagedAttn a;
  int blocks, parts, group;
  uint32_t group_mul;  // 2^32 / group, rounded up: one too many at most
  uint64_t page_mul;
  bool even;           // pages of multiples of 32 rows
  int per_token;       // without shares: blocks that stand for a token (0: tokens together, and one more a sequence)
  int unit, least;     // a share is at least `least` times 2^unit tiles of keys
  float2 *ml;
  int2 *dealt;
  __device__ int token(int row) const {
    if (group == 1) return row;
    const int i = __umulhi((uint32_t)row, group_mul);
    return i * group > row ? i - 1 : i;
  }
};

// The tiles of KT keys that the tokens at positions p0 .. p1 of a sequence see, counted through: those with rows < S,
// then from the window's first one on.
template <int KT>
struct Tiles {
  int front, skip, n;
  __device__ __forceinline__ Tiles(const PagedAttn &a, int p0, int p1) {
    const int from = a.window > 0 ? max(0, p0 - a.window + 1) / KT : 0;
    front = min(a.sinks / KT + (a.sinks % KT != 0), from);
    skip = from - front;
    n = p1 < 0 ? 0 : front + p1 / KT + 1 - from;
  }
  __device__ __forceinline__ int key(int u) const { return (u < front ? u : u + skip) * KT; }
};

// What block `index` has to do: tiles [first, end) of row tile `tile` of sequence b, whose rows are shared by n blocks (0:
// nothing is left for this one).  A sequence's last tokens, which see most, come first.
struct Share {
  int b, tile, n, first, end;
};
// Blocks with all keys of a row tile: those of a sequence stand from a number on that its first token alone tells, with room
// for as many as it can have, so that a wave finds its own in a search by 64 starts.  (By all sequences' row tiles, a lane a
// sequence, 64 at a time: 2,048 tokens over 200 .. 499 rows 778 us for 518, 16,384 over 64 rows 11,540 for 730.)
//
// Where a block stands for several tokens: the sequence of block `place`, or (TOKEN) of token `place`, its first block and blocks
// (b = -1: none).  A sequence has its blocks if it has its tokens (owner_of) and all blocks lead to it too.
template <int ROWS, bool TOKEN>
__device__ __forceinline__ Owner blocks_of(const Args &p, int place) {
  const PagedAttn &a = p.a;
  const int lane = threadIdx.x & 63;
  auto keys = [&](int start, int b) { return make_int2(start, min(max(start, 0), a.tokens) * p.group / ROWS + b); };
  const Way w = way_to<!TOKEN>(a.batch, place, [&](int b) { return keys(a.starts[b], b); });
  const bool in = lane < w.n;
  const int start = in ? a.starts[w.b0 + lane] : 0, end = in ? a.starts[w.b0 + lane + 1] : 0, block = keys(start, w.b0 + lane).y;
  const bool has = start >= 0 && end > start && end <= a.tokens;
  const int n = has ? ((end - start) * p.group + ROWS - 1) / ROWS : 0;
  // (the first one: blocks of a sequence that starts behind all earlier ones' ends stand behind theirs)
  const uint64_t holds = __ballot(TOKEN ? has && start <= place && place < end : block <= place && place < block + n);
  if (holds == 0) return Owner{-1, 0, 0};
  const int i = __builtin_ctzll(holds), first = __builtin_amdgcn_readlane(start, i), stop = __builtin_amdgcn_readlane(end, i);
  const Owner of{w.b0 + i, __builtin_amdgcn_readlane(block, i), __builtin_amdgcn_readlane(n, i)};
  if (__ballot(has && lane < i && end > first) != 0 || !w.leads_x(first, stop - 1) || !w.leads_y(of.first, of.first + of.n - 1)) return Owner{-1, 0, 0};
  return of;
}
template <int ROWS>
__device__ __forceinline__ Share whole_of(const Args &p, int index) {
  const PagedAttn &a = p.a;
  Owner of;  // (its blocks)
  if (p.per_token > 0) {
    of = owner_of(a.starts, a.batch, a.tokens, p.per_token == 1 ? index : index / p.per_token);
    of.first *= p.per_token, of.n = (of.n * p.group + ROWS - 1) / ROWS;
  } else {
    of = blocks_of<ROWS, false>(p, index);
  }
  const int local = index - of.first;
  if (of.b < 0 || local >= of.n) return Share{0, 0, 0, 0, 0};
  return Share{of.b, of.n - 1 - local, 1, 0, 1 << 30};
}

// The number of tokens of sequence b0 + lane: as owner_of has it, but of all sequences, 64 after the other.  reach: the furthest
// end of those before.
__device__ __forceinline__ int tokens_of(const PagedAttn &a, int b0, int &reach) {
  const int lane = threadIdx.x & 63;
  const bool in = b0 + lane < a.batch;
  const int start = in ? a.starts[b0 + lane] : 0, end = in ? a.starts[b0 + lane + 1] : 0;
  const bool rises = start >= 0 && end >= start && end <= a.tokens, has = rises && end > start;
  int before = reach;  // the furthest end in front of the lane's sequence
  if (__ballot(!rises) == 0) {  // (each starts where the one in front of it ends)
    reach = max(reach, __builtin_amdgcn_readlane(end, min(a.batch - b0, 64) - 1));
  } else {
    int to = has ? end : 0;
#pragma unroll
    for (int step = 1; step < 64; step *= 2) {
      const int up = __shfl_up(to, step, 64);
      if (lane >= step) to = max(to, up);
    }
    const int up = __shfl_up(to, 1, 64);
    before = lane > 0 ? max(reach, up) : reach;
    reach = max(reach, __builtin_amdgcn_readlane(to, 63));
  }
  return has && start >= before ? end - start : 0;
}

// Blocks that share the keys: every share has the same size, the smallest one with which `blocks` are enough.  Found by
// every wave from the starts and lengths, a lane a sequence.
template <int ROWS, int KT>
__device__ __forceinline__ Share share_of(const Args &p, int index, int hk) {
  if (p.parts == 0) return whole_of<ROWS>(p, index);
  const PagedAttn &a = p.a;
  const int lane = threadIdx.x & 63;
  // (the first block of all says for every sequence where its shares are)
  const bool tells = index == 0 && hk == 0;
  // row tiles of a sequence, and the units of keys that one of them sees at most
  // (those of the first 64 once for all turns)
  int reach = 0;
  const int tokens0 = tokens_of(a, 0, reach), reach0 = reach, len0 = a.lengths[min(lane, a.batch - 1)];
  auto count = [&](int b0, int &tiles, int &units) {
    if (b0 == 0) reach = reach0;
    const int rows = (b0 == 0 ? tokens0 : tokens_of(a, b0, reach)) * p.group, len = b0 == 0 ? len0 : a.lengths[min(b0 + lane, a.batch - 1)];
    tiles = (rows + ROWS - 1) / ROWS;
    int seen = len < 0 || len > a.max_rows ? 1 : max(len, 1);
    if (a.window > 0) seen = (int)min((int64_t)seen, (int64_t)a.window + min(a.sinks, a.max_rows) + (ROWS - 1) / p.group + 1 + 2 * KT);
    units = tiles == 0 ? 0 : ((seen + KT - 1) / KT + (1 << p.unit) - 1) >> p.unit;
  };
  float total = 0.0f, longest = 0.0f;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    int tiles, units;
    count(b0, tiles, units);
    total += (float)tiles * units, longest = fmaxf(longest, units);
  }
  total = wave_sum(total), longest = wave_max(longest);
  // (64 blocks of a row tile at most: the joining kernel's lanes)
  int size = (int)fmaxf(ceilf(fmaxf(total / p.parts, longest / 64)), (float)p.least);
  for (int i = 0; i < 16; i++) {
    float blocks = 0.0f;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
      int tiles, units;
      count(b0, tiles, units);
      blocks += (float)tiles * ((units + size - 1) / size);
    }
    blocks = wave_sum(blocks);
    if (blocks <= p.parts) break;
    // (at last a share for each row tile; blocks are enough for those)
    size = i < 14 ? max(size + 1, (int)ceilf(size * (blocks / p.parts))) : (int)longest + 1;
  }
  size = __builtin_amdgcn_readfirstlane(size);
  Share share{0, 0, 0, 0, 0};
  int before = 0;
  for (int b0 = 0; b0 < a.batch && (share.n == 0 || tells); b0 += 64) {
    int tiles, units;
    count(b0, tiles, units);
    const int each = (int)(((int64_t)units + size - 1) / size), own = tiles * each;
    int to = own;  // (counted to one more than there are blocks)
#pragma unroll
    for (int step = 1; step < 64; step *= 2) {
      const int up = __shfl_up(to, step, 64);
      if (lane >= step) to = min(to + up, p.blocks + 1);
    }
    if (tells && b0 + lane < a.batch) p.dealt[b0 + lane] = before + to <= p.parts ? make_int2(before + to - own, each) : make_int2(0, 0);
    if (const uint64_t at = __ballot(index < before + to); at != 0 && share.n == 0) {
      const int src = __builtin_ctzll(at), from = before + (src > 0 ? __builtin_amdgcn_readlane(to, src - 1) : 0);
      share.b = b0 + src, share.n = __builtin_amdgcn_readlane(each, src);
      const int local = index - from, tile = local / share.n;
      share.tile = __builtin_amdgcn_readlane(tiles, src) - 1 - tile;
      const int part = local - tile * share.n;
      share.first = share.n == 1 ? 0 : part * size << p.unit;
      share.end = share.n == 1 ? 1 << 30 : share.first + (size << p.unit);
    }
    before = min(before + __builtin_amdgcn_readlane(to, 63), p.blocks + 1);
  }
  if (a.batch > 64 && share.n > 0 && owner_of(a.starts, a.batch, a.tokens, uniform_load(a.starts + share.b)).b != share.b) share.n = 0;
  return share;
}

// What a block knows of its rows.
struct Seq {
  int first_token, n, len, rows;  // tokens of the sequence, its length (0 for a bad one), its rows n * group
  int p0, p1;                     // positions of the block's first and last token
  bool bad;
};
template <int ROWS>
__device__ __forceinline__ Seq seq_of(const Args &p, const Share &share) {
  const PagedAttn &a = p.a;
  const Span span = span_of(uniform_load(a.starts + share.b), uniform_load(a.starts + share.b + 1), a.tokens);
  const int len = uniform_load(a.lengths + share.b);
  Seq s;
  s.bad = len < 0 || len > a.max_rows;
  s.first_token = span.first, s.n = span.n, s.len = s.bad ? 0 : len, s.rows = span.n * p.group;
  const int before = s.len - s.n;
  s.p0 = before + p.token(share.tile * ROWS), s.p1 = s.bad ? -1 : before + p.token(min(s.rows, (share.tile + 1) * ROWS) - 1);
  return s;
}

// Rows of a tile that the token at position pos sees, as bits.
__device__ __forceinline__ uint32_t below(int n) { return n <= 0 ? 0 : n >= 32 ? ~0u : (1u << n) - 1; }
__device__ __forceinline__ uint32_t seen_bits(const PagedAttn &a, int pos, int key0) {
  uint32_t seen = below(pos + 1 - key0);
  if (a.window > 0) seen &= ~below(pos + 1 - a.window - key0) | below(a.sinks - key0);
  return seen;
}
// Whether the tokens at p0 .. p1 all see the whole tile.
template <int KT>
__device__ __forceinline__ bool all_see(const PagedAttn &a, int p0, int p1, int key0) {
  return key0 + KT <= p0 + 1 && (a.window == 0 || key0 > p1 - a.window || key0 + KT <= a.sinks);
}

// The pages of a tile's halves.  Rows from `end` on are not looked up: nothing sees them, the other half's page stands in.
struct Ids {
  int page[2], at[2];  // at: the half's first row in its page
  // halves whose page does not exist: no memory is read for them (page 0 stands in)
  __device__ __forceinline__ int missing(const PagedAttn &a) const {
    return ((uint32_t)page[0] >= (uint32_t)a.pages.n ? 1 : 0) | ((uint32_t)page[1] >= (uint32_t)a.pages.n ? 2 : 0);
  }
};
__device__ __forceinline__ Ids ids_of(const Args &p, const int32_t *table, int key0, int end) {
  Ids ids;
  if (p.even) {  // (pages of whole tiles)
    const int page = page_of(key0, p.page_mul);
    ids.page[0] = ids.page[1] = uniform_load(table + page);
    ids.at[0] = key0 - page * p.a.pages.size, ids.at[1] = ids.at[0] + 16;
    return ids;
  }
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const int key = h == 1 && key0 + 16 >= end ? key0 : key0 + 16 * h, page = page_of(key, p.page_mul);
    ids.page[h] = uniform_load(table + page);
    ids.at[h] = key - page * p.a.pages.size;
  }
  return ids;
}
__device__ __forceinline__ void bases_of(const Args &p, const Ids &ids, const char *pages, int64_t page_step, int64_t row_step,
                                         const char *(&base)[2]) {
  // (pages are less than 2^32 bytes apart, rows less than 2^31)
  auto at = [&](int h) {
    const uint32_t page = (uint32_t)ids.page[h] < (uint32_t)p.a.pages.n ? ids.page[h] : 0;
    return pages + (uint64_t)page * (uint32_t)page_step + (uint64_t)(uint32_t)ids.at[h] * (uint32_t)row_step;
  };
  base[0] = at(0);
  if (p.even) base[1] = base[0] + 16 * (uint32_t)row_step;
  else base[1] = at(1);
}

// A wave's keys and values of one tile: key rows 16 h + c, in runs of 8 elements 32 j + 8 g, and value rows 16 h + 4 g + r,
// elements D / 16 c ...
template <int D, class T>
struct PageRegs {
  static constexpr int kK = 8 * T::kBytes / 4, kV = D / 16 * T::kBytes / 4;  // dwords of a run
  uint32_t k[2][D / 32][kK];
  uint32_t v[8][kV];
  uint32_t k_at, v_at[4];
  __device__ __forceinline__ void place(const Pages &g, int c, int q) {
    k_at = c * (uint32_t)g.k_r + 8 * q * T::kBytes;
#pragma unroll
    for (int r = 0; r < 4; r++) v_at[r] = (4 * q + r) * (uint32_t)g.v_r + D / 16 * c * T::kBytes;
  }
  __device__ __forceinline__ void load_k(const Args &p, const Ids &ids, int hk) {
    const char *base[2];
    bases_of(p, ids, p.a.pages.k + hk * p.a.pages.k_h, p.a.pages.k_p, p.a.pages.k_r, base);
#pragma unroll
    for (int h = 0; h < 2; h++) {
      asm volatile("" : "+v"(k_at));  // (kept as 32 bits)
#pragma unroll
      for (int j = 0; j < D / 32; j++) load_dwords<kK>(base[h] + 32 * j * T::kBytes + k_at, k[h][j]);
    }
  }
  __device__ __forceinline__ void load_v(const Args &p, const Ids &ids, int hk) {
    const char *base[2];
    bases_of(p, ids, p.a.pages.v + hk * p.a.pages.v_h, p.a.pages.v_p, p.a.pages.v_r, base);
#pragma unroll
    for (int i = 0; i < 8; i++) {
      asm volatile("" : "+v"(v_at[i & 3]));
      load_dwords<kV>(base[i >> 2] + v_at[i & 3], v[i]);
    }
  }
};

// Of a tile of 4 bits: codes 64 G + 16 g .. + 15 of each key row 16 h + c, codes 64 G + 4 c .. + 3 of each value row
// 16 h + 4 g + r, and the pairs of rows 16 h + 4 g + r of both.
template <int D>
struct CodeRegs {
  static constexpr int G = D / 64;
  uint32_t k[2][G][2], v[8][G], kp[8][G], vp[8][G];
};

// Of a dword with four codes in each half, codes d as 16-bit pairs 1 + code / 16: one shift and one mask, the bits above are
// the exponent of 1.  Sums of such products minus the sum of the other operand are 1/16 of those of the codes.
// TURNED: those of the upper half, all bits turned round, are (code - 31) / 16.
template <class T, bool TURNED>
struct CodeBits {
  static constexpr int kAt = std::is_same_v<T, Bf16> ? 3 : 6;  // the highest bits of a fraction of 7 or 10
  // (in registers of their own: one instruction takes both)
  uint32_t mask = 0x000f000fu << kAt;
  uint32_t one = (std::is_same_v<T, Bf16> ? 0x3f803f80u : 0x3c003c00u) | (TURNED ? (0x80000000u | 0x000f0000u << kAt) : 0u);
  __device__ __forceinline__ CodeBits() { asm volatile("" : "+s"(mask), "+v"(one)); }
  __device__ __forceinline__ void pairs(uint32_t w, uint32_t (&o)[4]) const {
#pragma unroll
    for (int d = 0; d < 4; d++) o[d] = ((4 * d < kAt ? w << (kAt - 4 * d) : w >> (4 * d - kAt)) & mask) ^ one;
  }
};
__device__ __forceinline__ float low_half(uint32_t w) { return (float)__builtin_bit_cast(f16x2v, w)[0]; }
__device__ __forceinline__ float high_half(uint32_t w) { return (float)__builtin_bit_cast(f16x2v, w)[1]; }

// Rows (attn_tiles.h) over 4 bits.  With key t's codes c, scale s and base b in each group of 64 elements,
//   q . k_t = sum_groups s sum_e q_e c_e + b sum_e q_e,
// so the products run on codes, exact in 16 bits, and the pairs come in by two multiply-adds a score and group.  In the second
// product the scale goes with the probability, and sum_t p_t b_t is one number a row and group: in bf16, whose
// range holds a probability times any scale.  (Two planes of it, 2^-16, also under fp16 queries, whose results are rounded by 2^-11:
// 2.055e-4 of their 2-norm off the 64-bit result, which rounded to fp16 is 2.052e-4 off.)
// Every second key's codes are turned round there: 16 + c of one and c - 31 of the other leave nothing of their 16 where keys
// weigh alike, and sums over long contexts do not grow.  (With 16 + c alone 60,000 keys of one weight came out 8e-4 of their mean off,
// four roundings to fp16; so it is 3e-8.)
template <int D, class TQ, int RT>
struct Rows4 {
  using TK = std::conditional_t<std::is_same_v<TQ, F16>, F16, Bf16>;  // of the scores' products
  static constexpr int G = D / 64, NQ = TQ::kBytes == 4 ? 3 : 1, NP = kProbPlanes<TQ>;
  static constexpr float kLag = 5.0f;
  uint32_t q[NQ][RT][G][2][4];  // elements 64 G + 16 g + 8 j + (i, i + 4)
  float qs[RT][G], qs16[RT][G]; // sums of a group's elements, and 1/16 of them
  float scale;
  floatx4 o[RT][D / 16];        // element 64 G + 4 (4 g + r) + d in register r of 4 G + d: sums with 1 + code / 16, (code - 31) / 16
  float ob[RT][G];              // sums of p (base - 16 scale), p (base + 31 scale), over this lane's keys
  float m[RT], l[RT];
  CodeBits<TK, false> key_bits;
  CodeBits<Bf16, true> value_bits;

  // at[t]: the first element of tile t's row c
  __device__ __forceinline__ void load(const char *const (&at)[RT], float score_scale, int g) {
    const float by = score_scale * kLog2e;
    // (fp32 queries carry the scale, rounded once as their caller's own product would; 16-bit ones stay exact)
    const float in = NQ == 3 ? by : score_scale < 0.0f ? -1.0f : 1.0f;
    scale = NQ == 3 ? 16.0f : fmaxf(16.0f * fabsf(by), 0x1p-120f);  // (0 times a mask's -inf would be NaN)
#pragma unroll
    for (int t = 0; t < RT; t++) {
#pragma unroll
      for (int i = 0; i < G; i++) {
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 2; j++) {
          uint32_t raw[2 * TQ::kBytes];
          load_dwords<2 * TQ::kBytes>(at[t] + (64 * i + 16 * g + 8 * j) * TQ::kBytes, raw);
          float x[8];
#pragma unroll
          for (int e = 0; e < 8; e++) {
            if constexpr (TQ::kBytes == 4) x[e] = __uint_as_float(raw[e]);
            else if constexpr (std::is_same_v<TQ, Bf16>) x[e] = __uint_as_float(e % 2 ? raw[e / 2] & 0xffff0000u : raw[e / 2] << 16);
            else x[e] = e % 2 ? high_half(raw[e / 2]) : low_half(raw[e / 2]);
            x[e] *= in;
            sum += x[e];
          }
#pragma unroll
          for (int e = 0; e < 4; e++) {
            float a = x[e], b = x[e + 4];
#pragma unroll
            for (int k = 0; k < NQ; k++) {
              if constexpr (std::is_same_v<TQ, F16>) q[k][t][i][j][e] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
              else q[k][t][i][j][e] = cut_pair(a, b);
              a -= cut_bits(a), b -= cut_bits(b);
            }
          }
        }
        qs[t][i] = col_sum(sum), qs16[t][i] = qs[t][i] * 0.0625f;
        ob[t][i] = 0.0f;
      }
      m[t] = -INFINITY, l[t] = 0.0f;
#pragma unroll
      for (int d = 0; d < D / 16; d++) o[t][d] = floatx4{};
    }
  }

  __device__ __forceinline__ void scores(floatx4 (&s)[2][RT], const CodeRegs<D> &x) const {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      floatx4 acc[G][RT];
#pragma unroll
      for (int i = 0; i < G; i++) {
#pragma unroll
        for (int t = 0; t < RT; t++) acc[i][t] = floatx4{-qs[t][i], -qs[t][i], -qs[t][i], -qs[t][i]};
#pragma unroll
        for (int j = 0; j < 2; j++) {
          uint32_t codes[4];
          key_bits.pairs(x.k[h][i][j], codes);
#pragma unroll
          for (int k = NQ - 1; k >= 0; k--)
#pragma unroll
            for (int t = 0; t < RT; t++) acc[i][t] = mfma16<TK>(codes, q[k][t][i][j], acc[i][t]);
        }
      }
#pragma unroll
      for (int t = 0; t < RT; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          float v = 0.0f;
#pragma unroll
          for (int i = 0; i < G; i++) {
            const uint32_t pair = x.kp[4 * h + r][i];
            v = __builtin_fmaf(high_half(pair), qs16[t][i], v);
            v = __builtin_fmaf(low_half(pair), acc[i][t][r], v);
          }
          s[h][t][r] = v;
        }
    }
  }
  // Running maxima; at an edge keys that are not seen count as -inf.
  __device__ __forceinline__ void limit(floatx4 (&s)[2][RT], bool edge, const uint32_t (&seen)[RT]) {
    float top[RT];
    bool grows = false;
#pragma unroll
    for (int t = 0; t < RT; t++) {
      if (edge) {
#pragma unroll
        for (int i = 0; i < 8; i++) s[i >> 2][t][i & 3] = seen[t] & 1u << (16 * (i >> 2) + (i & 3)) ? s[i >> 2][t][i & 3] : -INFINITY;
      }
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
        for (int i = 0; i < G; i++) ob[t][i] *= f;
#pragma unroll
        for (int d = 0; d < D / 16; d++) o[t][d] *= f;
      }
    }
  }
  __device__ __forceinline__ void weigh(floatx4 (&s)[2][RT]) {
#pragma unroll
    for (int t = 0; t < RT; t++) {
      const float ms = m[t] == -INFINITY ? 0.0f : m[t];
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i >> 2][t][i & 3], scale, -ms));
        s[i >> 2][t][i & 3] = p;
        l[t] += p;
      }
    }
  }
  template <bool EDGE>
  __device__ __forceinline__ void add(const floatx4 (&s)[2][RT], const uint32_t (&seen)[RT], const CodeRegs<D> &x) {
#pragma unroll
    for (int i = 0; i < G; i++) {
      uint32_t planes[RT][NP][4];
#pragma unroll
      for (int n = 0; n < 4; n++) {
        const float s0 = low_half(x.vp[2 * n][i]), s1 = low_half(x.vp[2 * n + 1][i]);
        const float b0 = __builtin_fmaf(s0, -16.0f, high_half(x.vp[2 * n][i])), b1 = __builtin_fmaf(s1, 31.0f, high_half(x.vp[2 * n + 1][i]));
#pragma unroll
        for (int t = 0; t < RT; t++) {
          const float p0 = s[n >> 1][t][2 * (n & 1)], p1 = s[n >> 1][t][2 * (n & 1) + 1];
          float a0 = __builtin_fmaf(p0, s0, 0.0f), a1 = __builtin_fmaf(p1, s1, 0.0f);  // (takes fp16 as it is)
          if constexpr (EDGE) {  // (0 times what a row that is not seen may hold: NaN)
            const uint32_t at = seen[t] >> (16 * (n >> 1) + 2 * (n & 1));
            a0 = at & 1 ? a0 : 0.0f, a1 = at & 2 ? a1 : 0.0f;
            ob[t][i] += (at & 1 ? p0 * b0 : 0.0f) + (at & 2 ? p1 * b1 : 0.0f);
          } else {
            ob[t][i] = __builtin_fmaf(p0, b0, __builtin_fmaf(p1, b1, ob[t][i]));
          }
          uint32_t w[NP];
          cut_pos<Bf16, NP>(a0, a1, w);
#pragma unroll
          for (int k = 0; k < NP; k++) planes[t][k][n] = w[k];
        }
      }
      uint32_t codes[4][4];  // [element][pair of keys]
#pragma unroll
      for (int n = 0; n < 4; n++) {
        uint32_t w[4];
        value_bits.pairs(x.v[2 * n][i] | x.v[2 * n + 1][i] << 16, w);
#pragma unroll
        for (int d = 0; d < 4; d++) codes[d][n] = w[d];
      }
#pragma unroll
      for (int t = 0; t < RT; t++)
#pragma unroll
        for (int k = NP - 1; k >= 0; k--)
#pragma unroll
          for (int d = 0; d < 4; d++) o[t][4 * i + d] = mfma16<Bf16>(codes[d], planes[t][k], o[t][4 * i + d]);
    }
  }
};

// Rows of tokens that belong to no sequence are zeros.  Blocks that share keys leave them to the joining kernel; others write them
// where they are done: of up to 64 sequences whose starts rise the tokens in front of the first one and behind the last; else
// each token is looked at, a wave a token.
template <int D, class TQ, int ROWS>
__device__ __forceinline__ void clear_rest(const Args &p) {
  const PagedAttn &a = p.a;
  if (p.parts > 0) return;
  const int per = a.H * (D / 4);
  auto clear = [&](int token, int at) {
    const int d = at % (D / 4) * 4, head = at / (D / 4);
    store4<TQ>(static_cast<char *>(a.out) + (token * a.o_t + head * a.o_h + d) * TQ::kBytes, 0.0f, 0.0f, 0.0f, 0.0f);
  };
  const int lane = threadIdx.x & 63, b = min(lane, a.batch - 1);
  if (a.batch <= 64) {
    const int start = a.starts[b], end = a.starts[b + 1];
    if (__ballot(start < 0 || end < start || end > a.tokens) == 0) {
      const int front = __builtin_amdgcn_readlane(start, 0), back = __builtin_amdgcn_readlane(end, 63);
      const int64_t n = (int64_t)(front + a.tokens - back) * per;
      for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
        const int k = (int)(i / per);
        clear(k < front ? k : back + k - front, (int)(i - (int64_t)k * per));
      }
      return;
    }
  }
  const int waves = gridDim.x * 4;
  for (int token = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6)); token < a.tokens; token += waves) {
    const Owner of = p.per_token > 0 ? owner_of(a.starts, a.batch, a.tokens, token) : blocks_of<ROWS, true>(p, token);
    if (of.b >= 0) continue;
    for (int at = lane; at < per; at += 64) clear(token, at);
  }
}

// Four elements d .. of row `row` of the block's row tile, to the output or the shares' results.  What the joining kernel
// cannot tell by itself goes with the statistics: a row that sees nothing has maximum +inf and sum 0, one of a bad sequence
// sum NaN.
template <int D, class TQ, int ROWS>
__device__ __forceinline__ void put4(const Args &p, const Share &share, const Seq &seq, int index, int hk, int row, int d, float *y,
                                     float top, float sum, bool any, bool keys) {
  const PagedAttn &a = p.a;
  if (share.n == 1) {
    const float inv = 1.0f / sum;
#pragma unroll
    for (int e = 0; e < 4; e++) y[e] = seq.bad ? NAN : any ? y[e] * inv : 0.0f;
    const int r = share.tile * ROWS + row, i = p.token(r), head = hk * p.group + r - i * p.group;
    store4<TQ>(static_cast<char *>(a.out) + ((seq.first_token + i) * a.o_t + head * a.o_h + d) * TQ::kBytes, y[0], y[1], y[2], y[3]);
  } else {
    const size_t at = ((size_t)hk * p.parts + index) * ROWS + row;
    if (keys) *reinterpret_cast<float4 *>(a.part + at * D + d) = make_float4(y[0], y[1], y[2], y[3]);
    if (d == 0) p.ml[at] = seq.bad ? make_float2(0.0f, NAN) : any ? make_float2(top, sum) : make_float2(INFINITY, 0.0f);
  }
}

// y[0 .. 4) += the values in tiles that not all rows see which are no finite numbers, of the keys that this row sees.
template <int D, class T, int KT>
__device__ inline void odd_values(float *y, const Args &p, const Seq &seq, const Tiles<KT> &tiles, int first, int end, const int32_t *table,
                                  int hk, int pos, int d) {
  const PagedAttn &a = p.a;
#pragma unroll 1
  for (int u = first; u < end; u++) {
    const int key_u = tiles.key(u);
    if (all_see<KT>(a, seq.p0, seq.p1, key_u)) continue;
#pragma unroll 1
    for (int key0 = key_u; key0 < min(key_u + KT, seq.p1 + 1); key0 += kTileKeys) {
      const Ids ids = ids_of(p, table, key0, seq.p1 + 1);
      const int missing = ids.missing(a);
      const char *base[2];
      bases_of(p, ids, a.pages.v + hk * a.pages.v_h, a.pages.v_p, a.pages.v_r, base);
      const uint32_t seen = seen_bits(a, pos, key0);
#pragma unroll 1
      for (int i = 0; i < kTileKeys; i++) {
        if (!(seen >> i & 1) || (missing >> (i >> 4) & 1)) continue;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float v = load1<T>(base[i >> 4] + (i & 15) * a.pages.v_r + (d + e) * T::kBytes);
          if (!(fabsf(v) < INFINITY)) y[e] += v;
        }
      }
    }
  }
}

// The results of a block's waves over keys of their own, joined and put away; more(y, position, d) adds to a row's elements.
template <int D, class TQ, int ROWS, int WK, class F>
__device__ __forceinline__ void join_waves(const Args &p, const Share &share, const Seq &seq, int index, int hk, bool keys,
                                           const float (&so)[WK][ROWS][D + 4], const float (&sm)[WK][ROWS], const float (&sl)[WK][ROWS], F more) {
  for (int i = threadIdx.x; i < ROWS * (D / 4); i += 64 * WK) {
    const int rr = i / (D / 4), d = i % (D / 4) * 4, r = share.tile * ROWS + rr;
    if (r >= seq.rows) continue;
    const int own = seq.len - seq.n + p.token(r);
    float top = -INFINITY, sum = 0.0f, y[4] = {};
#pragma unroll
    for (int w = 0; w < WK; w++) top = fmaxf(top, sm[w][rr]);
    const float ms = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int w = 0; w < WK; w++) {
      const float f = __builtin_amdgcn_exp2f(sm[w][rr] - ms);
      const float4 v = *reinterpret_cast<const float4 *>(&so[w][rr][d]);
      sum += f * sl[w][rr];
      y[0] += f * v.x, y[1] += f * v.y, y[2] += f * v.z, y[3] += f * v.w;
    }
    more(y, own, d);
    put4<D, TQ, ROWS>(p, share, seq, index, hk, rr, d, y, top, sum, own >= 0, keys);
  }
}

// Few query rows (many over fp32 caches): 4 waves over tiles of keys of their own, straight from memory into registers, one tile
// ahead; joined at the end.  Decode steps are bound by memory: 64 tokens, 8 key heads of 128, 501 .. 6,001 bf16 rows in pages of 16,
// 853 MB, 164 us (5.2 TB/s); 24 sequences of up to 3 tokens, 16 heads of 64, a window of 4,000 fp16 rows, 394 MB, 75 us.  Short
// ones by the chain from load to result: one token, 20 heads, 235 rows 7.6 us.  Many rows over fp32 caches by the fp32 matrix
// instructions: 4 x 547 tokens, a window of 256 rows and 232 first ones 70 us, 39 of them those instructions' time at full rate;
// keys and values cut into three bf16 planes in LDS for 128 rows at a time (six products of bf16 for one) took as long: the cutting and
// the chain of one tile's steps cost what the matrix units saved.  Two row tiles a wave there: 124 -> 121 us for 4 x 547 tokens over
// 1,200 rows.
template <int D, class TQ, class TKV, int RT>
__global__ __launch_bounds__(256, (D == 128 && TKV::kBytes == 4 ? 1 : 2)) void paged_attn_kernel(Args p) {
  constexpr int WK = 4, kRows = 16 * RT;
  __shared__ float so[WK][kRows][D + 4];
  __shared__ float sm[WK][kRows], sl[WK][kRows];
  __shared__ int sodd[WK];
  const PagedAttn &a = p.a;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
  const int hk = blockIdx.x % a.pages.Hk, index = blockIdx.x / a.pages.Hk;
  const Share share = share_of<kRows, kTileKeys>(p, index, hk);
  if (share.n == 0) return clear_rest<D, TQ, kRows>(p);
  const Seq seq = seq_of<kRows>(p, share);
  const Tiles<kTileKeys> tiles(a, seq.p0, seq.p1);
  const int first = min(share.first, tiles.n), end = min(share.end, tiles.n);
  const int32_t *table = a.table + share.b * a.tab_b;

  const char *at[RT];
  int pos[RT];
#pragma unroll
  for (int t = 0; t < RT; t++) {
    const int r = min(share.tile * kRows + 16 * t + c, seq.rows - 1), i = p.token(r), head = hk * p.group + r - i * p.group;
    pos[t] = seq.len - seq.n + i;
    at[t] = static_cast<const char *>(a.q) + ((seq.first_token + i) * a.q_t + head * a.q_h + 8 * g) * TQ::kBytes;
  }
  Rows<D, TQ, TKV, RT, false> rows;
  PageRegs<D, TKV> x;
  x.place(a.pages, c, g);
  uint32_t odd = 0;  // a value that is no finite number was taken out
  int u = first + wave;
  Ids ids, next;
  if (u < end) {
    ids = ids_of(p, table, tiles.key(u), seq.p1 + 1);
    next = ids_of(p, table, tiles.key(min(u + WK, end - 1)), seq.p1 + 1);
    x.load_k(p, ids, hk);
    x.load_v(p, ids, hk);
  }
  rows.load(at, a.scale);

  for (; u < end; u += WK) {
    const int key0 = tiles.key(u), missing = ids.missing(a);
    floatx4 s[2][RT] = {};
#pragma unroll
    for (int j = 0; j < D / 32; j++) rows.scores(s, j, x.k[0][j], x.k[1][j]);
    // the wave's next tile (past the last one: that one again)
    ids = next;
    x.load_k(p, ids, hk);
    next = ids_of(p, table, tiles.key(min(u + 2 * WK, end - 1)), seq.p1 + 1);
    const bool edge = !all_see<kTileKeys>(a, seq.p0, seq.p1, key0) || missing != 0;
    uint32_t seen[RT] = {};
    if (edge) {
#pragma unroll
      for (int t = 0; t < RT; t++) seen[t] = seen_bits(a, pos[t], key0) >> (4 * g);
      if (missing) {  // scores of rows that are seen but not there
#pragma unroll
        for (int t = 0; t < RT; t++)
#pragma unroll
          for (int i = 0; i < 8; i++)
            if (missing >> (i >> 2) & 1) s[i >> 2][t][i & 3] = NAN;
      }
    }
    rows.limit(s, edge, seen);
    rows.weigh(s);
    if (edge) odd |= take_odd<TKV>(x.v, key0, 0, seq.p1 + 1, g);
    if constexpr (TKV::kBytes == 4) {
      rows.add_wide(s, x.v);
    } else {
      typename decltype(rows)::Probs probs;
      rows.pack(s, probs);
      rows.add_rows(probs, x.v);
    }
    x.load_v(p, ids, hk);
  }

  // The waves joined.
  const bool any = __ballot(odd != 0) != 0;
  if (lane == 0) sodd[wave] = any;
#pragma unroll
  for (int t = 0; t < RT; t++) {
    const float l = col_sum(rows.l[t]);
    if (g == 0) sm[wave][16 * t + c] = rows.m[t], sl[wave][16 * t + c] = l;
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
      for (int d = 0; d < D / 16; d += 4)
        *reinterpret_cast<float4 *>(&so[wave][16 * t + c][D / 16 * (4 * g + r) + d]) =
            make_float4(rows.o[t][d][r], rows.o[t][d + 1][r], rows.o[t][d + 2][r], rows.o[t][d + 3][r]);
  }
  __syncthreads();
  int odd_any = 0;
#pragma unroll
  for (int w = 0; w < WK; w++) odd_any |= sodd[w];
  join_waves<D, TQ, kRows>(p, share, seq, index, hk, first < end, so, sm, sl, [&](float *y, int own, int d) {
    if (odd_any) odd_values<D, TKV>(y, p, seq, tiles, first, end, table, hk, own, d);
  });
  clear_rest<D, TQ, kRows>(p);
}

// ---- 4 bits ----
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// 16 or 4 bytes a lane from anywhere to LDS at lds + 16 (4) lane, without a register in between.  The compiler does not know of
// these loads: copies_wait() has to come before what they bring is read.
__device__ __forceinline__ void copy16(const char *from, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ void copy4(const char *from, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(from), "s"(lds) : "memory", "m0");
}
// (from a base that all lanes share)
__device__ __forceinline__ void copy16(const char *base, uint32_t offset, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "s"(lds) : "memory", "m0");
}
#pragma clang diagnostic pop
// Waits until at most N of the wave's copies are on their way, and for its reads of LDS.
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint32_t lds_address(const void *p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void *)p;
}

// Few query rows (or many) over 4 bits: 4 waves over tiles of 32 keys of their own, each with a ring of tiles in LDS that direct
// loads fill: few instructions for many small rows, no registers for what is on its way, and the operands' order comes from
// how LDS is read.  Row r of 16 lies in slot 4 (r % 4) + r / 4, its 16-byte pieces in another order by row (piece ^ r % 4, of two
// pieces piece ^ r / 2 % 2): reads of 16 key rows' same piece and of four value rows' same part fall on different banks.
// Bound by instructions: 16 tokens, 8 key heads of 128, 8,191 .. 32,768 rows, 378 MB, 86 us (4.4 TB/s), about 400 vector and 180
// scalar instructions a tile and wave, the vector units busy 58% of the time.  Straight into registers, 36 loads a tile, the call
// that takes 91 us now took 125.  Three blocks a compute unit with two tiles each 99 us, two with four tiles 112 (16-bit queries,
// D 128).  Two row tiles of 16 for prompts: 4,096 tokens 484 -> 400 us (343 TFLOP/s).  fp16 queries as they are, by fp16 products of the
// codes, instead of two bf16 planes: 487 -> 399 us there, 109 -> 105 for 16 tokens.
template <int D, class TQ>
constexpr int kCodeBlocks = D == 64 ? (TQ::kBytes == 4 ? 3 : 4) : TQ::kBytes == 4 ? 2 : 3;  // a compute unit
template <int D, class TQ, int RT>
__global__ __launch_bounds__(256, (RT == 2 ? 2 : kCodeBlocks<D, TQ>)) void paged_codes_kernel(Args p) {
  constexpr int WK = 4, kRows = 16 * RT, G = D / 64, kStages = kCodeBlocks<D, TQ> == 2 ? 4 : D == 64 ? 3 : 2, kLoads = D == 128 ? 6 : 3;
  constexpr int kRow = D / 2, kCodes = kTileKeys * kRow, kPairs = kTileKeys * 4 * G, kStage = 2 * (kCodes + kPairs);  // bytes
  struct Join {
    float so[WK][kRows][D + 4], sm[WK][kRows], sl[WK][kRows];
  };
  constexpr size_t kRing = (size_t)WK * kStages * kStage, kBytes = kRing > sizeof(Join) ? kRing : sizeof(Join);
  __shared__ __attribute__((aligned(256))) char mem[kBytes];
  const PagedAttn &a = p.a;
  const Pages &pg = a.pages;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
  const int hk = blockIdx.x % pg.Hk, index = blockIdx.x / pg.Hk;
  const Share share = share_of<kRows, kTileKeys>(p, index, hk);
  if (share.n == 0) return clear_rest<D, TQ, kRows>(p);
  const Seq seq = seq_of<kRows>(p, share);
  const Tiles<kTileKeys> tiles(a, seq.p0, seq.p1);
  const int first = min(share.first, tiles.n), end = min(share.end, tiles.n);
  const int32_t *table = a.table + share.b * a.tab_b;

  // Copies of a tile.
  const uint32_t ring = lds_address(mem) + wave * kStages * kStage;
  const int slot = D == 128 ? lane >> 2 : (lane & 31) >> 1, row = (slot & 3) * 4 + (slot >> 2);
  const int piece = D == 128 ? (lane & 3) ^ (row & 3) : (lane & 1) ^ (row >> 1 & 1);
  const uint32_t k_at = row * (uint32_t)pg.k_r + 16 * piece, v_at = row * (uint32_t)pg.v_r + 16 * piece;
  const uint32_t kp_at = D == 128 ? (lane >> 1 & 15) * (uint32_t)pg.kp_r + 4 * (lane & 1) : (lane & 15) * (uint32_t)(lane < 32 ? pg.kp_r : pg.vp_r);
  const uint32_t vp_at = (lane >> 1 & 15) * (uint32_t)pg.vp_r + 4 * (lane & 1);
  const char *kb = pg.k + hk * pg.k_h, *vb = pg.v + hk * pg.v_h, *kpb = pg.kp + hk * pg.kp_h, *vpb = pg.vp + hk * pg.vp_h;
  auto copy = [&](const Ids &ids, uint32_t lds) {
    const char *k[2], *v[2], *kp[2], *vp[2];
    bases_of(p, ids, kb, pg.k_p, pg.k_r, k), bases_of(p, ids, vb, pg.v_p, pg.v_r, v);
    bases_of(p, ids, kpb, pg.kp_p, pg.kp_r, kp), bases_of(p, ids, vpb, pg.vp_p, pg.vp_r, vp);
    if constexpr (D == 128) {
#pragma unroll
      for (int h = 0; h < 2; h++) {
        copy16(k[h], k_at, lds + h * 16 * kRow);
        copy16(v[h], v_at, lds + kCodes + h * 16 * kRow);
      }
      copy4((lane < 32 ? kp[0] : kp[1]) + kp_at, lds + 2 * kCodes);
      copy4((lane < 32 ? vp[0] : vp[1]) + vp_at, lds + 2 * kCodes + kPairs);
    } else {
      copy16((lane < 32 ? k[0] : k[1]) + k_at, lds);
      copy16((lane < 32 ? v[0] : v[1]) + v_at, lds + kCodes);
      const char *lo = lane < 32 ? kp[0] : vp[0], *hi = lane < 32 ? kp[1] : vp[1];
      copy4((lane & 16 ? hi : lo) + kp_at, lds + 2 * kCodes);
    }
  };
  // Reads of a tile.
  const uint32_t key_at = ((c & 3) * 4 + (c >> 2)) * kRow + 16 * ((g >> 1) ^ (D == 128 ? c & 3 : c >> 1 & 1)) + 8 * (g & 1);
  const uint32_t value_at = kCodes + g * kRow + 16 * (c >> 3) + 2 * (c & 7), pair_at = 2 * kCodes + 16 * G * g;
  auto read = [&](CodeRegs<D> &x, uint32_t lds) {
    using Two = __attribute__((address_space(3))) const u32x2;
    using Four = __attribute__((address_space(3))) const u32x4;
    using Short = __attribute__((address_space(3))) const uint16_t;
#pragma unroll
    for (int h = 0; h < 2; h++) {
#pragma unroll
      for (int i = 0; i < G; i++) {
        const u32x2 w = *(Two *)(uintptr_t)(lds + (key_at ^ 32 * i) + h * 16 * kRow);
        x.k[h][i][0] = w[0], x.k[h][i][1] = w[1];
      }
#pragma unroll
      for (int i = 0; i < G; i++) {
        const u32x4 kp = *(Four *)(uintptr_t)(lds + pair_at + h * 64 * G + 16 * i);
        const u32x4 vp = *(Four *)(uintptr_t)(lds + pair_at + kPairs + h * 64 * G + 16 * i);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int at = 4 * i + e;  // dwords [row][group]
          x.kp[4 * h + at / G][at % G] = kp[e], x.vp[4 * h + at / G][at % G] = vp[e];
        }
      }
#pragma unroll
      for (int r = 0; r < 4; r++)
#pragma unroll
        for (int i = 0; i < G; i++)
          x.v[4 * h + r][i] = *(Short *)(uintptr_t)(lds + (value_at ^ 32 * i ^ 16 * (D == 128 ? r : r >> 1)) + (4 * r + 16 * h) * kRow);
    }
  };

  const char *at[RT];
  int pos[RT];
#pragma unroll
  for (int t = 0; t < RT; t++) {
    const int r = min(share.tile * kRows + 16 * t + c, seq.rows - 1), i = p.token(r), head = hk * p.group + r - i * p.group;
    pos[t] = seq.len - seq.n + i;
    at[t] = static_cast<const char *>(a.q) + ((seq.first_token + i) * a.q_t + head * a.q_h) * TQ::kBytes;
  }
  Rows4<D, TQ, RT> rows;
  rows.load(at, a.scale, g);
  copies_wait<0>();  // (the queries are there: from here on the wave's loads are counted by hand)

  // Tiles first + wave, in steps of WK: n of them.  `missing`: two bits a tile, the next one's lowest.
  const int n = max(0, (end - first - wave + WK - 1) / WK), u0 = first + wave;
  uint32_t missing = 0;
  Ids next;
  auto fetch = [&](int i) { return ids_of(p, table, tiles.key(u0 + WK * min(i, n - 1)), seq.p1 + 1); };
  auto issue = [&](int i) {
    missing |= next.missing(a) << 2 * (kStages - 1);
    copy(next, ring + i % kStages * kStage);
    next = fetch(i + 1);
  };
  if (n > 0) {
    next = fetch(0);
#pragma unroll
    for (int i = 0; i < kStages - 1; i++) {
      if (i < n) issue(i);
      missing >>= 2;
    }
  }
  auto step = [&](auto is_edge, int i, int key0, int gone) {
    constexpr bool kEdge = decltype(is_edge)::value;
    CodeRegs<D> x;
    read(x, ring + i % kStages * kStage);
    floatx4 s[2][RT];
    rows.scores(s, x);
    uint32_t seen[RT] = {};
    if constexpr (kEdge) {
#pragma unroll
      for (int t = 0; t < RT; t++) {
        seen[t] = seen_bits(a, pos[t], key0) >> (4 * g);
#pragma unroll
        for (int e = 0; e < 8; e++)
          if (gone >> (e >> 2) & 1) s[e >> 2][t][e & 3] = NAN;
      }
    }
    rows.limit(s, kEdge, seen);
    rows.weigh(s);
    rows.template add<kEdge>(s, seen, x);
  };
  // waits for tile i, sends for the one kStages - 1 later into the place of the one before
  auto turn = [&](int i, int &key0, int &gone) {
    if (i + kStages - 2 < n) copies_wait<kLoads * (kStages - 2)>();
    else copies_wait<0>();
    if (i + kStages - 1 < n) issue(i + kStages - 1);
    key0 = tiles.key(u0 + WK * i), gone = missing & 3;
    missing >>= 2;
  };
  for (int i = 0; i < n;) {
    int key0, gone;
    turn(i, key0, gone);
    while (all_see<kTileKeys>(a, seq.p0, seq.p1, key0) && gone == 0) {
      step(std::false_type{}, i, key0, 0);
      if (++i == n) break;
      turn(i, key0, gone);
    }
    if (i == n) break;
    step(std::true_type{}, i, key0, gone);
    i++;
  }

  copies_wait<0>();
  __syncthreads();  // (the rings' memory is used again)
  Join &join = *reinterpret_cast<Join *>(mem);
#pragma unroll
  for (int t = 0; t < RT; t++) {
    const float l = col_sum(rows.l[t]);
    if (g == 0) join.sm[wave][16 * t + c] = rows.m[t], join.sl[wave][16 * t + c] = l;
#pragma unroll
    for (int i = 0; i < G; i++) {
      const float plus = col_sum(rows.ob[t][i]);
#pragma unroll
      for (int r = 0; r < 4; r++) {
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; e++) y[e] = __builtin_fmaf(rows.o[t][4 * i + e][r], 16.0f, plus);
        *reinterpret_cast<float4 *>(&join.so[wave][16 * t + c][64 * i + 4 * (4 * g + r)]) = make_float4(y[0], y[1], y[2], y[3]);
      }
    }
  }
  __syncthreads();
  join_waves<D, TQ, kRows>(p, share, seq, index, hk, first < end, join.so, join.sm, join.sl, [](float *, int, int) {});
  clear_rest<D, TQ, kRows>(p);
}

// ---- many query rows ----
constexpr int kLongKeys = 64;  // keys of a tile
constexpr int kLongRows = 128; // rows of a block: 32 a wave

// A row's 16-byte pieces lie in LDS in the order piece ^ swizzle(row): what a wave reads at a time, one piece of many key rows
// or a few neighbours of 4 value rows, then falls on different banks.
template <int D>
__device__ __forceinline__ int swizzle(int row) {
  return D == 128 ? (row & 3) << 2 | (row >> 2 & 3) : (row >> 1 & 1) << 2 | (row >> 2 & 3);
}
template <class T>
__device__ __forceinline__ floatx16 mfma32(const uint32_t (&a)[4], const uint32_t (&b)[4], floatx16 c) {
  const u32x4 x = {a[0], a[1], a[2], a[3]}, y = {b[0], b[1], b[2], b[3]};
  if constexpr (std::is_same_v<T, Bf16>) return ITTS_MFMABF(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
  else return ITTS_MFMA16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, y), c, 0, 0, 0);
}

// A pair of 16-bit values times a power of two (what is not 0 stays so).
template <class T>
__device__ __forceinline__ uint32_t scale_pair(uint32_t w, float f) {
  float a, b;
  if constexpr (std::is_same_v<T, Bf16>) a = __uint_as_float(w << 16), b = __uint_as_float(w & 0xffff0000u);
  else a = low_half(w), b = high_half(w);
  constexpr float kLeast = std::is_same_v<T, Bf16> ? 0x1p-126f : 0x1p-24f;
  const float x = __builtin_copysignf(fmaxf(fabsf(a * f), fminf(fabsf(a), kLeast)), a);
  const float y = __builtin_copysignf(fmaxf(fabsf(b * f), fminf(fabsf(b), kLeast)), b);
  if constexpr (std::is_same_v<T, Bf16>) return cut_pair(x, y);
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x, y));
}

// Whether it is so anywhere in a block of four waves, by way of LDS that is no longer needed.
__device__ __forceinline__ bool any_in_block(bool v, void *mem) {
  int *flags = static_cast<int *>(mem);
  const bool wave = __ballot(v) != 0;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) flags[threadIdx.x >> 6] = wave;
  __syncthreads();
  return (flags[0] | flags[1] | flags[2] | flags[3]) != 0;
}

// Many query rows over 16-bit caches: 4 waves with 32 rows each over the same tiles of 64 keys, which come to LDS by direct
// loads, a tile ahead of their use (keys two: a tile's scores are formed while the exponentials of the one before are).
// S^T = K Q^T by 32 x 32 products: lane (c, h) holds keys 8 (i / 4) + 4 h + i % 4 of query c in register i, the B operand of
// O^T = V^T P^T in the order in which the transposing LDS load gives V's rows.
// One prompt of 8,192 tokens, 32 heads of 128 over 8 key heads, bf16: 680 to 780 us by the card's clock, 809 to 705 TFLOP/s (in turn
// on one card 755 us, without the waves' priorities 803); the
// matrix units are busy 58% of its cycles (a probability's second plane is a third of their work), the vector units 51%, at
// 1.74 GHz (the card lowers its clock under this load).  On the way there: 16 x 16 tiles copied through registers 1,380 us;
// 32 x 32 with both kinds of tiles in one loop 1,083 (accumulators copied every turn, queries spilled); a loop of its own for tiles
// that all see 828; probabilities of a tile's second half left waiting for the next tile's first exponentials 820; keys read
// ahead of their products 796.
template <int D, class TQ, class TKV>
__global__ __launch_bounds__(256, (TQ::kBytes == 4 ? (D == 64 ? 2 : 1) : D == 64 ? 3 : 2)) void paged_rows_kernel(Args p) {
  constexpr int KT = kLongKeys, kPieces = D * TKV::kBytes / 16, kTile = KT * kPieces, kCopies = kTile / 256;
  constexpr int NQ = TQ::kBytes == 4 ? 3 : 1, NP = kProbPlanes<TQ>;
  constexpr float kLag = 5.0f, kUp = std::is_same_v<TKV, F16> ? 10.0f : 0.0f;
  __shared__ __attribute__((aligned(65536))) u32x4 key_mem[2][kTile];
  __shared__ __attribute__((aligned(256))) u32x4 value_mem[3][kTile];
  const PagedAttn &a = p.a;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 31, h = lane >> 5;
  const int hk = blockIdx.x % a.pages.Hk, index = blockIdx.x / a.pages.Hk;
  const Share share = share_of<kLongRows, KT>(p, index, hk);
  if (share.n == 0) return clear_rest<D, TQ, kLongRows>(p);
  const Seq seq = seq_of<kLongRows>(p, share);
  const Tiles<KT> tiles(a, seq.p0, seq.p1);
  const int first = min(share.first, tiles.n), end = min(share.end, tiles.n);
  const int32_t *table = a.table + share.b * a.tab_b;

  // This wave's copies: rows 16 wave .. of a tile, in kCopies loads of 64 pieces.
  const char *kb = a.pages.k + hk * a.pages.k_h, *vb = a.pages.v + hk * a.pages.v_h;
  uint32_t k_at[kCopies], v_at[kCopies];
#pragma unroll
  for (int i = 0; i < kCopies; i++) {
    const int row = (64 * i + lane) / kPieces, piece = (lane % kPieces) ^ swizzle<D>(row);
    k_at[i] = row * (uint32_t)a.pages.k_r + 16 * piece, v_at[i] = row * (uint32_t)a.pages.v_r + 16 * piece;
  }
  // page of the wave's rows of a tile (rows that nothing sees: the tile's first page), and which of a tile's pages do not exist
  auto place = [&](int u, int &at) {
    const int key0 = tiles.key(u), key = key0 + 16 * wave < seq.p1 + 1 ? key0 + 16 * wave : key0, page = page_of(key, p.page_mul);
    at = key - page * a.pages.size;
    return uniform_load(table + page);
  };
  auto missing_of = [&](int u) {
    const int key0 = tiles.key(u);
    int missing = 0;
#pragma unroll
    for (int i = 0; i < KT / 16; i++) {
      const int key = key0 + 16 * i < seq.p1 + 1 ? key0 + 16 * i : key0;
      missing |= (uint32_t)uniform_load(table + page_of(key, p.page_mul)) < (uint32_t)a.pages.n ? 0 : 1 << i;
    }
    return missing;
  };
  auto copy = [&](const char *from, int64_t page_step, int64_t row_step, const uint32_t (&offset)[kCopies], int page, int at, u32x4 *to) {
    const char *base = from + ((uint32_t)page < (uint32_t)a.pages.n ? page : 0) * page_step + at * row_step;
#pragma unroll
    for (int i = 0; i < kCopies; i++) copy16(base, offset[i], lds_address(to + 16 * kPieces * wave + 64 * i));
  };

  // The wave's query rows: lane (c, h) elements 16 j + 8 h .. of row c.
  uint32_t q[NQ][D / 16][4];
  const int r = min(share.tile * kLongRows + 32 * wave + c, seq.rows - 1), token = p.token(r), pos = seq.len - seq.n + token;
  const float by = a.scale * kLog2e, scale = NQ == 3 ? 1.0f : fmaxf(fabsf(by), 0x1p-120f);
  {
    const char *at = static_cast<const char *>(a.q) + ((seq.first_token + token) * a.q_t + (hk * p.group + r - token * p.group) * a.q_h + 8 * h) * TQ::kBytes;
    const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0;
#pragma unroll
    for (int j = 0; j < D / 16; j++) {
      uint32_t raw[2 * TQ::kBytes];
      load_dwords<2 * TQ::kBytes>(at + 16 * j * TQ::kBytes, raw);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        if constexpr (NQ == 3) {
          uint32_t w[3];
          cut3(__uint_as_float(raw[2 * e]) * by, __uint_as_float(raw[2 * e + 1]) * by, w);
#pragma unroll
          for (int i = 0; i < 3; i++) q[i][j][e] = w[i];
        } else {
          q[0][j][e] = raw[e] ^ flip;
        }
      }
    }
  }
  floatx16 o[D / 32] = {};
  float m = -INFINITY, l = 0.0f;
  uint32_t odd = 0;

  // LDS addresses from a base each, every one an exclusive or away: kept for all reads of a tile they would not fit the registers.
  // Keys: row c, piece 2 j + h.  Values: rows 8 i + 4 h + (lane / 4) % 4 of 16, the four elements that the transposing load takes.
  constexpr uint32_t kRowBytes = 16 * kPieces, kTileBytes = KT * kRowBytes;
  using Lds = __attribute__((address_space(3))) const char;
  uint32_t key_at, value_at;
  {
    const int row = 4 * h + (lane >> 2 & 3), piece = 2 * (lane >> 4 & 1) + (lane >> 1 & 1);
    key_at = (uint32_t)(uintptr_t)(Lds *)key_mem + c * kRowBytes + 16 * (h ^ swizzle<D>(c));
    value_at = (uint32_t)(uintptr_t)(Lds *)value_mem + row * kRowBytes + 16 * (piece ^ swizzle<D>(row)) + 8 * (lane & 1);
  }
  static_assert(2 * kTileBytes <= 65536 && (2 * kTileBytes & (2 * kTileBytes - 1)) == 0, "a buffer's bit in an address");
  auto read_keys = [&](u32x4 (&k)[D / 16], int t, uint32_t base) {
#pragma unroll
    for (int j = 0; j < D / 16; j++)
      k[j] = *(__attribute__((address_space(3))) const u32x4 *)(uintptr_t)((base ^ 32 * j) + 32 * t * kRowBytes);
  };
  auto scores = [&](floatx16 &s, const u32x4 (&w)[D / 16]) {
    s = floatx16{};
#pragma unroll
    for (int j = 0; j < D / 16; j++) {
      const uint32_t k[4] = {w[j][0], w[j][1], w[j][2], w[j][3]};
#pragma unroll
      for (int i = NQ - 1; i >= 0; i--) s = mfma32<TKV>(k, q[i][j], s);
    }
  };

  floatx16 s[2];                      // scores of a tile's halves
  uint32_t planes[2][2][NP][4] = {};  // their probabilities, of 16 keys each
  auto weigh = [&](int t, float ms) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][2 * i], scale, -ms));
      const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][2 * i + 1], scale, -ms));
      l += p0, l += p1;
      uint32_t w[NP];
      cut_pos<TKV, NP>(p0, p1, w);
#pragma unroll
      for (int k = 0; k < NP; k++) planes[t][i >> 2][k][i & 3] = w[k];
    }
  };
  auto add = [&](int t, uint32_t base) {
#pragma unroll
    for (int g = 0; g < 2; g++)
#pragma unroll
      for (int d = 0; d < D / 32; d++) {
        uint32_t vt[4];
#pragma unroll
        for (int i = 0; i < 2; i++) {  // keys 8 i + 4 h .. of the 16
          typedef short s16x4 __attribute__((ext_vector_type(4)));
          using Piece = __attribute__((address_space(3))) s16x4;
          const uint32_t at = (base ^ 64 * d ^ 32 * i) + (32 * t + 16 * g + 8 * i) * kRowBytes;
          const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Piece *)(uintptr_t)at));
          vt[2 * i] = w[0], vt[2 * i + 1] = w[1];
        }
#pragma unroll
        for (int k = NP - 1; k >= 0; k--) o[d] = mfma32<TKV>(vt, planes[t][g][k], o[d]);
      }
  };

  if (first < end) {
    int next_page, next_at;  // the page of the tile after the next
    int page1, at1, at0;     // and of the next one
    const int page0 = place(first, at0);
    page1 = place(min(first + 1, end - 1), at1);
    next_page = place(min(first + 2, end - 1), next_at);
    copy(kb, a.pages.k_p, a.pages.k_r, k_at, page0, at0, key_mem[0]);
    copy(kb, a.pages.k_p, a.pages.k_r, k_at, page1, at1, key_mem[1]);
    copy(vb, a.pages.v_p, a.pages.v_r, v_at, page0, at0, value_mem[0]);
#pragma unroll
    for (int i = 0; i < kCopies; i++) value_mem[2][64 * kCopies * wave + 64 * i + lane] = u32x4{};  // (probabilities of 0 times it)
    copies_wait<0>();
    __syncthreads();
    u32x4 k[D / 16];
    read_keys(k, 0, key_at);
    scores(s[0], k);
    read_keys(k, 1, key_at);
    scores(s[1], k);
    __syncthreads();
    // Here: a tile's scores and values (ring), the next one's keys, the probabilities of the second half of the one before and its
    // values; on their way: what follows.  While the scores of one half become probabilities, the products of what is there run.
    int ring = 0;
    for (int u = first; u < end; u++) {
      const int buf = u - first & 1, ring1 = ring == 2 ? 0 : ring + 1, ring2 = ring == 0 ? 2 : ring - 1;
      copy(vb, a.pages.v_p, a.pages.v_r, v_at, page1, at1, value_mem[ring1]);
      copy(kb, a.pages.k_p, a.pages.k_r, k_at, next_page, next_at, key_mem[buf]);
      page1 = next_page, at1 = next_at;
      next_page = place(min(u + 3, end - 1), next_at);
      const int key0 = tiles.key(u), missing = missing_of(u);
      if (!all_see<KT>(a, seq.p0, seq.p1, key0) || missing != 0) {
        // values that are no finite numbers leave the tile (odd_values), and whatever lies past the last row; keys that are not
        // seen count as -inf, those of missing pages as NaN
#pragma unroll
        for (int i = 0; i < kCopies; i++) {
          u32x4 &at = value_mem[ring][64 * kCopies * wave + 64 * i + lane];
          const bool in = key0 + 16 * wave + (64 * i + lane) / kPieces <= seq.p1;
          u32x4 w = at;
#pragma unroll
          for (int e = 0; e < 4; e++) {
            uint32_t keep = (w[e] & TKV::kOddBits) == TKV::kOddBits ? 0xffff0000u : ~0u;
            keep = (w[e] & TKV::kOddBits << 16) == TKV::kOddBits << 16 ? keep & 0xffffu : keep;
            odd |= in ? ~keep : 0;
            w[e] &= in ? keep : 0;
          }
          at = w;
        }
#pragma unroll
        for (int t = 0; t < 2; t++) {
          const uint32_t seen = seen_bits(a, pos, key0 + 32 * t) >> (4 * h);
#pragma unroll
          for (int i = 0; i < 16; i++) {
            if (missing >> (2 * t + (i >> 3)) & 1) s[t][i] = NAN;
            s[t][i] = seen & 1u << (8 * (i >> 2) + (i & 3)) ? s[t][i] : -INFINITY;
          }
        }
        __syncthreads();
      }
      float top = fmaxf(s[0][0], s[1][0]);
#pragma unroll
      for (int i = 1; i < 16; i++) top = fmaxf(fmaxf(s[0][i], s[1][i]), top);
      top *= scale;
      if (__ballot(top > m + kLag)) {
        // (maxima are whole numbers: the probabilities that wait rescale exactly)
        const float mn = ceilf(fmaxf(m, fmaxf(top, __shfl_xor(top, 32, 64))));
        const float f = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.0f : mn));
        m = mn;
        l *= f;
#pragma unroll
        for (int d = 0; d < D / 32; d++) o[d] *= f;
#pragma unroll
        for (int g = 0; g < 2; g++)
#pragma unroll
          for (int k = 0; k < NP; k++)
#pragma unroll
            for (int i = 0; i < 4; i++) planes[1][g][k][i] = scale_pair<TKV>(planes[1][g][k][i], f);
      }
      const float ms = (m == -INFINITY ? 0.0f : m) - kUp;
      uint32_t keys = key_at ^ (buf ? 0 : kTileBytes), values = value_at + ring * kTileBytes, waiting = value_at + ring2 * kTileBytes;
      asm volatile("" : "+v"(keys), "+v"(values), "+v"(waiting));
      // (the barriers keep what is read ahead where it is)
      read_keys(k, 0, keys);
      weigh(0, ms);
      add(1, waiting);
      __builtin_amdgcn_sched_barrier(0);
      // (whoever is in this half goes first: two waves of a SIMD then leave each other the vector unit and the matrix unit in turn)
      __builtin_amdgcn_s_setprio(1);
      scores(s[0], k);
      read_keys(k, 1, keys);
      weigh(1, ms);
      add(0, values);
      __builtin_amdgcn_sched_barrier(0);
      scores(s[1], k);
      __builtin_amdgcn_s_setprio(0);
      ring = ring1;
      copies_wait<0>();
      __syncthreads();
    }
    add(1, value_at + (ring == 0 ? 2 : ring - 1) * kTileBytes);
  }

  const bool odd_any = any_in_block(odd != 0, key_mem);  // (a wave has cleaned its rows of the tiles)
  l += __shfl_xor(l, 32, 64);
  const int row = 32 * wave + c;
  if (share.tile * kLongRows + row < seq.rows) {
#pragma unroll
    for (int d = 0; d < D / 32; d++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        float y[4] = {o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
        const int e = 32 * d + 8 * i + 4 * h;
        if (odd_any) odd_values<D, TKV>(y, p, seq, tiles, first, end, table, hk, pos, e);
        put4<D, TQ, kLongRows>(p, share, seq, index, hk, row, e, y, m, l, pos >= 0, first < end);
      }
  }
  clear_rest<D, TQ, kLongRows>(p);
}

// Joins the shares' results of a row: a wave a row, D / 4 lanes with four elements each for every fourth (D 128: second)
// share, added in their order there and then over the lane groups.  4 to 5 us, most of them the launch.
template <int D, class TQ, int ROWS>
__global__ __launch_bounds__(256) void paged_join_kernel(Args p) {
  constexpr int kLanes = D / 4, kGroups = 64 / kLanes;
  const PagedAttn &a = p.a;
  const int lane = threadIdx.x & 63, d = lane % kLanes * 4, s0 = lane / kLanes;
  const int item = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
  if (item >= a.tokens * a.H) return;
  const int token = item / a.H, head = item - token * a.H, hk = head / p.group;
  const Owner of = owner_of(a.starts, a.batch, a.tokens, token);
  const int2 dealt = of.b < 0 ? make_int2(0, 0) : p.dealt[of.b];
  const int S = dealt.y;
  char *out = static_cast<char *>(a.out) + (token * a.o_t + head * a.o_h + d) * TQ::kBytes;
  if (S <= 1) {  // (1: that block has written the row; 0: the token belongs to no sequence)
    if (S == 0 && s0 == 0) store4<TQ>(out, 0.0f, 0.0f, 0.0f, 0.0f);
    return;
  }
  const int r = (token - of.first) * p.group + head - hk * p.group, tile = r / ROWS, tiles = (of.n * p.group + ROWS - 1) / ROWS;
  const int index = dealt.x + (tiles - 1 - tile) * S;
  const size_t at = ((size_t)hk * p.parts + index) * ROWS + (r - tile * ROWS);
  const float *part = a.part + at * D + d;
  const float2 own = p.ml[at + (size_t)min(lane, S - 1) * ROWS];  // (at most 64 blocks)
  float4 o = *reinterpret_cast<const float4 *>(part + (size_t)min(s0, S - 1) * ROWS * D);  // (before what weighs it is there)
  const float top = wave_max(own.x), ms = top == -INFINITY ? 0.0f : top;
  const bool none = __ballot(own.x == INFINITY && own.y == 0.0f) != 0;
  const float f_own = __builtin_amdgcn_exp2f(own.x - ms);
  // (a weight that is positive, if not as a float: times an infinity it is that)
  auto weighed = [](float f, float y) { return fabsf(y) < INFINITY ? f * y : y; };
  float sum = 0.0f, x[4] = {};
  for (int s1 = 0; s1 < S; s1 += kGroups) {
    const int s = min(s1 + s0, S - 1);
    const float4 next = *reinterpret_cast<const float4 *>(part + (size_t)min(s + kGroups, S - 1) * ROWS * D);
    const float m = __shfl(own.x, s, 64), l = __shfl(own.y, s, 64), f = __shfl(f_own, s, 64);
    const bool in = s1 + s0 < S && !(m == -INFINITY && l == 0.0f);  // without keys nothing was stored
    const bool num = in && l == l;  // (else the sum is NaN, and nothing may have been stored)
    sum += in ? f * l : 0.0f;
    x[0] += num ? weighed(f, o.x) : 0.0f, x[1] += num ? weighed(f, o.y) : 0.0f;
    x[2] += num ? weighed(f, o.z) : 0.0f, x[3] += num ? weighed(f, o.w) : 0.0f;
    o = next;
  }
#pragma unroll
  for (int step = kLanes; step < 64; step *= 2) {
    sum += __shfl_xor(sum, step, 64);
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] += __shfl_xor(x[e], step, 64);
  }
  if (s0 > 0) return;
  const float inv = 1.0f / sum;
#pragma unroll
  for (int e = 0; e < 4; e++) x[e] = none ? 0.0f : x[e] * inv;
  store4<TQ>(out, x[0], x[1], x[2], x[3]);
}

int code_blocks(int D, int type) {
  return D == 64 ? (type == kOpF32 ? kCodeBlocks<64, F32> : kCodeBlocks<64, Bf16>)
                 : (type == kOpF32 ? kCodeBlocks<128, F32> : kCodeBlocks<128, Bf16>);
}
// How a launch is laid out: rows of a block, blocks of a key head, or `parts` that share the keys.
struct Plan {
  bool many;  // paged_rows_kernel
  int RT;     // tiles of 16 rows of a block otherwise
  int rows, blocks, parts, unit, least, per_token;
};
Plan make_plan(const PagedAttn &a, int n_cu) {
  Plan p;
  const int group = a.H / a.pages.Hk, D = a.pages.D;
  const bool wide = a.type == kOpF32, codes = a.pages.type == kOpI4;
  // Query rows of a sequence on average.  Shared tiles pay from here on (8 sequences of 4,000 rows, us, waves with keys of their own
  // and shared tiles): bf16, 8 key heads of 128, 32 rows 34, 41, 64 rows 51, 43, 128 rows 81, 50; 16 of 64, 64 rows 38, 45, 128
  // rows 52, 51; fp32 over bf16 64 rows 53, 74, 128 rows 83, 83; of 64, 128 rows 57, 70.
  const int64_t rows = (int64_t)a.tokens * group / std::max(1, a.batch);
  p.many = !codes && a.pages.type != kOpF32 && rows >= 8192 / D * (wide ? 2 : 1);
  // (fp32 queries of 128 elements would not fit the registers twice)
  p.RT = !p.many && rows >= 32 && (D == 64 || (codes && !wide)) ? 2 : 1;
  p.rows = p.many ? kLongRows : 16 * p.RT, p.unit = p.many ? 1 : 2, p.least = 2;
  // row tiles at most: a sequence's last one may be short
  const int a_token = (group + p.rows - 1) / p.rows;
  const int64_t apart = (int64_t)a.tokens * a_token, together = (int64_t)a.tokens * group / p.rows + a.batch, most = std::min(apart, together);
  p.per_token = apart <= together ? a_token : 0;
  p.parts = 0, p.blocks = (int)most;
  const int at_once = n_cu * (codes && !p.many && p.RT == 1 ? code_blocks(D, a.type) : 2) / a.pages.Hk;
  const int64_t seen = a.window > 0 ? std::min<int64_t>(a.max_rows, (int64_t)a.window + std::min(a.sinks, a.max_rows)) : a.max_rows;
  // Keys are shared where row tiles alone would not fill the card and rows may be enough for the second launch to pay: a wave's
  // time goes by their bytes, over 4 bits by their number.  One token, us a call, alone and shared: 20 bf16 heads of 64 over
  // 1,734 rows 15.4, 18.6, 2,000 rows 17.4, 16.0, 3,200 rows 22.1, 16.2; 8 of 128 over 1,100 rows 16.5, 16.2, 2,800 rows 30.3, 16.3;
  // 20 fp32 heads of 64 over 850 rows 15.4, 16.3, 1,100 rows 17.7, 16.7; 4 bits, 16 of 64 over 1,100 rows 16.6, 17.5, 1,600 rows
  // 20.9, 17.9; 8 of 128 over 1,100 rows 18.4, 18.0, 3,000 rows 38.1, 18.4.  Shared tiles of 64 keys pay where a block loses more
  // than ten of them, one of two on a compute unit being slower by 1.6: 128 of 1,100 rows, 20 heads of 64, 30.5, 19.7; 512 of them
  // 31.3, 29.3; 1,100 of them 30.0, 37.1; 1,536 of 4,000 88.6, 80.7; 32 heads of 128 over 8, 512 of 2,000 62.3, 46.7; 1,024 of
  // them 64.9, 66.7; 1,024 of 6,000 173, 146.
  const bool far = p.many ? seen / 64 * (5 * at_once - 8 * most) > (int64_t)50 * at_once
                   : codes ? seen > 1152 : seen * D * (a.pages.type == kOpF32 ? 4 : 2) > (224 << 10);
  if (most < at_once && far) p.parts = p.blocks = std::max(at_once, (int)most);
  return p;
}

size_t part_rows(const PagedAttn &a, const Plan &p) { return (size_t)a.pages.Hk * p.parts * p.rows; }
Args make_args(const PagedAttn &a, const Plan &p) {
  const int group = a.H / a.pages.Hk;
  float *ml = a.part + part_rows(a, p) * a.pages.D;
  return Args{a, p.blocks, p.parts, group, (uint32_t)(((1ull << 32) + group - 1) / group), page_mul(a.pages.size), a.pages.size % 32 == 0, p.per_token, p.unit, p.least,
              reinterpret_cast<float2 *>(ml), reinterpret_cast<int2 *>(ml + 2 * part_rows(a, p))};
}
template <int D, class TQ, int ROWS, class K>
hipError_t launch_kernel(K kernel, const PagedAttn &a, const Plan &p, hipStream_t s) {
  const Args args = make_args(a, p);
  hipLaunchKernelGGL(kernel, dim3((unsigned)((int64_t)p.blocks * a.pages.Hk)), dim3(256), 0, s, args);
  if (hipError_t e = hipGetLastError(); e != hipSuccess || p.parts == 0) return e;
  hipLaunchKernelGGL((paged_join_kernel<D, TQ, ROWS>), dim3((unsigned)(((int64_t)a.tokens * a.H + 3) / 4)), dim3(256), 0, s, args);
  return hipGetLastError();
}
template <int D, class TQ, class TKV>
hipError_t launch_d(const PagedAttn &a, const Plan &p, hipStream_t s) {
  if constexpr (std::is_same_v<TKV, Bf16> || std::is_same_v<TKV, F16>)
    if (p.many) return launch_kernel<D, TQ, kLongRows>(paged_rows_kernel<D, TQ, TKV>, a, p, s);
  if constexpr (std::is_same_v<TKV, I4>) {
    if constexpr (D == 64 || TQ::kBytes == 2)
      if (p.RT == 2) return launch_kernel<D, TQ, 32>(paged_codes_kernel<D, TQ, 2>, a, p, s);
    return launch_kernel<D, TQ, 16>(paged_codes_kernel<D, TQ, 1>, a, p, s);
  } else {
    if constexpr (D == 64)
      if (p.RT == 2) return launch_kernel<D, TQ, 32>(paged_attn_kernel<D, TQ, TKV, 2>, a, p, s);
    return launch_kernel<D, TQ, 16>(paged_attn_kernel<D, TQ, TKV, 1>, a, p, s);
  }
}
template <class TQ, class TKV>
hipError_t launch(const PagedAttn &a, const Plan &p, hipStream_t s) {
  return a.pages.D == 64 ? launch_d<64, TQ, TKV>(a, p, s) : launch_d<128, TQ, TKV>(a, p, s);
}

}  // namespace

// (blocks that share keys are no more than fill the card)
bool paged_attn_fits(const PagedAttn &a) { return a.tokens == 0 || 256ll * make_plan(a, 1).blocks * a.pages.Hk <= kMaxLaunch; }

size_t paged_attn_ws(const PagedAttn &a, int n_cu) {
  const Plan p = make_plan(a, n_cu);
  return p.parts == 0 ? 0 : part_rows(a, p) * (a.pages.D + 2) + 2 * (size_t)a.batch;
}

hipError_t paged_attn(const PagedAttn &a, int n_cu, hipStream_t s) {
  if (a.batch <= 0 || a.tokens <= 0) return hipSuccess;
  const Plan p = make_plan(a, n_cu);
  if (p.parts > 0 && !a.part) return hipErrorInvalidValue;
  const int kv = a.pages.type;
  if (a.type == kOpF32) {
    if (kv == kOpF32) return launch<F32, F32>(a, p, s);
    if (kv == kOpBf16) return launch<F32, Bf16>(a, p, s);
    if (kv == kOpI4) return launch<F32, I4>(a, p, s);
  } else if (a.type == kOpBf16) {
    if (kv == kOpBf16) return launch<Bf16, Bf16>(a, p, s);
    if (kv == kOpI4) return launch<Bf16, I4>(a, p, s);
  } else if (a.type == kOpF16) {
    if (kv == kOpF16) return launch<F16, F16>(a, p, s);
    if (kv == kOpI4) return launch<F16, I4>(a, p, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace itts
