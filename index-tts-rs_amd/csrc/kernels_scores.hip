// Scores of rows of logits x [rows][vocab]: with m the row's maximum, c the number of tokens at m
// and s the sum of exp(x - m) over the others,
//   log p(t) = x_t - m - log(c + s),   entropy = log(c + s) - sum (x - m) exp(x - m) / (c + s).
// Keeping s apart from c makes log(c + s) = log1p(s + (c - 1)) where one token has nearly all the
// probability, so that small entropies and log-probabilities near 0 keep their relative accuracy.
// Alternatives are ordered by (logit, lowest token first); NaN counts as -inf there.
//
// One pass over the logits: a block holds 8 16-byte pieces a thread of its row in registers (rows that
// are longer go on piece by piece), takes each thread's maximum, then its sums.  The same registers
// give the alternatives: any n of the row's elements bound the n-th largest from below, so the
// threads' maxima give a bound that few elements pass; those go to a list in LDS and are ranked
// against each other.  Where many pass (masks of one low value, ties, rising rows) the n-th value is found first:
// 64 rows of 8,194 with all but five at the type's lowest value, 64 alternatives, 15 us a call (12 without a
// mask); n rounds over the row took 438.  Rows that are few and long are split over blocks and joined by a second
// kernel.  Vector instructions an element, as counted: 23 where a block holds its row at once, 19 in longer rows,
// one of them the exponential; memory alone would take half to three quarters of the time.  Waves of short rows wait
// 40% of their cycles for data or barriers and 39% for an issue slot, those of long rows 56% and 15%.  2,188 fp32
// rows of 8,194 with 5 alternatives 19 us (72 MB), 1,000 bf16 rows of 60,510 with 20 50 us (121 MB); one row of
// 8,194 6.2 us.
#include <algorithm>

#include "kernels.h"

namespace itts {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kPieces = 8;       // 16-byte pieces a thread holds
constexpr int kList = 1024;      // room for elements that pass the bound
constexpr int kRank = 256;       // most of them that are ranked against each other
constexpr int kMaxSplits = 16;
static_assert(kMaxSplits * kScoresMaxTop <= kList, "the joined lists fit");
constexpr float kLog2e = 1.4426950408889634f;

template <int TYPE>
constexpr uint32_t kStep = TYPE == kOpF32 ? 1u : TYPE == kOpBf16 ? 1u << 16 : 1u << 13;  // between neighbours, as `order`s
template <int TYPE>
constexpr int kPer = TYPE == kOpF32 ? 4 : 8;  // elements of a 16-byte piece

template <int TYPE>
__device__ __forceinline__ float logit(const void *row, int i) {
  if constexpr (TYPE == kOpF32) return static_cast<const float *>(row)[i];
  else if constexpr (TYPE == kOpBf16) return bf16_bits_to_float(static_cast<const uint16_t *>(row)[i]);
  else return half_bits_to_float(static_cast<const uint16_t *>(row)[i]);
}
template <int TYPE>
__device__ __forceinline__ float element(const uint4 &v, int e) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  if constexpr (TYPE == kOpF32) return __uint_as_float(w[e]);
  else if constexpr (TYPE == kOpBf16) return e % 2 ? __uint_as_float(w[e / 2] & 0xffff0000u) : __uint_as_float(w[e / 2] << 16);
  else return half_bits_to_float(e % 2 ? w[e / 2] >> 16 : w[e / 2] & 0xffffu);
}

// The piece as a new value: what was unpacked from it before is not kept in registers for later.
// Nor does the compiler start on the next piece before this one is done: it would hold both.
__device__ __forceinline__ void again(uint4 &v) {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" : "+v"(v.x), "+v"(v.y), "+v"(v.z), "+v"(v.w));
}

// Floats in order as integers (-inf and NaN alike; -0 as 0), and back.
__device__ __forceinline__ uint32_t order(float x) {
  const uint32_t u = __float_as_uint(fmaxf(x, -INFINITY) + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unorder(uint32_t u) {
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
constexpr uint32_t kOrderNone = 0x007fffffu;  // order(-inf)
// (value, token) as one number, larger for what comes first; 0 is below every token's.
__device__ __forceinline__ uint64_t rank_key(float x, int token) { return (uint64_t)order(x) << 32 | (uint32_t)~token; }
__device__ __forceinline__ int key_token(uint64_t k) { return (int)~(uint32_t)k; }
__device__ __forceinline__ float key_value(uint64_t k) { return unorder((uint32_t)(k >> 32)); }

// Maximum, tokens at it, sums over the others of p = exp(x - m) and p (x - m).  m = -inf: none.
struct Stats {
  float m, c, s, d;
  // what these sums are above a maximum `top` >= m (-inf: nothing was summed, but for a NaN in s)
  __device__ Stats under(float top) const {
    if (m == top || m == -INFINITY) return Stats{top, m == top && m != -INFINITY ? c : 0.0f, s, m == top ? d : 0.0f};
    const float by = m - top, f = __builtin_amdgcn_exp2f(by * kLog2e), w = c + s;
    return Stats{top, 0.0f, f * w, f == 0.0f ? 0.0f : f * (d + by * w)};
  }
  __device__ void join(const Stats &o) {
    const float top = fmaxf(m, o.m);
    const Stats x = under(top), y = o.under(top);
    *this = Stats{top, x.c + y.c, x.s + y.s, x.d + y.d};
  }
};

__device__ __forceinline__ float wave_sum_f(float v) { return wave64_sum_dpp(v); }

// A wave's statistics from its threads', to LDS, and the block's from those.
__device__ __forceinline__ void put_stats(const Stats &t, float (*red)[4]) {
  const float m = wave64_max_dpp(t.m);
  const Stats top = t.under(m);
  const Stats w{m, wave_sum_f(top.c), wave_sum_f(top.s), wave_sum_f(top.d)};
  if ((threadIdx.x & 63) == 0) {
    float *r = red[threadIdx.x >> 6];
    r[0] = w.m, r[1] = w.c, r[2] = w.s, r[3] = w.d;
  }
}
__device__ __forceinline__ Stats get_stats(const float (*red)[4]) {
  Stats o{red[0][0], red[0][1], red[0][2], red[0][3]};
#pragma unroll
  for (int i = 1; i < kWaves; i++) o.join(Stats{red[i][0], red[i][1], red[i][2], red[i][3]});
  return o;
}

// log-probabilities and entropy of a row with statistics t.
struct Row {
  float m, lz;
  bool none;
  float entropy;
  __device__ explicit Row(const Stats &t) {
    none = t.m == -INFINITY && t.s == 0.0f;  // every token is masked: probability 0 for all
    lz = t.m == INFINITY ? NAN : log1pf(t.s + (t.c - 1.0f));
    if (t.m == -INFINITY) lz = NAN;  // NaN and -inf alone
    m = t.m;
    entropy = none ? 0.0f : lz - t.d / (t.c + t.s);
  }
  __device__ float log_prob(float x) const { return none ? -INFINITY : (x - m) - lz; }
};

// The largest 16-bit prefix that at least n of a wave's values reach (0: none).
__device__ __forceinline__ uint32_t reached(uint32_t v, int n) {
  uint32_t p = 0;
#pragma unroll
  for (uint32_t bit = 1u << 31; bit >= 1u << 16; bit >>= 1)
    if (__popcll(__ballot(v >= (p | bit))) >= n) p |= bit;
  return p;
}

struct Select {
  uint64_t list[kList + kScoresMaxTop];
  uint64_t top[kScoresMaxTop];
  uint32_t bound[kWaves];
  int hot[2][kWaves], reach[2][kWaves];
  int count;
};

// The n first of list[0 .. have), in order, to top (0 past have).  All threads.
__device__ inline void rank_list(Select &sel, int have, int n) {
  for (int i = threadIdx.x; i < have; i += kThreads) {
    const uint64_t k = sel.list[i];
    int r = 0;
    for (int j = 0; j < have; j++) r += sel.list[j] > k;
    if (r < n) sel.top[r] = k;
  }
  for (int i = threadIdx.x; i < n; i += kThreads)
    if (i >= have) sel.top[i] = 0;
  __syncthreads();
}

// Fills a list that the row's numbers leave short: tokens of -inf and NaN, the lowest first.  Wave 0.
template <int TYPE>
__device__ inline void fill_masked(const void *x, int vocab, uint64_t *top, int n) {
  const int lane = threadIdx.x & 63;
  int have = 0;
  while (have < n && top[have]) have++;
  for (int i0 = 0; i0 < vocab && have < n; i0 += 64) {
    const bool masked = i0 + lane < vocab && !(logit<TYPE>(x, min(i0 + lane, vocab - 1)) > -INFINITY);
    const uint64_t b = __ballot(masked);
    const int at = have + __popcll(b & ((1ull << lane) - 1));
    if (masked && at < n) top[at] = rank_key(-INFINITY, i0 + lane);
    have += __popcll(b);
  }
}

// Wave 0.
template <int TYPE>
__device__ inline void write_row(const TokenScores &a, int r, const void *x, const Row &row, Select &sel) {
  if (threadIdx.x == 0 && a.entropy) a.entropy[r] = row.entropy;
  if (a.top) {
    if (!sel.top[a.top - 1]) fill_masked<TYPE>(x, a.vocab, sel.top, a.top);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (int k = threadIdx.x; k < a.top; k += 64) {
      const uint64_t key = sel.top[k];
      a.top_tokens[(int64_t)r * a.top + k] = key_token(key);
      // (from the logit itself: the order does not tell NaN from -inf)
      a.top_log_probs[(int64_t)r * a.top + k] = row.log_prob(key >> 32 == kOrderNone ? logit<TYPE>(x, key_token(key)) : key_value(key));
    }
  }
}

// The splits' results: statistics [rows][S], then ordered lists [rows][S][top].
__host__ __device__ inline size_t list_offset(int rows, int S) { return sizeof(Stats) * (size_t)rows * S; }

// LONG: a block's tokens are more than its threads hold, and the next ones are on their way while these
// are counted: 1,000 rows of 60,510 50 us, without 54 (also with half the registers and more blocks a unit), and 49 to 50
// since later turns look for tokens above the n-th so far alone.
template <int TYPE, bool LONG>
__global__ __launch_bounds__(kThreads, LONG ? 4 : 6) void token_scores_kernel(TokenScores a, int S) {
  __shared__ float red[kWaves][4];
  __shared__ Select sel;
  constexpr int P = kPer<TYPE>, kBytes = 16 / P;
  const int r = blockIdx.x / S, split = blockIdx.x % S, t = threadIdx.x;
  const char *x = static_cast<const char *>(a.x) + r * a.x_row * kBytes;
  const int n = a.top;
  // this block's tokens: i0 .. i1, in whole pieces from i0 (wherever in memory that is: a thread's share
  // does not depend on it, nor do the results) and the rest
  const int per = ((a.vocab + S - 1) / S + P - 1) / P * P;
  const int i0 = min(split * per, a.vocab), i1 = min(i0 + per, a.vocab);
  const int pieces = (i1 - i0) / P, rest = i1 - i0 - pieces * P;
  const char *body = x + (int64_t)i0 * kBytes;
  // a given token's logit, early
  const int64_t tok_at = r * a.tok_row;
  const int tok = S == 1 && t < min(a.given, 64) ? a.tokens[tok_at + t] : -1;
  const float tok_x = tok >= 0 && tok < a.vocab ? logit<TYPE>(x, tok) : 0.0f;

  Stats st{-INFINITY, 0.0f, 0.0f, 0.0f};
  int found = 0;  // entries of the list that the last turn left
  if (n > 0) {
    if (t < n) sel.top[t] = 0;
    if (t == 0) sel.count = 0;
  }
  uint4 v[kPieces];
  auto load = [&](uint4 (&to)[kPieces], int base) {
    const uint32_t none = TYPE == kOpF32 ? 0xff800000u : TYPE == kOpBf16 ? 0xff80ff80u : 0xfc00fc00u;  // -inf
#pragma unroll
    for (int k = 0; k < kPieces; k++) {
      const int at = base + k * kThreads + t;
      to[k] = make_uint4(none, none, none, none);
      if (at < pieces) __builtin_memcpy(&to[k], body + (int64_t)at * 16, 16);  // (at any element's alignment)
    }
  };
  load(v, 0);
  for (int base = 0; base == 0 || base < pieces; base += kThreads * kPieces) {
    uint4 coming[kPieces];
    if constexpr (LONG) load(coming, base + kThreads * kPieces);
    const int odd = i1 - rest + t;  // one element a thread of the rest, in the first round
    const bool has_odd = base == 0 && t < rest;
    const float odd_x = has_odd ? logit<TYPE>(x, odd) : -INFINITY;

    const int filled = (pieces - base + kThreads - 1) / kThreads;  // pieces of the first thread, and of others at most
    float gm[kPieces], mx = odd_x;
#pragma unroll
    for (int k = 0; k < kPieces; k++) {
      gm[k] = -INFINITY;
      if (k >= filled) continue;
      again(v[k]);
      gm[k] = element<TYPE>(v[k], 0);
#pragma unroll
      for (int e = 1; e < P; e++) gm[k] = fmaxf(gm[k], element<TYPE>(v[k], e));
      mx = fmaxf(mx, gm[k]);
    }
    Stats u{fmaxf(mx, -INFINITY), 0.0f, 0.0f, 0.0f};
    const float ms = u.m == -INFINITY ? 0.0f : u.m;
    int at_top = 0;
    auto add = [&](float y) {
      // (at the maximum: as a token of probability 0, and counted)
      const float d = y == ms ? -INFINITY : y - ms, p = __builtin_amdgcn_exp2f(d * kLog2e);
      at_top += y == ms;
      u.s += p;
      u.d += p * fmaxf(d, -3e38f);
    };
#pragma unroll
    for (int k = 0; k < kPieces; k++) {
      if (k >= filled) break;
      again(v[k]);
#pragma unroll
      for (int e = 0; e < P; e++) add(element<TYPE>(v[k], e));
    }
    if (has_odd) add(odd_x);
    u.c = (float)at_top;
    if constexpr (LONG) {
      st.join(u);
    } else {
      put_stats(u, red);
    }

    uint32_t bound = kOrderNone + 1;
    const uint32_t own = u.m > -INFINITY ? order(u.m) : 0;
    bool any = n > 0, narrow = any;
    if constexpr (LONG) {
      // A token has to come before the n-th so far: to be larger, or as large where that one is of the row's
      // rest, whose tokens are the last.  Where few threads have one, that is bound enough.
      if (any) {
        if (base > 0) {
          const uint64_t worst = sel.top[n - 1];  // (0 before n are found)
          bound = max(bound, (uint32_t)(worst >> 32) + (key_token(worst) < i1 - rest ? 1u : 0u));
        }
        int *hot = sel.hot[base / (kThreads * kPieces) & 1];
        const uint64_t here = __ballot(own >= bound);
        if ((t & 63) == 0) hot[t >> 6] = __popcll(here);
        __syncthreads();
        int threads = 0;
#pragma unroll
        for (int w = 0; w < kWaves; w++) threads += hot[w];
        any = threads > 0, narrow = threads > 64;
      }
    }
    if (any) {
      // (-inf has no part in this: a row's last places go to masked tokens at the end)
      // A bound for the n-th largest: an equal share of n of every full wave's threads reach it.  (Without a
      // full wave the list has room for all.)
      const int full = min(pieces - base, kThreads) / 64;
      if (narrow && full > 0) {
        const uint32_t share = reached(own, (n + full - 1) / full);
        if ((t & 63) == 0) sel.bound[t >> 6] = share;
        __syncthreads();
        uint32_t low = ~0u;
#pragma unroll
        for (int w = 0; w < kWaves; w++) low = w < full ? min(low, sel.bound[w]) : low;
        if (low == 0) {  // masks leave a wave fewer: n threads of one wave reach it
          const uint32_t all = reached(own, n);
          __syncthreads();
          if ((t & 63) == 0) sel.bound[t >> 6] = all;
          __syncthreads();
#pragma unroll
          for (int w = 0; w < kWaves; w++) low = max(low, sel.bound[w]);
        }
        bound = max(bound, low);
      }
      auto offer = [&](float y, int token, float least) {
        if (!(y >= least)) return;
        const int at = atomicAdd(&sel.count, 1);
        if (at < kList) sel.list[at] = rank_key(y, token);
      };
      const float first = unorder(bound);
#pragma unroll
      for (int k = 0; k < kPieces; k++) {
        if (!(gm[k] >= first)) continue;
        again(v[k]);
#pragma unroll
        for (int e = 0; e < P; e++) offer(element<TYPE>(v[k], e), i0 + (base + k * kThreads + t) * P + e, first);
      }
      if (has_odd) offer(odd_x, odd, first);
      __syncthreads();
      int count = sel.count;  // (with the `found` ones from before)
      bool ties = false;
      if (count - found > kRank) {
        // Ties by the hundred, or the largest all in a few threads: the n-th value itself, bit by bit from the
        // top, until no more than can be ranked reach it; if that never is so, what is above it.  (From memory
        // again: this is rare, and the registers are the others'.)
        auto each = [&](auto &&f) {
#pragma unroll 1
          for (int at = base + t; at < min(base + kThreads * kPieces, pieces); at += kThreads) {
            uint4 w;
            __builtin_memcpy(&w, body + (int64_t)at * 16, 16);
#pragma unroll
            for (int e = 0; e < P; e++) f(element<TYPE>(w, e), i0 + at * P + e);
          }
          if (has_odd) f(odd_x, odd);
        };
        int buf = 0;
        auto reaching = [&](uint32_t from) {
          const float least = unorder(from);
          int c = 0;
          each([&](float y, int) { c += y >= least; });
          const float sum = wave_sum_f((float)c);
          if ((t & 63) == 0) sel.reach[buf][t >> 6] = (int)sum;
          __syncthreads();
          int all = 0;
#pragma unroll
          for (int w = 0; w < kWaves; w++) all += sel.reach[buf][w];
          buf ^= 1;
          return all;
        };
        // The least of the threads' largest is that value where one stands in nearly every place (a mask's).
        const float low = -wave64_max_dpp(own >= bound ? -u.m : -INFINITY);
        if ((t & 63) == 0) sel.bound[t >> 6] = order(low);
        __syncthreads();
        uint32_t nth = ~0u;
#pragma unroll
        for (int w = 0; w < kWaves; w++) nth = min(nth, sel.bound[w]);
        int reach = reaching(nth);
        if (reach >= n) bound = nth;
        if (reach < n || (reach > kRank && reaching(nth + kStep<TYPE>) >= n)) {
          nth = 0, reach = count - found;
          for (uint32_t bit = 1u << 31; bit >= kStep<TYPE> && reach > kRank; bit >>= 1) {
            const uint32_t to = nth | bit;
            if (to > bound) {
              const int all = reaching(to);
              if (all < n) continue;
              reach = all;
            }
            nth = to;
          }
        }
        ties = reach > kRank;
        bound = ties ? nth + kStep<TYPE> : max(nth, bound);
        __syncthreads();  // (the list and its length are read)
        if (t == 0) sel.count = found;
        __syncthreads();
        const float least = unorder(bound);
        each([&](float y, int token) { offer(y, token, least); });
        __syncthreads();
        count = sel.count;
      }
      if (ties) {  // fewer than n are above that value: its lowest tokens follow
        __syncthreads();
        if (t < 64) {
          int have = count;
          const int body_end = i1 - rest;
          for (int part = 0; part < (base == 0 ? 2 : 1); part++) {  // (the first turn has the row's rest too)
            const int from = part == 0 ? i0 + base * P : body_end;
            const int to = part == 0 ? min(from + kThreads * kPieces * P, body_end) : i1;
            for (int at = from; at < to && have < found + n; at += 64) {
              const uint32_t o = order(logit<TYPE>(x, min(at + t, to - 1)));
              const bool tie = at + t < to && o < bound && bound - o <= kStep<TYPE>;
              const uint64_t b = __ballot(tie);
              const int place = have + __popcll(b & ((1ull << t) - 1));
              if (tie && place < found + n) sel.list[place] = rank_key(unorder(o), at + t);
              have = min(have + (int)__popcll(b), found + n);
            }
          }
          if (t == 0) sel.count = have;
        }
        __syncthreads();
        count = sel.count;
      }
      if (count > 0) {
        rank_list(sel, count, n);
        if constexpr (LONG) {
          found = min(count, n);
          if (t < n) sel.list[t] = sel.top[t];
          if (t == 0) sel.count = found;
        }
      }
    }
    if constexpr (!LONG) break;
#pragma unroll
    for (int k = 0; k < kPieces; k++) v[k] = coming[k];
  }
  if constexpr (LONG) put_stats(st, red);
  __syncthreads();
  if (t >= 64) return;
  st = get_stats(red);

  if (S == 1) {
    const Row row(st);
    for (int i = t; i < a.given; i += 64) {
      const int k = i == t ? tok : a.tokens[tok_at + i];
      const bool in = k >= 0 && k < a.vocab;
      const float y = i == t ? tok_x : in ? logit<TYPE>(x, k) : 0.0f;
      a.log_probs[(int64_t)r * a.given + i] = k == -1 ? 0.0f : in ? row.log_prob(y) : NAN;
    }
    write_row<TYPE>(a, r, x, row, sel);
  } else {
    if (t == 0) static_cast<Stats *>(a.ws)[(int64_t)r * S + split] = st;
    uint64_t *lists = reinterpret_cast<uint64_t *>(static_cast<char *>(a.ws) + list_offset(a.rows, S));
    if (t < n) lists[((int64_t)r * S + split) * n + t] = sel.top[t];
  }
}

// Joins a row's splits.  Lists are ordered: the first ceil(n / S) of each together, or n of one, bound
// the n-th largest from below.
template <int TYPE>
__global__ __launch_bounds__(kThreads) void scores_join_kernel(TokenScores a, int S) {
  __shared__ Select sel;
  __shared__ uint64_t keys[kMaxSplits * kScoresMaxTop];
  const int r = blockIdx.x, t = threadIdx.x, n = a.top;
  const char *x = static_cast<const char *>(a.x) + r * a.x_row * (16 / kPer<TYPE>);
  const Stats *parts = static_cast<const Stats *>(a.ws) + (int64_t)r * S;
  const uint64_t *lists = reinterpret_cast<const uint64_t *>(static_cast<const char *>(a.ws) + list_offset(a.rows, S)) + (int64_t)r * S * n;
  for (int i = t; i < S * n; i += kThreads) keys[i] = lists[i];
  if (n > 0) {
    if (t == 0) sel.count = 0;
    __syncthreads();
    uint64_t all = 0, share = ~0ull;
    const int q = (n + S - 1) / S - 1;
    for (int s = 0; s < S; s++) all = max(all, keys[s * n + n - 1]), share = min(share, keys[s * n + q]);
    const uint64_t least = max(max(all, share), (uint64_t)1);
    for (int i = t; i < S * n; i += kThreads) {
      if (keys[i] < least) continue;
      sel.list[atomicAdd(&sel.count, 1)] = keys[i];
    }
    __syncthreads();
    rank_list(sel, sel.count, n);
  }
  if (t >= 64) return;
  Stats st = parts[0];
  for (int s = 1; s < S; s++) st.join(parts[s]);
  const Row row(st);
  for (int i = t; i < a.given; i += 64) {
    const int k = a.tokens[r * a.tok_row + i];
    const bool in = k >= 0 && k < a.vocab;
    a.log_probs[(int64_t)r * a.given + i] = k == -1 ? 0.0f : in ? row.log_prob(logit<TYPE>(x, k)) : NAN;
  }
  write_row<TYPE>(a, r, x, row, sel);
}

// Blocks of a row: so many that each holds its tokens at once, up to 16 (the joining takes longer with
// every one: an fp32 row of 131,000 15.5 us with 16, 18 with 8, 21 with 32; 64 rows with 64 alternatives 27, 37, 39).
// Where that is more than eight blocks a compute unit: three, or one (300 rows of 131,000 40 us with 3, 44 with
// 6, 54 with 1; 700 rows of 33,000 with 20 alternatives 41 with 2, 35 with 1).  A second turn costs less than a second
// launch while few alternatives are asked for: a row of 12,000 with 10 11.5 and 10.2 us, a call 10.5 and 12.3;
// 64 rows with 64 23 and 16 us.
int splits(const TokenScores &a, int n_cu) {
  const int pieces = a.vocab / (a.type == kOpF32 ? 4 : 8), turn = kThreads * kPieces;
  if (pieces <= (a.top <= 16 ? 2 : 1) * turn) return 1;
  const int want = std::min((pieces + turn - 1) / turn, kMaxSplits), room = 8 * n_cu / a.rows;
  return want <= room ? want : room >= 3 ? 3 : 1;
}

template <int TYPE>
hipError_t launch(const TokenScores &a, int S, hipStream_t s) {
  const int pieces = S == 1 ? a.vocab / kPer<TYPE> : ((a.vocab + S - 1) / S + kPer<TYPE> - 1) / kPer<TYPE>;  // of a block, at most
  if (pieces > kThreads * kPieces) hipLaunchKernelGGL((token_scores_kernel<TYPE, true>), dim3((unsigned)a.rows * S), dim3(kThreads), 0, s, a, S);
  else hipLaunchKernelGGL((token_scores_kernel<TYPE, false>), dim3((unsigned)a.rows * S), dim3(kThreads), 0, s, a, S);
  if (hipError_t e = hipGetLastError(); e != hipSuccess || S == 1) return e;
  hipLaunchKernelGGL(scores_join_kernel<TYPE>, dim3(a.rows), dim3(kThreads), 0, s, a, S);
  return hipGetLastError();
}

}  // namespace

size_t token_scores_ws(const TokenScores &a, int n_cu) {
  const int S = splits(a, n_cu);
  return S == 1 ? 0 : list_offset(a.rows, S) + sizeof(uint64_t) * (size_t)a.rows * S * a.top;
}

hipError_t token_scores(const TokenScores &a, int n_cu, hipStream_t s) {
  if (a.rows <= 0) return hipSuccess;
  if (a.top > kScoresMaxTop || a.top > a.vocab) return hipErrorInvalidValue;
  const int S = splits(a, n_cu);
  if (S > 1 && !a.ws) return hipErrorInvalidValue;
  switch (a.type) {
    case kOpF32: return launch<kOpF32>(a, S, s);
    case kOpBf16: return launch<kOpBf16>(a, S, s);
    case kOpF16: return launch<kOpF16>(a, S, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace itts
