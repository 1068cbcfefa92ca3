// Decoding with drafted trees: attention of every node of a tree of tokens over its sequence's
// cached keys and values and its own ancestors, and the accepted nodes' rows moved up in the cache.
//
// Attention.  Node i of sequence b sees the rows t < lengths[b] and the rows lengths[b] + j of the
// nodes j on its path to the root, itself among them:
//   o_i = sum_t p_it v_t / sum_t p_it,   p_it = exp(scale q_i . k_t - m_i).
// The M = n H / Hk query rows that share a key head are the columns of the products (attn_tiles.h).
#include <algorithm>
#include <cmath>
#include <numeric>
#include <type_traits>

#include "attn_tiles.h"
#include "kernels.h"

namespace itts {
namespace {

// The tree of one sequence: every node's ancestors (itself among them) as bits, none for a slot
// that is unused or hangs below one, and the number of slots up to the last used one.  W words of
// 64 nodes.  The parents are followed by doubling: after step k a node knows 2^k of its ancestors.
template <int W>
struct Tree;

// Up to 64 nodes: node i in lane i of every wave, no memory.
template <>
struct Tree<1> {
  uint64_t anc;
  int live;
  struct Shared {};
  __device__ void read(int par, int n, Shared &) {
    const int i = threadIdx.x & 63;
    int up = i < n && par >= -1 && par < i ? par : -2;  // -1: the root is reached; -2: not in the tree
    anc = up != -2 ? 1ull << i : 0;
    while (__ballot(up >= 0)) {
      const int at = max(up, 0);
      const uint64_t a = __shfl((unsigned long long)anc, at, 64);
      const int u = __shfl(up, at, 64);
      if (up >= 0) anc |= a, up = u;
    }
    if (up == -2) anc = 0;
    live = 64 - __clzll(__ballot(anc != 0));
  }
  // node's words, in registers of the lanes that ask
  struct Row {
    uint64_t anc;
    __device__ bool sees(int j) const { return j < 64 && (anc >> (j & 63) & 1); }
    // of the 32 rows from j0 on (counted from node 0's; negative: the sequence's) those that are seen
    __device__ uint32_t tile(int j0) const {
      if (j0 >= 0) return j0 < 64 ? (uint32_t)(anc >> (j0 & 63)) : 0;
      return j0 > -32 ? (uint32_t)(anc << -j0) | ((1u << -j0) - 1) : ~0u;
    }
    __device__ bool any() const { return anc != 0; }
  };
  __device__ Row row(int node, const Shared &) const { return Row{__shfl((unsigned long long)anc, node, 64)}; }
};

template <>
struct Tree<4> {
  int live;
  struct Shared {
    uint64_t anc[kTreeMaxNodes][4];
    int up[kTreeMaxNodes];
    int live;
  };
  __device__ void read(int par, int n, Shared &t) {
    const int i = threadIdx.x;
    // (a thread for each node: blocks have four waves at least)
    if (i == 0) t.live = 0;
    if (i < n) {
      t.up[i] = par >= -1 && par < i ? par : -2;
#pragma unroll
      for (int w = 0; w < 4; w++) t.anc[i][w] = w == i >> 6 ? 1ull << (i & 63) : 0;
    }
    __syncthreads();
    for (int s = 1; s < n; s *= 2) {
      int up = -2;
      uint64_t a[4] = {};
      if (i < n) {
        up = t.up[i];
#pragma unroll
        for (int w = 0; w < 4; w++) a[w] = t.anc[i][w] | (up >= 0 ? t.anc[up][w] : 0);
        if (up >= 0) up = t.up[up];
      }
      __syncthreads();
      if (i < n) {
        t.up[i] = up;
#pragma unroll
        for (int w = 0; w < 4; w++) t.anc[i][w] = a[w];
      }
      __syncthreads();
    }
    if (i < n) {
      if (t.up[i] == -2) {
#pragma unroll
        for (int w = 0; w < 4; w++) t.anc[i][w] = 0;
      } else {
        atomicMax(&t.live, i + 1);
      }
    }
    __syncthreads();
    live = __builtin_amdgcn_readfirstlane(t.live);
  }
  struct Row {
    const uint64_t *anc;
    __device__ bool sees(int j) const { return j < kTreeMaxNodes && (anc[j >> 6] >> (j & 63) & 1); }
    __device__ uint32_t tile(int j0) const {
      if (j0 >= kTreeMaxNodes) return 0;
      if (j0 >= 0) {
        const int w = j0 >> 6, s = j0 & 63;
        return (uint32_t)(anc[w] >> s | (s > 0 && w < 3 ? anc[w + 1] << (64 - s) : 0));
      }
      return j0 > -32 ? (uint32_t)(anc[0] << -j0) | ((1u << -j0) - 1) : ~0u;
    }
    __device__ bool any() const { return (anc[0] | anc[1] | anc[2] | anc[3]) != 0; }
  };
  __device__ Row row(int node, const Shared &t) const { return Row{t.anc[node]}; }
};

// A launch: the query rows of a key head (row r being head r % group of node r / group), and what
// shares the keys: one block a sequence, key head and row tile (parts 0), or `parts` blocks for all
// sequences of a key head and row tile, with results of their own (o [Hk][M][parts][D], then (max,
// sum) [Hk][M][parts], then (first block, blocks) [batch]) that a second kernel joins.
struct Args {
  TreeAttn a;
  int parts, M, group;
  uint32_t group_mul;  // 2^32 / group, rounded up: exact for rows < 2^32 / group
  int unit, least;     // a block's rows are at least `least` times 2^unit
  float2 *ml;
  int2 *dealt;
  __device__ int node(int row) const { return group == 1 ? row : __umulhi((uint32_t)row, group_mul); }
};

// Query rows row0 + 16 t + c (past the last one: that one), elements 8 g .., to the wave's registers, and their nodes.
template <int D, class TQ, class Wave, int RT>
__device__ __forceinline__ void load_rows(const Args &p, int b, int hk, int row0, int c, int g, Wave &rows, int (&node)[RT]) {
  const TreeAttn &a = p.a;
  const char *at[RT];
#pragma unroll
  for (int t = 0; t < RT; t++) {
    const int row = min(row0 + 16 * t + c, p.M - 1);
    node[t] = p.node(row);
    const int64_t head = hk * p.group + (row - node[t] * p.group);
    at[t] = static_cast<const char *>(a.q) + (b * a.q_b + node[t] * a.q_n + head * a.q_h + 8 * g) * TQ::kBytes;
  }
  rows.load(at, a.scale);
}

// What block `index` of `parts` has to do: rows [first, end) of sequence b, whose rows are shared by
// n blocks (0: nothing is left for this one).  Every block gets the same number of rows, whatever
// the sequences' lengths and however long the cache could become: the smallest one with which `parts`
// blocks are enough (within a few percent).  Every wave finds it by itself from the lengths, a lane a
// sequence.  12 x 64 nodes over 1,000 .. 8,191 rows, 8 key heads: with the rows of max_seq shared equally
// 115 us, with these 107 (one plane of probabilities, 131 with two).  A block still waits for the longest
// one, a fifth above the mean there; runs that go on into the next sequence made that kernel 7 us faster and the one
// for few rows 1 to 10 slower (registers kept over the turns, a second start), and are not taken.
struct Share {
  int b, n, first, end, index, from;
};
__device__ __forceinline__ Share share_of(const Args &p) {
  const TreeAttn &a = p.a;
  const int index = blockIdx.x, lane = threadIdx.x & 63;
  if (p.parts == 0) return Share{index, 1, 0, a.max_seq, 0, 0};
  auto units = [&](int b) -> uint32_t {
    if (b >= a.batch) return 0;
    const int len = a.lengths[b];
    return len < 0 || len > a.max_seq ? 1 : (uint32_t)((min(len + a.n, a.max_seq) - 1) >> p.unit) + 1;
  };
  float total = 0.0f, longest = 0.0f;
  for (int b = lane; b < a.batch + lane; b += 64) {
    const float u = units(b);
    total += u, longest = fmaxf(longest, u);
  }
  total = wave_sum(total), longest = wave_max(longest);
  // (64 blocks of a sequence at most: the joining kernel's lanes)
  uint32_t size = (uint32_t)fmaxf(ceilf(fmaxf(total / p.parts, longest / 64)), (float)p.least);
  for (int i = 0; i < 16; i++) {
    float blocks = 0.0f;
    for (int b = lane; b < a.batch + lane; b += 64) blocks += (units(b) + size - 1) / size;
    blocks = wave_sum(blocks);
    if (blocks <= p.parts) break;
    size = i < 14 ? max(size + 1, (uint32_t)ceilf(size * (blocks / p.parts))) : (uint32_t)longest + 1;  // (parts >= batch)
  }
  size = __builtin_amdgcn_readfirstlane(size);
  Share share{0, 0, 0, 0, index, 0};
  int before = 0;
  for (int b0 = 0; b0 < a.batch && share.n == 0; b0 += 64) {
    const int own = (units(b0 + lane) + size - 1) / size;
    int to = own;
#pragma unroll
    for (int step = 1; step < 64; step *= 2) {
      const int up = __shfl_up(to, step, 64);
      if (lane >= step) to += up;
    }
    if (const uint64_t at = __ballot(index >= before + to - own && index < before + to); at != 0) {
      const int src = __builtin_ctzll(at);
      share.b = b0 + src, share.n = __builtin_amdgcn_readlane(own, src);
      share.from = before + __builtin_amdgcn_readlane(to, src) - share.n;
    }
    before += __builtin_amdgcn_readlane(to, 63);
  }
  share.first = (int)((uint32_t)(index - share.from) * size << p.unit), share.end = share.first + (int)(size << p.unit);
  return share;
}

// A wave's keys and values of one tile: key rows 16 h + c, in runs of 8 elements 32 j + 8 g, and value
// rows 16 h + 4 g + r, elements D / 16 c ...  Rows lie at the same offsets from every tile's first row
// (32 bits, kept), so that a tile's loads need a new base alone, in scalar registers.
template <int D, class T>
struct TileRegs {
  static constexpr int kK = 8 * T::kBytes / 4, kV = D / 16 * T::kBytes / 4;  // dwords of a run
  uint32_t k[2][D / 32][kK];
  uint32_t v[8][kV];
  uint32_t k_at[2], v_at[8];
  // offsets of a tile whose rows past row `last` are read as that one
  __device__ __forceinline__ void place(uint32_t k_step, uint32_t v_step, int last, int c, int g) {
#pragma unroll
    for (int h = 0; h < 2; h++) k_at[h] = min(16 * h + c, last) * k_step + 8 * g * T::kBytes;
#pragma unroll
    for (int i = 0; i < 8; i++) v_at[i] = min(16 * (i >> 2) + 4 * g + (i & 3), last) * v_step + D / 16 * c * T::kBytes;
  }
  // (the offsets pass as new values, or they are kept widened to 64 bits)
  __device__ __forceinline__ void load_k(const char *tile) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      asm volatile("" : "+v"(k_at[h]));
#pragma unroll
      for (int j = 0; j < D / 32; j++) load_dwords<kK>(tile + 32 * j * T::kBytes + k_at[h], k[h][j]);
    }
  }
  __device__ __forceinline__ void load_v(const char *tile) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      asm volatile("" : "+v"(v_at[i]));
      load_dwords<kV>(tile + v_at[i], v[i]);
    }
  }
};

// y[0 .. N) += such values of the nodes that a row sees (a positive probability times an infinity or
// NaN is that); at: element y[0]'s place in node 0's row.
template <class T, int N, class Seen>
__device__ inline void odd_values(float *y, const Seen &seen, int live, const char *at, uint32_t step) {
#pragma unroll 1
  for (int j = 0; j < live; j++) {
    if (!seen.sees(j)) continue;
#pragma unroll
    for (int e = 0; e < N; e++) {
      const float v = load1<T>(at + (uint64_t)(uint32_t)j * step + e * T::kBytes);
      if (!(fabsf(v) < INFINITY)) y[e] += v;
    }
  }
}

// Four elements d .. of a row's result to the output, or to the planes (their sum comes back).
template <int D, class TQ>
__device__ __forceinline__ float put_result(const Args &p, int b, int hk, int row, int node, int d, const float *y) {
  const TreeAttn &a = p.a;
  const int head = hk * p.group + (row - node * p.group);
  if constexpr (D == 64 && std::is_same_v<TQ, F32>) {
    if (a.planes.hi) {
      const size_t at = (((size_t)b * a.n + node) * a.H + head) * 64 + d;
      uint32_t h0, l0, h1, l1;
      split_f16x2(y[0], y[1], h0, l0);
      split_f16x2(y[2], y[3], h1, l1);
      *reinterpret_cast<uint2 *>(a.planes.hi + at) = make_uint2(h0, h1);
      *reinterpret_cast<uint2 *>(a.planes.lo + at) = make_uint2(l0, l1);
      return (y[0] + y[1]) + (y[2] + y[3]);
    }
  }
  const int64_t at = b * a.o_b + node * a.o_n + head * a.o_h + d;
  store4<TQ>(static_cast<char *>(a.out) + at * TQ::kBytes, y[0], y[1], y[2], y[3]);
  return 0.0f;
}
// The planes' sum of a row.
template <int D, class TQ>
__device__ __forceinline__ void put_sum(const Args &p, int b, int hk, int row, int node, float sum) {
  if constexpr (D == 64 && std::is_same_v<TQ, F32>)
    p.a.planes.gs[((size_t)b * p.a.n + node) * p.a.H + hk * p.group + (row - node * p.group)] = sum;
}
template <int D, class TQ>
__device__ __forceinline__ bool has_planes(const Args &p) {
  return D == 64 && std::is_same_v<TQ, F32> && p.a.planes.hi;
}

// Four elements d .. of a row's result over this block's keys, to the output or the splits' results.
// What the joining kernel cannot tell by itself goes with the statistics: a row that sees nothing
// has maximum +inf and sum 0, one of a bad sequence sum NaN.
// Returns the sum of what went to the planes.
template <int D, class TQ>
__device__ __forceinline__ float put4(const Args &p, const Share &share, int hk, int row, int node, int d, float *y, float top,
                                      float sum, bool bad, bool any, bool keys) {
  if (share.n == 1) {
    const float inv = 1.0f / sum;
#pragma unroll
    for (int e = 0; e < 4; e++) y[e] = bad ? NAN : any ? y[e] * inv : 0.0f;
    return put_result<D, TQ>(p, share.b, hk, row, node, d, y);
  } else {
    const size_t at = ((size_t)hk * p.M + row) * p.parts + share.index;
    if (keys) *reinterpret_cast<float4 *>(p.a.part + at * D + d) = make_float4(y[0], y[1], y[2], y[3]);
    if (d == 0) p.ml[at] = bad ? make_float2(0.0f, NAN) : any ? make_float2(top, sum) : make_float2(INFINITY, 0.0f);
    return 0.0f;
  }
}

// Few query rows: 4 waves over tiles of keys of their own, straight from memory into registers, one
// tile ahead; joined at the end.  Long caches are bound by memory: 2 x 16 heads, 61 nodes, 40,001 and 65,500
// fp16 rows, 433 MB, 79 us; 32 single tokens, 4 key heads of 128, 513 .. 4,097 bf16 rows, 152 MB, 27.  Short ones
// by the chain from load to result: 8 nodes, 20 heads, 235 rows 6.3 us.  fp32 caches by the fp32
// products, of 4 keys at a time: 33 nodes, 20 heads, 1,734 rows 13.3 us.  fp32 queries over bf16 by the
// three planes' instructions: 8 x 27 nodes, 250 .. 1,400 rows 16.3 us.
template <int D, class TQ, class TKV, int RT, int W>
__global__ __launch_bounds__(256, 2) void tree_attn_kernel(Args p) {
  constexpr int WK = kKeyWaves;
  __shared__ typename Tree<W>::Shared tree_mem;
  __shared__ float so[WK][16 * RT][D + 4];
  __shared__ float sm[WK][16 * RT], sl[WK][16 * RT];
  __shared__ int sodd[WK];
  const TreeAttn &a = p.a;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
  const int hk = blockIdx.y % a.Hk, row0 = blockIdx.y / a.Hk * (16 * RT);
  const Share share = share_of(p);
  if (share.n == 0) return;
  const int b = share.b;
  if (p.parts > 0 && share.first == 0 && blockIdx.y == 0 && threadIdx.x == 0) p.dealt[b] = make_int2(share.from, share.n);

  // Everything that does not wait for something else is loaded first: this wave's first tile too,
  // wherever the length ends.
  const char *kb = static_cast<const char *>(a.k) + (b * a.k_b + hk * a.k_h) * TKV::kBytes;
  const char *vb = static_cast<const char *>(a.v) + (b * a.v_b + hk * a.v_h) * TKV::kBytes;
  const uint32_t k_step = (uint32_t)a.k_r * TKV::kBytes, v_step = (uint32_t)a.v_r * TKV::kBytes;
  constexpr int stride = WK * kTileKeys;
  int key0 = share.first + wave * kTileKeys;
  const int len = a.lengths[b];
  const int par_at = W == 1 ? lane : threadIdx.x;
  const int par = par_at < a.n ? a.parents[b * a.par_b + par_at] : -2;
  TileRegs<D, TKV> x;
  {
    const int first = min(key0, a.max_seq - 1);
    x.place(k_step, v_step, a.max_seq - 1 - first, c, g);
    x.load_k(kb + (uint64_t)(uint32_t)first * k_step);
    x.load_v(vb + (uint64_t)(uint32_t)first * v_step);
  }
  using Wave = Rows<D, TQ, TKV, RT, false>;
  Wave rows;
  int node[RT];
  load_rows<D, TQ>(p, b, hk, row0, c, g, rows, node);
  Tree<W> tree;
  tree.read(par, a.n, tree_mem);
  const int live = tree.live;
  const bool bad = len < 0 || live > a.max_seq || len > a.max_seq - live;
  const int total = bad ? 0 : len + live, end = min(total, share.end);
  typename Tree<W>::Row sees[RT];
#pragma unroll
  for (int t = 0; t < RT; t++) sees[t] = tree.row(node[t], tree_mem);

  uint32_t odd = 0;  // a node's value that is no finite number was taken out
  for (; key0 < end; key0 += stride) {
    floatx4 s[2][RT] = {};
#pragma unroll
    for (int j = 0; j < D / 32; j++) rows.scores(s, j, x.k[0][j], x.k[1][j]);
    // the wave's next tile; past the last one every lane asks for the last row (one line), so that no
    // register is left as it was on some path
    const int next = key0 + stride < end ? key0 + stride : total - 1;
    if (next + kTileKeys > total) x.place(k_step, v_step, total - 1 - next, c, g);
    x.load_k(kb + (uint64_t)(uint32_t)next * k_step);
    const bool edge = key0 + kTileKeys > len;  // holds nodes, or ends past the last row
    uint32_t seen[RT] = {};
    if (edge) {
#pragma unroll
      for (int t = 0; t < RT; t++) seen[t] = sees[t].tile(key0 - len) >> (4 * g);
    }
    rows.limit(s, edge, seen);
    rows.weigh(s);
    if (edge) odd |= take_odd<TKV>(x.v, key0, len, total, g);
    if constexpr (TKV::kBytes == 4) {
      rows.add_wide(s, x.v);
    } else {
      typename Wave::Probs probs;
      rows.pack(s, probs);
      rows.add_rows(probs, x.v);
    }
    x.load_v(vb + (uint64_t)(uint32_t)next * v_step);
  }

  // The waves joined: lane (c, g) holds dims D/4 g .. of row c, in runs of D/16 a register.
  if (const bool any = __ballot(odd != 0) != 0; lane == 0) sodd[wave] = any;
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
  for (int i0 = 0; i0 < 16 * RT * (D / 4); i0 += 64 * WK) {
    const int i = i0 + threadIdx.x;
    const int rr = min(i / (D / 4), 16 * RT - 1), d = i % (D / 4) * 4, row = row0 + rr, i_node = p.node(min(row, p.M - 1));
    const auto seen = tree.row(i_node, tree_mem);
    if (row >= p.M || i >= 16 * RT * (D / 4)) continue;
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
    if (odd_any) odd_values<TKV, 4>(y, seen, live, vb + (uint64_t)(uint32_t)len * v_step + d * TKV::kBytes, v_step);
    float planes = put4<D, TQ>(p, share, hk, row, i_node, d, y, top, sum, bad, seen.any(), share.first < total);
    if (has_planes<D, TQ>(p) && share.n == 1) {  // (a row's D / 4 lanes are neighbours)
#pragma unroll
      for (int step = 1; step < D / 4; step *= 2) planes += __shfl_xor(planes, step, 64);
      if (d == 0) put_sum<D, TQ>(p, b, hk, row, i_node, planes);
    }
  }
}

// Many query rows over 16-bit caches: 4 waves with rows of their own over the same tiles, which the
// block copies to LDS (through registers), so that a tile is read from memory once for 64 RT
// rows.  A tile's scores are formed a tile ahead, so that their products run under the exponentials
// of the one before: keys lie a tile further than values.  In LDS a row's 16-byte pieces lie in the
// order p ^ row: what a wave reads at a time, one piece of 16 key rows or two neighbours of 16 value
// rows, falls on different banks.  Values are read through the transposing load: lane 4 j + a of 16
// reads elements 4 a .. of row j, and lane i gets element i of the four rows.
// 12 x 64 nodes, 32 heads of 128 over 8 key heads, 1,000 .. 8,191 bf16 rows: 132 us, 355 TFLOP/s.  The matrix
// units are busy 43% of its cycles (at 1.6 GHz: the card lowers its clock under this load), the waves
// wait 41% of theirs for an issue slot and 20% for data or the barrier.  With one plane of probabilities
// (98 us) tiles two ahead in registers spilled (161 us for 144 then), and two ahead by direct loads to LDS gained 4% at
// best; blocks of 8 waves read every tile half as often and were no faster (103 us with the joining for 104;
// 2 x 144 nodes over 3,700 rows 38, 38).
template <int D, class TQ, class TKV, int RT, int W>
__global__ __launch_bounds__(64 * kRowWaves, 2) void tree_attn_rows_kernel(Args p) {
  constexpr int WR = kRowWaves, kPieces = D * TKV::kBytes / 16, kThreads = 64 * WR, kTile = kTileKeys * kPieces, kCopy = 2 * kTile / kThreads;
  static_assert(2 * kTile % kThreads == 0 && TKV::kBytes == 2, "whole pieces a thread");
  __shared__ typename Tree<W>::Shared tree_mem;
  __shared__ u32x4 key_mem[2][kTile], value_mem[2][kTile];
  const TreeAttn &a = p.a;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
  const int hk = blockIdx.y % a.Hk, row0 = (blockIdx.y / a.Hk * WR + wave) * (16 * RT);
  const Share share = share_of(p);
  if (share.n == 0) return;
  const int b = share.b;
  if (p.parts > 0 && share.first == 0 && blockIdx.y == 0 && threadIdx.x == 0) p.dealt[b] = make_int2(share.from, share.n);
  const char *kb = static_cast<const char *>(a.k) + (b * a.k_b + hk * a.k_h) * TKV::kBytes;
  const char *vb = static_cast<const char *>(a.v) + (b * a.v_b + hk * a.v_h) * TKV::kBytes;
  const uint32_t k_step = (uint32_t)a.k_r * TKV::kBytes, v_step = (uint32_t)a.v_r * TKV::kBytes;
  int key0 = share.first;
  const int len = a.lengths[b];
  const int par_at = W == 1 ? lane : threadIdx.x;
  const int par = par_at < a.n ? a.parents[b * a.par_b + par_at] : -2;

  // A thread's pieces of two tiles: row i / kPieces of the first, then of the second, piece i % kPieces.
  // Rows past `last` are read as that one.
  auto fetch = [&](u32x4 (&copy)[kCopy], int key, const char *other, uint32_t other_step, int other_key, int last) {
#pragma unroll
    for (int i = 0; i < kCopy; i++) {
      const int at = i * kThreads + threadIdx.x, in = at % kTile;
      const char *row = at < kTile ? kb + (uint64_t)(uint32_t)min(key + in / kPieces, last) * k_step
                                   : other + (uint64_t)(uint32_t)min(other_key + in / kPieces, last) * other_step;
      copy[i] = *reinterpret_cast<const u32x4 *>(row + in % kPieces * 16);
    }
  };
  auto keep = [&](const u32x4 (&copy)[kCopy], u32x4 *first, u32x4 *second) {
#pragma unroll
    for (int i = 0; i < kCopy; i++) {
      const int at = i * kThreads + threadIdx.x, in = at % kTile, row = in / kPieces;
      (at < kTile ? first : second)[row * kPieces + ((in ^ row) & (kPieces - 1))] = copy[i];
    }
  };
  // Everything that does not wait for something else is loaded first: the keys of tiles 0 and 1, then
  // those of tile 2 and the values of tile 0, wherever the length ends.
  u32x4 copy0[kCopy], copy[kCopy];
  const int last_row = a.max_seq - 1;
  fetch(copy0, min(key0, last_row), kb, k_step, min(key0 + kTileKeys, last_row), last_row);
  fetch(copy, min(key0 + 2 * kTileKeys, last_row), vb, v_step, min(key0, last_row), last_row);
  using Wave = Rows<D, TQ, TKV, RT, true>;
  Wave rows;
  int node[RT];
  load_rows<D, TQ>(p, b, hk, row0, c, g, rows, node);
  Tree<W> tree;
  tree.read(par, a.n, tree_mem);
  const int live = tree.live;
  const bool bad = len < 0 || live > a.max_seq || len > a.max_seq - live;
  const int total = bad ? 0 : len + live, end = min(total, share.end);
  typename Tree<W>::Row sees[RT];
#pragma unroll
  for (int t = 0; t < RT; t++) sees[t] = tree.row(node[t], tree_mem);

  uint32_t odd = 0;
  const bool keys = key0 < total;
  auto next = [&](int tiles) {  // (past the last tile: one row, once more)
    const int key = key0 + tiles * kTileKeys;
    return key < end ? key : total - 1;
  };
  auto scores = [&](floatx4 (&s)[2][RT], int buf) {
#pragma unroll
    for (int j = 0; j < D / 32; j++) {
      uint32_t k[2][4];
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const u32x4 w = key_mem[buf][(16 * h + c) * kPieces + ((4 * j + g) ^ (c & (kPieces - 1)))];
        k[h][0] = w[0], k[h][1] = w[1], k[h][2] = w[2], k[h][3] = w[3];
      }
      rows.scores(s, j, k[0], k[1]);
    }
  };
  floatx4 s[2][RT] = {};
  if (keys) {
    keep(copy0, key_mem[0], key_mem[1]);
    __syncthreads();
    scores(s, 0);
    __syncthreads();
    keep(copy, key_mem[0], value_mem[0]);
    fetch(copy, next(2), vb, v_step, next(1), total - 1);
    __syncthreads();
  }
  int buf = 0;
  auto step = [&](auto is_edge) {
    constexpr bool kEdge = decltype(is_edge)::value;
    // here: this tile's scores and values (buf), the next one's keys (buf ^ 1); to LDS: the keys after
    // those, the next values; on their way: what follows
    keep(copy, key_mem[buf], value_mem[buf ^ 1]);
    fetch(copy, next(3), vb, v_step, next(2), total - 1);
    uint32_t seen[RT] = {};
    if constexpr (kEdge) {
#pragma unroll
      for (int t = 0; t < RT; t++) seen[t] = sees[t].tile(key0 - len) >> (4 * g);
    }
    rows.limit(s, kEdge, seen);
    floatx4 s_next[2][RT] = {};
    scores(s_next, buf ^ 1);
    rows.weigh(s);
    typename Wave::Probs probs;
    rows.pack(s, probs);
    rows.add_sums(probs);
#pragma unroll
    for (int d0 = 0; d0 < D / 16; d0 += 4) {  // (four at a time: fewer registers)
      uint32_t vt[4][4];
#pragma unroll
      for (int d = 0; d < 4; d++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const int row = 16 * h + 4 * g + (c >> 2), piece = 2 * (d0 + d) + (c >> 1 & 1);
          const u32x2 w = load_transposed(&value_mem[buf][row * kPieces + (piece ^ (row & (kPieces - 1)))], c & 1);
          vt[d][2 * h] = w[0], vt[d][2 * h + 1] = w[1];
        }
      if constexpr (kEdge) odd |= take_odd_columns<TKV>(vt, key0, len, total, g);
      rows.add(probs, d0, vt);
    }
#pragma unroll
    for (int t = 0; t < RT; t++) s[0][t] = s_next[0][t], s[1][t] = s_next[1][t];
    key0 += kTileKeys;
    buf ^= 1;
    __syncthreads();
  };
  while (key0 + kTileKeys <= min(end, len)) step(std::false_type{});
  while (key0 < end) step(std::true_type{});  // tiles with nodes, or past the last row

  const bool odd_any = __ballot(odd != 0) != 0;
#pragma unroll
  for (int t = 0; t < RT; t++) {
    const int row = row0 + 16 * t + c;
    if (row >= p.M) continue;
    float planes = 0.0f;
#pragma unroll
    for (int d = 0; d < D / 16; d++) {  // lane (c, g) holds dims 16 d + 4 g .. of row c
      float y[4] = {rows.o[t][d][0], rows.o[t][d][1], rows.o[t][d][2], rows.o[t][d][3]};
      const int e = 16 * d + 4 * g;
      if (odd_any) odd_values<TKV, 4>(y, sees[t], live, vb + (uint64_t)(uint32_t)len * v_step + e * TKV::kBytes, v_step);
      planes += put4<D, TQ>(p, share, hk, row, node[t], e, y, rows.m[t], rows.l[t][0], bad, sees[t].any(), keys);
    }
    if (has_planes<D, TQ>(p) && share.n == 1) {
      planes = col_sum(planes);
      if (g == 0) put_sum<D, TQ>(p, b, hk, row, node[t], planes);
    }
  }
}

// Joins the blocks' results of a row: a wave a row, D / 4 lanes with four elements each for every fourth
// (D 128: second) block, added in their order there and then over the lane groups.  Bound by memory where
// it counts: 33 MB of results 12 us.
template <int D, class TQ>
__global__ __launch_bounds__(256) void tree_join_kernel(Args p) {
  constexpr int kLanes = D / 4, kGroups = 64 / kLanes;
  const TreeAttn &a = p.a;
  const int lane = threadIdx.x & 63, d = lane % kLanes * 4, s0 = lane / kLanes, M = p.M;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (item >= (int64_t)a.batch * a.Hk * M) return;
  const int row = item % M, hk = item / M % a.Hk, b = item / M / a.Hk;
  const int2 dealt = p.dealt[b];
  const int S = dealt.y;
  if (S == 1) return;  // (that block has written the row)
  const size_t at = ((size_t)hk * M + row) * p.parts + dealt.x;
  const float *part = a.part + at * D + d;
  const float2 own = p.ml[at + min(lane, S - 1)];  // (at most 64 blocks)
  float4 o = *reinterpret_cast<const float4 *>(part + (size_t)min(s0, S - 1) * D);  // (before what weighs it is there)
  const float top = wave_max(own.x), ms = top == -INFINITY ? 0.0f : top;
  const bool none = __ballot(own.x == INFINITY && own.y == 0.0f) != 0;
  const float f_own = __builtin_amdgcn_exp2f(own.x - ms);
  // (a weight that is positive, if not as a float: times an infinity it is that)
  auto weighed = [](float f, float y) { return fabsf(y) < INFINITY ? f * y : y; };
  float sum = 0.0f, x[4] = {};
  for (int s1 = 0; s1 < S; s1 += kGroups) {
    const int s = min(s1 + s0, S - 1);
    const float4 next = *reinterpret_cast<const float4 *>(part + (size_t)min(s + kGroups, S - 1) * D);
    const float m = __shfl(own.x, s, 64), l = __shfl(own.y, s, 64), f = __shfl(f_own, s, 64);
    const bool in = s1 + s0 < S && !(m == -INFINITY && l == 0.0f);  // without keys nothing was stored
    const bool num = in && l == l;
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
  const int node = p.node(row);
  float planes = put_result<D, TQ>(p, b, hk, row, node, d, x);
  if (has_planes<D, TQ>(p)) {
#pragma unroll
    for (int step = 1; step < kLanes; step *= 2) planes += __shfl_xor(planes, step, 64);
    if (d == 0) put_sum<D, TQ>(p, b, hk, row, node, planes);
  }
}

// Most tiles of 16 query rows a wave takes: as many as its registers hold (256 a lane, two waves a
// SIMD).  fp32 queries take up to three times the registers of 16-bit ones.
constexpr int most_tiles(int D, int q_bytes) { return (q_bytes == 4 ? 128 : 256) / D; }
// The same where the waves share tiles, and hold none themselves.
constexpr int rows_tiles(int D, int q_bytes) { return D == 128 && q_bytes == 4 ? 1 : 2; }

// How a launch is laid out: every wave with keys of its own and all RT tiles of 16 query rows of its
// block (tree_attn_kernel), or with RT tiles of its own and the block's keys (shared,
// tree_attn_rows_kernel); one block a sequence (parts 0) or `parts` for all of them.
struct Plan {
  bool shared;
  int parts, RT, row_tiles, unit, least;
  double us;  // what it should take
};

// The time of a layout: a block's start and end, and for every 2^unit keys `turn`, as often as a compute
// unit has blocks (in pairs, those with shared tiles); dealing a sequence's keys
// to several blocks adds a wait for the lengths, the second launch and its traffic.  The figures (us) are
// those of launches that fill the card.  Given the sequences' mean length, they lie between 0.65 and 1.09 of what nine in ten of
// 304 layouts of 16-bit caches take (median 0.94; low where lengths differ or trees are larger than 64 nodes).  Of
// 311 shapes whose sequences use 0.65 to 1 of max_seq, where half is expected, the layout taken was 4% slower than the
// best of all on average, more than 10% in 40, 43% at worst.  What they decide, over 3,000 | 300 rows that all
// sequences use (one block a sequence or dealt, whichever is faster):
//   bf16, 4 x 16 heads of 64, 64 nodes            RT 1 21.8 | 6.5   RT 2 20.4 | 7.6    RT 4 20.2 | 10.0   shared 28.2 | 13.8
//   bf16, 4 x 8 key heads of 128, 128 rows each   RT 1 32.5 | 8.2   RT 2 27.9 | 10.4   shared 34.3 | 17.2
//   the same, 256 rows each                       RT 1 58.8 | 12.9  RT 2 35.2 | 11.0   shared 44.1 | 19.2
//   fp32 over bf16, 2 x 20 heads of 64, 48 nodes  RT 1 19.0 | 7.0   RT 2 19.6 | 9.2    shared 28.1 | 15.5
//   256 rows each, 12 sequences up to 8,191 rows  RT 2 235          shared 139
// and fp32 caches, 20 heads of 64, 1,734 rows: 48 nodes RT 1 15.7, RT 2 18.6; 3 x 4 key heads, 189 rows each, up to
// 5,936 rows 51, 44.
Plan plan_of(const TreeAttn &a, int n_cu, int RT, bool shared) {
  Plan p;
  const int M = a.n * (a.H / a.Hk), per = 16 * RT * (shared ? kRowWaves : 1);
  const bool wide = a.qt == kOpF32, d128 = a.D == 128;
  p.shared = shared, p.RT = RT, p.row_tiles = (M + per - 1) / per;
  p.unit = shared ? 5 : 7, p.least = shared ? 8 : 2;
  double start, turn;
  if (shared) {
    start = d128 ? 10.0 : 8.5;
    turn = wide ? (d128 ? 1.7 : 1.6) : d128 ? 1.6 : 0.95;
  } else if (a.kvt == kOpF32) {
    start = d128 ? 9.7 : 4.6 + 2.2 * RT;
    turn = d128 ? 2.2 : 0.2 + 0.9 * RT;
  } else {
    start = (wide ? 4.5 : 4.0) + (d128 ? 2.2 : 1.2) * RT;
    turn = d128 ? 1.0 + 0.1 * RT : 0.63 + 0.08 * RT;
  }
  const int at_once = n_cu * (shared ? 2 : 1), groups = a.Hk * p.row_tiles;
  const double rows = std::max(1.0, (double)a.used * a.max_seq), units = std::ceil(rows / (1 << p.unit));
  p.us = (start + units * turn) * (((int64_t)a.batch * groups + at_once - 1) / at_once);
  // A block a compute unit: 2 x 16 heads over 40,001 and 65,500 rows 86 us, two a unit 90, half as many
  // 128.  Two of shared tiles, with one plane of probabilities: 2 x 20 heads, 84 nodes over 15,765 rows 48 us, one a unit 62;
  // 24 x 4 key heads, 72 rows over 4,748 .. 5,359 58, 80 (with two planes 64 and 77, two a unit).
  p.parts = (int)std::min<int64_t>(at_once / groups, 64ll * a.batch);
  // (row tiles with the same keys on the same eighth of the card, which has an L2 of its own: 6 heads of a
  // key head, 6 nodes, 2 x 52,834 rows 36 -> 29 us)
  if (p.row_tiles > 1 && p.parts > 8) p.parts -= p.parts % (8 / std::gcd(8, a.Hk));
  // Lengths are not known here: dealing has to pay at the part of max_seq that is used on average.  20
  // heads, 8 nodes, a bf16 cache of 512, 1,024, 2,048, 4,096 rows: one block 8, 11, 16, 26 us, dealt 11, 11, 12, 13; fp32:
  // 11, 16, 24, 46 and 12, 13, 13, 16; 8 sequences over bf16: 8, 12, 18, 29 and 12, 16, 22, 33.
  const double dealt = p.parts > a.batch ? start + 4.5 + std::max<double>(p.least, std::ceil(units * a.batch / p.parts)) * turn +
                                               2e-6 * p.parts * a.H * a.n * a.D
                                         : p.us;
  if (dealt < p.us) p.us = dealt;
  else p.parts = 0;
  return p;
}
Plan make_plan(const TreeAttn &a, int n_cu) {
  const int bytes = a.qt == kOpF32 ? 4 : 2, most = most_tiles(a.D, bytes);
  Plan best;
  best.us = INFINITY;
  auto offer = [&](int RT, bool shared) {
    const Plan p = plan_of(a, n_cu, RT, shared);
    if (p.us < best.us) best = p;
  };
  for (int rt = 1; rt <= most; rt *= 2)
    if (a.n <= 64 || rt == std::min(most, 2)) offer(rt, false);  // (larger trees: one of them)
  if (a.kvt != kOpF32) offer(rows_tiles(a.D, bytes), true);
  return best;
}

size_t part_rows(const TreeAttn &a, const Plan &p) { return (size_t)a.H * a.n * p.parts; }
Args make_args(const TreeAttn &a, const Plan &p) {
  const int group = a.H / a.Hk;
  float *ml = a.part + part_rows(a, p) * a.D;
  return Args{a, p.parts, a.n * group, group, (uint32_t)(((1ull << 32) + group - 1) / group), p.unit, p.least,
              reinterpret_cast<float2 *>(ml), reinterpret_cast<int2 *>(ml + 2 * part_rows(a, p))};
}
template <int D, class TQ, class K>
hipError_t launch_kernel(K kernel, int threads, const TreeAttn &a, const Plan &p, hipStream_t s) {
  const Args args = make_args(a, p);
  hipLaunchKernelGGL(kernel, dim3(p.parts > 0 ? p.parts : a.batch, a.Hk * p.row_tiles), dim3(threads), 0, s, args);
  if (hipError_t e = hipGetLastError(); e != hipSuccess || p.parts == 0) return e;
  const int64_t rows = (int64_t)a.batch * a.H * a.n;
  hipLaunchKernelGGL((tree_join_kernel<D, TQ>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, args);
  return hipGetLastError();
}
template <int D, class TQ, class TKV>
hipError_t launch_d(const TreeAttn &a, const Plan &p, hipStream_t s) {
  constexpr int kMost = most_tiles(D, TQ::kBytes), kRows = rows_tiles(D, TQ::kBytes), kKeyThreads = 64 * kKeyWaves;
  if constexpr (TKV::kBytes == 2) {
    if (p.shared && a.n > 64) return launch_kernel<D, TQ>(tree_attn_rows_kernel<D, TQ, TKV, kRows, 4>, 64 * kRowWaves, a, p, s);
    if (p.shared) return launch_kernel<D, TQ>(tree_attn_rows_kernel<D, TQ, TKV, kRows, 1>, 64 * kRowWaves, a, p, s);
  }
  if (a.n > 64) return launch_kernel<D, TQ>(tree_attn_kernel<D, TQ, TKV, std::min(kMost, 2), 4>, kKeyThreads, a, p, s);
  if constexpr (kMost >= 4)
    if (p.RT == 4) return launch_kernel<D, TQ>(tree_attn_kernel<D, TQ, TKV, 4, 1>, kKeyThreads, a, p, s);
  if constexpr (kMost >= 2)
    if (p.RT == 2) return launch_kernel<D, TQ>(tree_attn_kernel<D, TQ, TKV, 2, 1>, kKeyThreads, a, p, s);
  return launch_kernel<D, TQ>(tree_attn_kernel<D, TQ, TKV, 1, 1>, kKeyThreads, a, p, s);
}
template <class TQ, class TKV>
hipError_t launch_t(const TreeAttn &a, const Plan &p, hipStream_t s) {
  return a.D == 64 ? launch_d<64, TQ, TKV>(a, p, s) : launch_d<128, TQ, TKV>(a, p, s);
}

__global__ void tree_seqs_kernel(const int32_t *in, int n, BatchSeq *seqs, DecodeCtl *ctl, void *k, void *v) {
  const int i = blockIdx.x * 64 + threadIdx.x;
  if (i >= n) return;
  ctl[i].tok = in[i];
  ctl[i].pos = in[n + i];
  ctl[i].valid_len = in[3 * n] + i;
  ctl[i].done = 0;
  seqs[i] = BatchSeq{ctl + i, k, v, nullptr};
}

// ---- kept rows ----
// A thread per 16-byte piece of a (layer, sequence, head)'s rows of K or V takes the path's rows in
// order: row i is read before a later row can be written over it, since path[i] >= i and rises.
__global__ __launch_bounds__(256) void cache_keep_kernel(CacheKeep a) {
  const int b = blockIdx.y;
  const int32_t *path = a.path + b * a.path_b;
  const int len = a.lengths[b];
  int n = 0, last = -1;
  bool ok = len >= 0;
  for (; n < a.n_path && path[n] >= 0; n++) {
    ok = ok && path[n] > last && path[n] < a.max_seq - len;
    last = path[n];
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) a.new_lengths[b] = ok ? len + n : -1;
  int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  // (past the last piece; caches without layers or heads have none, only lengths)
  if (!ok || i >= (int64_t)a.caches * a.layers * a.heads * a.row_pieces) return;
  const int piece = i % a.row_pieces;
  i /= a.row_pieces;
  const int head = i % a.heads;
  i /= a.heads;
  const int layer = i % a.layers, is_v = (int)(i / a.layers);
  uint4 *base = is_v ? static_cast<uint4 *>(a.v) + layer * a.v_l + b * a.v_b + head * a.v_h
                     : static_cast<uint4 *>(a.k) + layer * a.k_l + b * a.k_b + head * a.k_h;
  const int64_t step = is_v ? a.v_r : a.k_r;
  base += len * step + piece;
  for (int j = 0; j < n; j++)
    if (path[j] != j) base[j * step] = base[path[j] * step];
}

}  // namespace

size_t tree_attn_ws(const TreeAttn &a, int n_cu) {
  const Plan p = make_plan(a, n_cu);
  return p.parts == 0 ? 0 : part_rows(a, p) * (a.D + 2) + 2 * (size_t)a.batch;
}

hipError_t tree_attn(const TreeAttn &a, int n_cu, hipStream_t s) {
  if (a.batch <= 0 || a.n <= 0) return hipSuccess;
  if (a.n > kTreeMaxNodes || (a.D != 64 && a.D != 128) || a.H % a.Hk) return hipErrorInvalidValue;
  const Plan p = make_plan(a, n_cu);
  if (p.parts > 0 && !a.part) return hipErrorInvalidValue;
  if (a.planes.hi && (a.D != 64 || a.qt != kOpF32)) return hipErrorInvalidValue;
  if (a.qt == kOpF32 && a.kvt == kOpF32) return launch_t<F32, F32>(a, p, s);
  if (a.qt == kOpF32 && a.kvt == kOpBf16) return launch_t<F32, Bf16>(a, p, s);
  if (a.qt == kOpBf16 && a.kvt == kOpBf16) return launch_t<Bf16, Bf16>(a, p, s);
  if (a.qt == kOpF16 && a.kvt == kOpF16) return launch_t<F16, F16>(a, p, s);
  return hipErrorInvalidValue;
}

hipError_t launch_tree_seqs(const int32_t *in, int n, BatchSeq *seqs, DecodeCtl *ctl, void *k, void *v, hipStream_t s) {
  hipLaunchKernelGGL(tree_seqs_kernel, dim3((n + 63) / 64), dim3(64), 0, s, in, n, seqs, ctl, k, v);
  return hipGetLastError();
}

hipError_t cache_keep(const CacheKeep &a, hipStream_t s) {
  if (a.batch <= 0) return hipSuccess;
  const int64_t items = (int64_t)a.caches * a.layers * a.heads * a.row_pieces;
  hipLaunchKernelGGL(cache_keep_kernel, dim3((unsigned)std::max<int64_t>(1, (items + 255) / 256), a.batch), dim3(256), 0, s,
                     a);
  return hipGetLastError();
}

}  // namespace itts
