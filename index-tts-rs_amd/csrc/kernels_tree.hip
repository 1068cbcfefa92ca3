// Decoding with drafted trees: attention of every node of a tree of tokens over its sequence's
// cached keys and values and its own ancestors, and the accepted nodes' rows moved up in the cache.
//
// Attention.  Node i of sequence b sees the rows t < lengths[b] and the rows lengths[b] + j of the
// nodes j on its path to the root, itself among them:
//   o_i = sum_t p_it v_t / sum_t p_it,   p_it = exp(scale q_i . k_t - m_i).
// The M = n H / Hk query rows that share a key head are the columns of one product, S^T = K Q^T, so
// that a lane of the 16 x 16 result holds four keys of one query: those are the B operand of the
// second product, O^T = V^T P^T, as they stand, when V's rows are read in the same key order.
// Softmax statistics stay in the lanes (max over the four lane groups of a column by two
// exchanges, sums only at the end).
#include <hip/hip_bf16.h>

#include <algorithm>

#include "kernels.h"

namespace itts {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;       // waves of a block, each over its own tiles of keys
constexpr int kTileKeys = 32;   // keys a wave takes at a time
constexpr float kLog2e = 1.4426950408889634f;

struct F32 {
  static constexpr int kBytes = 4;
};
struct Bf16 {
  static constexpr int kBytes = 2;
};
struct F16 {
  static constexpr int kBytes = 2;
};

// N consecutive elements at p (16-byte aligned where N elements fill 16 bytes) as floats.
template <class T, int N>
__device__ __forceinline__ void load_row(const void *p, float *o) {
  if constexpr (T::kBytes == 4) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 v = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + i);
      o[i] = v.x, o[i + 1] = v.y, o[i + 2] = v.z, o[i + 3] = v.w;
    }
  } else {
    uint32_t w[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; i += (N >= 8 ? 4 : 2)) {
      if constexpr (N >= 8) {
        const uint4 v = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p) + 2 * i);
        w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
      } else {
        const uint2 v = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(p) + 2 * i);
        w[i] = v.x, w[i + 1] = v.y;
      }
    }
#pragma unroll
    for (int i = 0; i < N / 2; i++) {
      if constexpr (std::is_same_v<T, Bf16>) {
        o[2 * i] = __uint_as_float(w[i] << 16);
        o[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        o[2 * i] = half_bits_to_float(w[i] & 0xffffu);
        o[2 * i + 1] = half_bits_to_float(w[i] >> 16);
      }
    }
  }
}

// One rounding to the output's type.
template <class T>
__device__ __forceinline__ void store4(void *p, float a, float b, float c, float d) {
  if constexpr (T::kBytes == 4) {
    *static_cast<float4 *>(p) = make_float4(a, b, c, d);
  } else if constexpr (std::is_same_v<T, Bf16>) {
    *static_cast<uint2 *>(p) = make_uint2(float_to_bf16_bits(a) | float_to_bf16_bits(b) << 16,
                                          float_to_bf16_bits(c) | float_to_bf16_bits(d) << 16);
  } else {
    const f16x2v x = __builtin_convertvector((f32x2e){a, b}, f16x2v), y = __builtin_convertvector((f32x2e){c, d}, f16x2v);
    *static_cast<uint2 *>(p) = make_uint2(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, y));
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

// The tree of one sequence: every node's ancestors (itself among them) as bits, none for a slot
// that is unused or hangs below one, and the number of slots up to the last used one.
struct Tree {
  uint64_t anc[kTreeMaxNodes][4];
  int up[kTreeMaxNodes];
  int live;
};

// Follows the parents by doubling: after step k a node knows 2^k of its ancestors.  All threads.
__device__ inline void read_tree(const int32_t *par, int n, Tree &t) {
  const int i = threadIdx.x;
  static_assert(64 * kWaves >= kTreeMaxNodes, "a thread for each node");
  if (i == 0) t.live = 0;
  if (i < n) {
    const int p = par[i];
    t.up[i] = p >= -1 && p < i ? p : -2;  // -1: the root is reached; -2: not in the tree
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
}

// Partial results of key split s: o [batch][Hk][M][S][D], then (max, sum) [batch][Hk][M][S].
__host__ __device__ inline size_t part_row(const TreeAttn &a, int S, int b, int hk, int row) {
  return (((size_t)b * a.Hk + hk) * (a.n * (a.H / a.Hk)) + row) * S;
}

template <int D, class TQ, class TKV, int RT>
__global__ __launch_bounds__(64 * kWaves) void tree_attn_kernel(TreeAttn a, int S, float2 *ml) {
  __shared__ Tree tree;
  __shared__ float so[kWaves][16 * RT][D + 4];
  __shared__ float sm[kWaves][16 * RT], sl[kWaves][16 * RT];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
  const int split = blockIdx.x, b = blockIdx.z;
  const int group = a.H / a.Hk, M = a.n * group;
  const int hk = blockIdx.y % a.Hk, row0 = blockIdx.y / a.Hk * (16 * RT);
  read_tree(a.parents + b * a.par_b, a.n, tree);
  const int len = a.lengths[b], live = tree.live;
  const bool bad = len < 0 || live > a.max_seq || len > a.max_seq - live;
  const int total = bad ? 0 : len + live;
  const int tiles = (total + kTileKeys - 1) / kTileKeys, per = (tiles + S - 1) / S;
  const int t_end = min(tiles, (split + 1) * per);

  // queries of this lane's columns, scaled for powers of two; k = 32 j + 8 g + e is element 8 j + e
  float q[RT][D / 4];
  int node[RT];
#pragma unroll
  for (int t = 0; t < RT; t++) {
    const int row = min(row0 + 16 * t + c, M - 1);
    node[t] = row / group;
    const int64_t at = b * a.q_b + node[t] * a.q_n + (hk * group + row % group) * a.q_h;
#pragma unroll
    for (int j = 0; j < D / 32; j++)
      load_row<TQ, 8>(static_cast<const char *>(a.q) + (at + 32 * j + 8 * g) * TQ::kBytes, &q[t][8 * j]);
  }
  const float scale = a.scale * kLog2e;
  const char *kb = static_cast<const char *>(a.k) + (b * a.k_b + hk * a.k_h) * TKV::kBytes;
  const char *vb = static_cast<const char *>(a.v) + (b * a.v_b + hk * a.v_h) * TKV::kBytes;

  f32x4 o[RT][D / 16] = {};
  float m[RT], l[RT];
#pragma unroll
  for (int t = 0; t < RT; t++) m[t] = -INFINITY, l[t] = 0.0f;

  for (int tile = split * per + wave; tile < t_end; tile += kWaves) {
    const int key0 = tile * kTileKeys;
    f32x4 s[2][RT] = {};
#pragma unroll
    for (int h = 0; h < 2; h++) {
      float kk[D / 4];
      const int64_t row = min(key0 + 16 * h + c, total - 1);
#pragma unroll
      for (int j = 0; j < D / 32; j++)
        load_row<TKV, 8>(kb + (row * a.k_r + 32 * j + 8 * g) * TKV::kBytes, &kk[8 * j]);
#pragma unroll
      for (int t = 0; t < RT; t++)
#pragma unroll
        for (int e = 0; e < D / 4; e++)
          s[h][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(kk[e], q[t][e], s[h][t], 0, 0, 0);
    }
    const bool edge = key0 + kTileKeys > len;  // holds nodes, or ends past the last row
#pragma unroll
    for (int t = 0; t < RT; t++) {
      float top = -INFINITY;
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          s[h][t][r] *= scale;
          if (edge) {
            const int j = key0 + 16 * h + 4 * g + r - len;
            const bool sees = j < 0 || (j < live && (tree.anc[node[t]][(j >> 6) & 3] >> (j & 63) & 1));
            s[h][t][r] = sees ? s[h][t][r] : -INFINITY;
          }
          top = fmaxf(top, s[h][t][r]);
        }
      const float mn = fmaxf(m[t], col_max(top)), ms = mn == -INFINITY ? 0.0f : mn;
      const float f = __builtin_amdgcn_exp2f(m[t] - ms);
      m[t] = mn;
      l[t] *= f;
#pragma unroll
      for (int d = 0; d < D / 16; d++) o[t][d] *= f;
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          s[h][t][r] = __builtin_amdgcn_exp2f(s[h][t][r] - ms);
          l[t] += s[h][t][r];
        }
    }
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const int key = key0 + 16 * h + 4 * g + r;
        float vv[D / 16];
        load_row<TKV, D / 16>(vb + ((int64_t)min(key, total - 1) * a.v_r + D / 16 * c) * TKV::kBytes, vv);
        if (edge) {
          // rows of nodes count only where they are seen: 0 times what a masked row may hold
          // (infinities, NaN) must stay out, so such values leave the product and are added
          // below, query by query
          bool odd = false;
#pragma unroll
          for (int d = 0; d < D / 16; d++) {
            const bool fin = key < len || fabsf(vv[d]) < INFINITY;
            odd = odd || (key < total && !fin);
            vv[d] = key < total && fin ? vv[d] : 0.0f;
          }
          if (__ballot(odd)) {
            for (int gg = 0; gg < 4; gg++) {
              const int kx = key0 + 16 * h + 4 * gg + r, j = kx - len;
              if (j < 0 || j >= live) continue;
#pragma unroll
              for (int t = 0; t < RT; t++) {
                const float p = __shfl(s[h][t][r], c + 16 * gg, 64);
                const bool sees = tree.anc[node[t]][j >> 6] >> (j & 63) & 1;
#pragma unroll
                for (int d = 0; d < D / 16; d++)
#pragma unroll
                  for (int rr = 0; rr < 4; rr++) {
                    float x;
                    const char *at = vb + ((int64_t)kx * a.v_r + D / 16 * (4 * g + rr) + d) * TKV::kBytes;
                    if constexpr (TKV::kBytes == 4) x = *reinterpret_cast<const float *>(at);
                    else if constexpr (std::is_same_v<TKV, Bf16>) x = bf16_bits_to_float(*reinterpret_cast<const uint16_t *>(at));
                    else x = half_bits_to_float(*reinterpret_cast<const uint16_t *>(at));
                    if (sees && !(fabsf(x) < INFINITY)) o[t][d][rr] += p * x;
                  }
              }
            }
          }
        }
#pragma unroll
        for (int t = 0; t < RT; t++)
#pragma unroll
          for (int d = 0; d < D / 16; d++)
            o[t][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(vv[d], s[h][t][r], o[t][d], 0, 0, 0);
      }
  }

  // the block's waves joined: lane (c, g) holds dims D/4 g .. of column c, in runs of D/16 a register
#pragma unroll
  for (int t = 0; t < RT; t++) {
    l[t] = col_sum(l[t]);
    if (g == 0) sm[wave][16 * t + c] = m[t], sl[wave][16 * t + c] = l[t];
#pragma unroll
    for (int r = 0; r < 4; r++)
#pragma unroll
      for (int d = 0; d < D / 16; d += 4)
        *reinterpret_cast<float4 *>(&so[wave][16 * t + c][D / 16 * (4 * g + r) + d]) =
            make_float4(o[t][d][r], o[t][d + 1][r], o[t][d + 2][r], o[t][d + 3][r]);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * RT * (D / 4); i += 64 * kWaves) {
    const int rr = i / (D / 4), d = i % (D / 4) * 4, row = row0 + rr;
    if (row >= M) continue;
    float top = -INFINITY, sum = 0.0f, x[4] = {};
#pragma unroll
    for (int w = 0; w < kWaves; w++) top = fmaxf(top, sm[w][rr]);
    const float ms = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
      const float f = __builtin_amdgcn_exp2f(sm[w][rr] - ms);
      const float4 v = *reinterpret_cast<const float4 *>(&so[w][rr][d]);
      sum += f * sl[w][rr];
      x[0] += f * v.x, x[1] += f * v.y, x[2] += f * v.z, x[3] += f * v.w;
    }
    const int i_node = row / group;
    uint64_t any = 0;
#pragma unroll
    for (int w = 0; w < 4; w++) any |= tree.anc[i_node][w];
    if (S == 1) {
      const float inv = 1.0f / sum;
#pragma unroll
      for (int e = 0; e < 4; e++) x[e] = bad ? NAN : any ? x[e] * inv : 0.0f;
      const int64_t at = b * a.o_b + i_node * a.o_n + (hk * group + row % group) * a.o_h + d;
      store4<TQ>(static_cast<char *>(a.out) + at * TQ::kBytes, x[0], x[1], x[2], x[3]);
    } else {
      // what the joining kernel cannot tell by itself goes with the statistics: a row that sees
      // nothing has maximum +inf and sum 0, one of a bad sequence sum NaN
      const size_t at = part_row(a, S, b, hk, row) + split;
      if (split * per < t_end) *reinterpret_cast<float4 *>(a.part + at * D + d) = make_float4(x[0], x[1], x[2], x[3]);
      if (d == 0) ml[at] = bad ? make_float2(0.0f, NAN) : any ? make_float2(top, sum) : make_float2(INFINITY, 0.0f);
    }
  }
}

// Joins the splits of a row: a wave a row, in split order.
template <int D, class TQ>
__global__ __launch_bounds__(256) void tree_join_kernel(TreeAttn a, int S, const float2 *ml) {
  const int lane = threadIdx.x & 63, group = a.H / a.Hk, M = a.n * group;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (item >= (int64_t)a.batch * a.Hk * M) return;
  const int row = item % M, hk = item / M % a.Hk, b = item / M / a.Hk;
  const size_t at = (size_t)item * S;
  float top = -INFINITY;
  for (int s = lane; s < S; s += 64) top = fmaxf(top, ml[at + s].x);
  top = wave_max(top);
  const float2 first = ml[at];
  const bool none = first.x == INFINITY && first.y == 0.0f;
  const float ms = top == -INFINITY ? 0.0f : top;
  constexpr int E = D / 64;
  float sum = 0.0f, x[E] = {};
  for (int s = 0; s < S; s++) {
    const float2 w = ml[at + s];
    if (w.x == -INFINITY && w.y == 0.0f) continue;  // no keys: nothing was stored
    const float f = __builtin_amdgcn_exp2f(w.x - ms);
    sum += f * w.y;
    if (none || w.y != w.y) continue;
#pragma unroll
    for (int e = 0; e < E; e++) x[e] += f * a.part[(at + s) * D + E * lane + e];
  }
  const float inv = 1.0f / sum;
  const int64_t to = b * a.o_b + row / group * a.o_n + (hk * group + row % group) * a.o_h + E * lane;
#pragma unroll
  for (int e = 0; e < E; e++) {
    const float y = none ? 0.0f : x[e] * inv;
    if constexpr (TQ::kBytes == 4) static_cast<float *>(a.out)[to + e] = y;
    else if constexpr (std::is_same_v<TQ, Bf16>) static_cast<uint16_t *>(a.out)[to + e] = (uint16_t)float_to_bf16_bits(y);
    else static_cast<_Float16 *>(a.out)[to + e] = (_Float16)y;
  }
}

struct Plan {
  int S, RT, row_tiles;
};
Plan make_plan(const TreeAttn &a, int n_cu) {
  Plan p;
  const int M = a.n * (a.H / a.Hk);
  const int most = a.D == 64 ? 4 : 2;
  p.RT = M <= 16 ? 1 : M <= 32 ? 2 : most;
  p.row_tiles = (M + 16 * p.RT - 1) / (16 * p.RT);
  const int tiles = (a.max_seq + kTileKeys - 1) / kTileKeys;
  const int64_t blocks = (int64_t)a.batch * a.Hk * p.row_tiles;
  const int64_t want = (2 * n_cu + blocks - 1) / blocks, can = (tiles + 4 * kWaves - 1) / (4 * kWaves);
  p.S = (int)std::max<int64_t>(1, std::min<int64_t>({want, can, 64}));
  return p;
}

template <int D, class TQ, class TKV, int RT>
hipError_t launch_rt(const TreeAttn &a, const Plan &p, hipStream_t s) {
  float2 *ml = reinterpret_cast<float2 *>(a.part + (size_t)a.batch * a.H * a.n * p.S * D);
  hipLaunchKernelGGL((tree_attn_kernel<D, TQ, TKV, RT>), dim3(p.S, a.Hk * p.row_tiles, a.batch), dim3(64 * kWaves), 0, s,
                     a, p.S, ml);
  if (hipError_t e = hipGetLastError(); e != hipSuccess || p.S == 1) return e;
  const int64_t rows = (int64_t)a.batch * a.H * a.n;
  hipLaunchKernelGGL((tree_join_kernel<D, TQ>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, a, p.S, ml);
  return hipGetLastError();
}
template <int D, class TQ, class TKV>
hipError_t launch_d(const TreeAttn &a, const Plan &p, hipStream_t s) {
  if (p.RT == 1) return launch_rt<D, TQ, TKV, 1>(a, p, s);
  if (D == 128 || p.RT == 2) return launch_rt<D, TQ, TKV, 2>(a, p, s);
  return launch_rt<D, TQ, TKV, D == 64 ? 4 : 2>(a, p, s);
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
  if (!ok) return;
  int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int piece = i % a.row_pieces;
  i /= a.row_pieces;
  const int head = i % a.heads;
  i /= a.heads;
  const int layer = i % a.layers, is_v = (int)(i / a.layers);
  if (is_v > 1) return;
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
  return p.S == 1 ? 0 : (size_t)a.batch * a.H * a.n * p.S * (a.D + 2);
}

hipError_t tree_attn(const TreeAttn &a, int n_cu, hipStream_t s) {
  if (a.batch <= 0 || a.n <= 0) return hipSuccess;
  if (a.n > kTreeMaxNodes || (a.D != 64 && a.D != 128) || a.H % a.Hk) return hipErrorInvalidValue;
  const Plan p = make_plan(a, n_cu);
  if (p.S > 1 && !a.part) return hipErrorInvalidValue;
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
  const int64_t items = 2ll * a.layers * a.heads * a.row_pieces;
  hipLaunchKernelGGL(cache_keep_kernel, dim3((unsigned)std::max<int64_t>(1, (items + 255) / 256), a.batch), dim3(256), 0, s,
                     a);
  return hipGetLastError();
}

}  // namespace itts
