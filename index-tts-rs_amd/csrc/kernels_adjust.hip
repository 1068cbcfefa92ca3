// Logits x of a row under penalties, biases and a mask: with c the times that token t is in the row's history,
//   y = (x < 0 ? x r : x / r) - (f c + p)   where c > 0, else x     (repetition r, frequency f, presence p),
//   y + bias of t, and -inf where t is not allowed.
// A block holds a piece of a row: its tokens' counts and biases come together in LDS, a word a token (the count below, the
// place of its last bias above: whole numbers, so that the order in which they come changes nothing), while its logits
// are on their way.  Bound by memory: each logit is read and written once.
#include <algorithm>

#include "kernels.h"

namespace itts {
namespace {

constexpr int kPer = 8;  // tokens a thread takes at a time

template <int TYPE>
struct Elem;
template <>
struct Elem<kOpF32> {
  using type = float;
  __device__ static float get(float v) { return v; }
  __device__ static float put(float v) { return v; }
};
template <>
struct Elem<kOpBf16> {
  using type = uint16_t;
  __device__ static float get(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
  __device__ static uint16_t put(float v) { return (uint16_t)__builtin_bit_cast(uint16_t, (__bf16)v); }
};
template <>
struct Elem<kOpF16> {
  using type = uint16_t;
  __device__ static float get(uint16_t v) { return (float)__builtin_bit_cast(_Float16, v); }
  __device__ static uint16_t put(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
};

// Eight neighbours of any alignment that their type allows.
template <class E>
struct __attribute__((packed, aligned(alignof(E)))) Run {
  E v[kPer];
};

// 8 x THREADS x RUNS tokens a block.  Every block goes through the row's whole lists, so pieces are large: 256 bf16 rows of 60,510
// under a mask, a history of 2,000 and 50 biases, a call: blocks of 4,096 tokens 29.3 us, 8,192 25.9, 16,384 20 (66 MB; without
// lists 13).  Blocks that take several pieces in turn, the next one's loads ahead of the lists of the one before: 22.
// All tokens pass with the mask alone; those of the lists, few, are then written again by whoever takes their word out of LDS
// first.
template <int TYPE, int kThreads, int RUNS>
__global__ __launch_bounds__(kThreads) void adjust_kernel(AdjustLogits a, int pieces) {
  using E = typename Elem<TYPE>::type;
  constexpr int kTurn = kThreads * kPer, kPiece = RUNS * kTurn, kAhead = 2;  // entries of a list that a thread has on their way
  __shared__ uint32_t there[kPiece];
  // (neighbouring blocks go to different eighths of the card: the pieces of all rows that lists are about, small tokens say, are
  // not left to one of them)
  const int row = blockIdx.x / pieces, first = (int)((blockIdx.x + row) % pieces) * kPiece, tid = threadIdx.x;
  const E *x = static_cast<const E *>(a.x) + row * a.x_row;
  E *y = static_cast<E *>(a.out) + row * a.out_row;
  const uint32_t *mask = a.allowed + row * a.allowed_row;
  Run<E> in[RUNS] = {};
  uint32_t allowed[RUNS];
#pragma unroll
  for (int j = 0; j < RUNS; j++) {
    const int t0 = first + kTurn * j + kPer * tid, left = a.vocab - t0;
    if (left >= kPer) {
      in[j] = *reinterpret_cast<const Run<E> *>(x + t0);
    } else {
#pragma unroll
      for (int e = 0; e < kPer; e++)
        if (e < left) in[j].v[e] = x[t0 + e];
    }
    allowed[j] = a.allowed && left > 0 ? mask[t0 >> 5] >> (t0 & 31) : 0xffu;
  }
  const bool lists = a.n_history > 0 || a.n_bias > 0;
  const int32_t *history = a.history + row * a.history_row, *bias_tokens = a.bias_tokens + row * a.bias_tokens_row;
  const float r = a.repetition ? a.repetition[row] : a.repetition_all, f = a.frequency ? a.frequency[row] : a.frequency_all,
              p = a.presence ? a.presence[row] : a.presence_all;
  // Entries of a list, kAhead of a thread at a time; those of the first turn stay in registers for the second pass.
  auto take = [&](const int32_t *list, int n, int i0, uint32_t (&t)[kAhead]) {
#pragma unroll
    for (int k = 0; k < kAhead; k++) t[k] = i0 + k * kThreads < n ? (uint32_t)list[i0 + k * kThreads] - first : ~0u;
  };
  const uint32_t room = min(kPiece, a.vocab - first);
  // a list turn by turn, as f(first entry, places)
  auto each = [&](const int32_t *list, int n, const uint32_t (&t0)[kAhead], auto f) {
    if (tid < n) f(tid, t0);
    for (int i0 = tid + kAhead * kThreads; i0 < n; i0 += kAhead * kThreads) {
      uint32_t t[kAhead];
      take(list, n, i0, t);
      f(i0, t);
    }
  };
  uint32_t history0[kAhead], bias0[kAhead];
  if (lists) {
    take(history, a.n_history, tid, history0);
    take(bias_tokens, a.n_bias, tid, bias0);
#pragma unroll
    for (int i = 0; i < kPiece / kThreads / 4; i++) reinterpret_cast<uint4 *>(there)[i * kThreads + tid] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    each(history, a.n_history, history0, [&](int, const uint32_t (&t)[kAhead]) {
#pragma unroll
      for (int k = 0; k < kAhead; k++) {
        if (t[k] >= room) continue;
        // the first lane's token, and whoever has it too, in one go: a token that comes back often would be added one by one
        const uint32_t one = __builtin_amdgcn_readfirstlane(t[k]);
        const uint64_t same = __ballot(t[k] == one);
        if (t[k] != one) atomicAdd(&there[t[k]], 1u);
        else if ((tid & 63) == __builtin_ctzll(same)) atomicAdd(&there[t[k]], (uint32_t)__builtin_popcountll(same));
      }
    });
  }
#pragma unroll
  for (int j = 0; j < RUNS; j++) {
    const int at = kTurn * j + kPer * tid, left = a.vocab - first - at;
    if (a.allowed) {
#pragma unroll
      for (int e = 0; e < kPer; e++) in[j].v[e] = allowed[j] >> e & 1 ? in[j].v[e] : Elem<TYPE>::put(-INFINITY);
    }
    if (left >= kPer) {
      *reinterpret_cast<Run<E> *>(y + first + at) = in[j];
    } else {
#pragma unroll
      for (int e = 0; e < kPer; e++)
        if (e < left) y[first + at + e] = in[j].v[e];
    }
  }
  if (!lists) return;
  __syncthreads();  // (the block's tokens are written, and counted)
  if (a.n_bias > 0) {
    each(bias_tokens, a.n_bias, bias0, [&](int i, const uint32_t (&t)[kAhead]) {
#pragma unroll
      for (int k = 0; k < kAhead; k++)
        if (t[k] < room) atomicMax(&there[t[k]], (uint32_t)(i + k * kThreads + 1) << 16 | (there[t[k]] & 0xffffu));
    });
    __syncthreads();
  }
  auto again = [&](int, const uint32_t (&t)[kAhead]) {
    // (step by step for all entries of the turn: their loads are on their way together)
    uint32_t w[kAhead];
    E v[kAhead];
    float bias[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; k++) w[k] = t[k] < room ? there[t[k]] : 0;
#pragma unroll
    for (int k = 0; k < kAhead; k++)
      if (w[k] != 0) w[k] = atomicExch(&there[t[k]], 0u);
#pragma unroll
    for (int k = 0; k < kAhead; k++) {
      if (w[k] == 0) continue;
      v[k] = x[first + t[k]];  // (written in place it is what it was, but where it is masked)
      if (a.allowed && !(mask[(first + t[k]) >> 5] >> ((first + t[k]) & 31) & 1)) w[k] = 0;
      bias[k] = w[k] >> 16 ? a.bias[row * a.bias_row + (w[k] >> 16) - 1] : 0.0f;
    }
#pragma unroll
    for (int k = 0; k < kAhead; k++) {
      if (w[k] == 0) continue;
      const uint32_t c = w[k] & 0xffffu;
      float y1 = Elem<TYPE>::get(v[k]);
      if (c > 0) y1 = (y1 < 0.0f ? y1 * r : y1 / r) - __builtin_fmaf(f, (float)c, p);
      if (w[k] >> 16) y1 += bias[k];
      y[first + t[k]] = Elem<TYPE>::put(y1);
    }
  };
  each(history, a.n_history, history0, again);
  each(bias_tokens, a.n_bias, bias0, again);
}

template <int TYPE, int kThreads, int RUNS>
hipError_t launch(const AdjustLogits &a, hipStream_t s) {
  constexpr int kPiece = kThreads * kPer * RUNS;
  const int pieces = (a.vocab + kPiece - 1) / kPiece;
  hipLaunchKernelGGL((adjust_kernel<TYPE, kThreads, RUNS>), dim3((unsigned)((int64_t)a.rows * pieces)), dim3(kThreads), 0, s, a, pieces);
  return hipGetLastError();
}
// Small rows in small blocks; the largest pieces where they are two blocks a compute unit.
template <int TYPE>
hipError_t launch(const AdjustLogits &a, int n_cu, hipStream_t s) {
  if (a.vocab <= 2048) return launch<TYPE, 256, 1>(a, s);
  if ((int64_t)a.rows * ((a.vocab + 16383) / 16384) >= 2 * n_cu) return launch<TYPE, 1024, 2>(a, s);
  return launch<TYPE, 1024, 1>(a, s);
}

}  // namespace

// (small pieces come with few rows)
bool adjust_logits_fits(int rows, int vocab) {
  return (vocab <= 2048 ? 256ll * rows : 1024ll * rows * ((vocab + 16383) / 16384)) <= kMaxLaunch;
}

hipError_t adjust_logits(const AdjustLogits &a, int n_cu, hipStream_t s) {
  if (a.rows <= 0) return hipSuccess;
  switch (a.type) {
    case kOpF32: return launch<kOpF32>(a, n_cu, s);
    case kOpBf16: return launch<kOpBf16>(a, n_cu, s);
    case kOpF16: return launch<kOpF16>(a, n_cu, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace itts
