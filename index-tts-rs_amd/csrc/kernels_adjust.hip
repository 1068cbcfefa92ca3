// Logits x of a row under penalties, biases and a mask: with c the times that token t is in the row's history,
//   y = (x < 0 ? x r : x / r) - (f c + p)   where c > 0, else x     (repetition r, frequency f, presence p),
//   y + bias of t, and -inf where t is not allowed.
// A block holds a piece of a row: its tokens' counts and biases come together in LDS, a word a token (the count below, the
// place of its last bias above: both orders of whole numbers, so that the same call gives the same bits), while its logits
// are on their way.  Bound by memory: each logit is read and written once.
#include <algorithm>

#include "kernels.h"

namespace itts {
namespace {

constexpr int kThreads = 256, kPer = 8;  // tokens a thread takes at a time
constexpr int kPiece = kThreads * kPer;  // and a block

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

template <int TYPE>
__global__ __launch_bounds__(kThreads) void adjust_kernel(AdjustLogits a, int pieces) {
  using E = typename Elem<TYPE>::type;
  __shared__ uint32_t there[kPiece];
  const int row = blockIdx.x / pieces, first = (blockIdx.x - row * pieces) * kPiece, tid = threadIdx.x;
  const int t0 = first + kPer * tid, left = a.vocab - t0;
  const E *x = static_cast<const E *>(a.x) + row * a.x_row + t0;
  E *y = static_cast<E *>(a.out) + row * a.out_row + t0;
  Run<E> in = {};
  if (left >= kPer) {
    in = *reinterpret_cast<const Run<E> *>(x);
  } else {
#pragma unroll
    for (int e = 0; e < kPer; e++)
      if (e < left) in.v[e] = x[e];
  }
  uint32_t allowed = 0xffu;
  if (a.allowed && left > 0) allowed = a.allowed[row * a.allowed_row + (t0 >> 5)] >> (t0 & 31);
  const float r = a.repetition ? a.repetition[row] : a.repetition_all, f = a.frequency ? a.frequency[row] : a.frequency_all,
              p = a.presence ? a.presence[row] : a.presence_all;

  const bool lists = a.n_history > 0 || a.n_bias > 0;
  const int32_t *bias_tokens = a.bias_tokens + row * a.bias_tokens_row;
  if (lists) {
#pragma unroll
    for (int i = 0; i < kPer; i++) there[i * kThreads + tid] = 0;
    __syncthreads();
    const int32_t *history = a.history + row * a.history_row;
    for (int i = tid; i < a.n_history; i += kThreads) {
      const uint32_t t = (uint32_t)history[i] - first;
      if (t < (uint32_t)kPiece) atomicAdd(&there[t], 1u);
    }
    __syncthreads();
    for (int i = tid; i < a.n_bias; i += kThreads) {
      const uint32_t t = (uint32_t)bias_tokens[i] - first;
      if (t < (uint32_t)kPiece) atomicMax(&there[t], (uint32_t)(i + 1) << 16 | (there[t] & 0xffffu));
    }
    __syncthreads();
  }
#pragma unroll
  for (int e = 0; e < kPer; e++) {
    float v = Elem<TYPE>::get(in.v[e]);
    if (lists) {
      const uint32_t w = there[kPer * tid + e], c = w & 0xffffu;
      if (c > 0) v = (v < 0.0f ? v * r : v / r) - __builtin_fmaf(f, (float)c, p);
      if (w >> 16) v += a.bias[row * a.bias_row + (w >> 16) - 1];
    }
    in.v[e] = Elem<TYPE>::put(allowed >> e & 1 ? v : -INFINITY);
  }
  if (left >= kPer) {
    *reinterpret_cast<Run<E> *>(y) = in;
  } else {
#pragma unroll
    for (int e = 0; e < kPer; e++)
      if (e < left) y[e] = in.v[e];
  }
}

template <int TYPE>
hipError_t launch(const AdjustLogits &a, hipStream_t s) {
  const int pieces = (a.vocab + kPiece - 1) / kPiece;
  hipLaunchKernelGGL(adjust_kernel<TYPE>, dim3((unsigned)((int64_t)a.rows * pieces)), dim3(kThreads), 0, s, a, pieces);
  return hipGetLastError();
}

}  // namespace

hipError_t adjust_logits(const AdjustLogits &a, int n_cu, hipStream_t s) {
  (void)n_cu;
  if (a.rows <= 0) return hipSuccess;
  switch (a.type) {
    case kOpF32: return launch<kOpF32>(a, s);
    case kOpBf16: return launch<kOpBf16>(a, s);
    case kOpF16: return launch<kOpF16>(a, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace itts
