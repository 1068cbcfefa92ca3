// Scores of rows of logits x [rows][vocab]: with m the row's maximum, c the number of tokens at m
// and s the sum of exp(x - m) over the others,
//   log p(t) = x_t - m - log(c + s),   entropy = log(c + s) - sum (x - m) exp(x - m) / (c + s).
// Keeping s apart from c makes log(c + s) = log1p(s) where one token has nearly all the
// probability, so that small entropies and log-probabilities near 0 keep their relative accuracy.
// Alternatives are ordered by (logit, lowest token first); NaN counts as -inf there.
#include "kernels.h"

namespace itts {
namespace {

constexpr int kThreads = 256;

template <int TYPE>
__device__ __forceinline__ float logit(const void *row, int i) {
  if constexpr (TYPE == kOpF32) return static_cast<const float *>(row)[i];
  else if constexpr (TYPE == kOpBf16) return bf16_bits_to_float(static_cast<const uint16_t *>(row)[i]);
  else return half_bits_to_float(static_cast<const uint16_t *>(row)[i]);
}

// (value, token) as one number that is larger for what comes first.
__device__ __forceinline__ uint64_t rank_key(float x, int token) {
  const uint32_t u = __float_as_uint(fmaxf(x, -INFINITY) + 0.0f);
  return (uint64_t)(u & 0x80000000u ? ~u : u | 0x80000000u) << 32 | (uint32_t)~token;
}

__device__ inline uint64_t block_max(uint64_t v, uint64_t *red) {
  for (int off = 32; off > 0; off >>= 1) {
    const uint64_t o = __shfl_xor((unsigned long long)v, off, 64);
    v = o > v ? o : v;
  }
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  for (int w = 0; w < kThreads / 64; w++) v = red[w] > v ? red[w] : v;
  __syncthreads();
  return v;
}

template <int TYPE>
__global__ __launch_bounds__(kThreads) void token_scores_kernel(TokenScores a) {
  __shared__ uint64_t red64[kThreads / 64];
  __shared__ float red[kThreads / 64];
  const int r = blockIdx.x;
  const void *x = static_cast<const char *>(a.x) + r * a.x_row * (TYPE == kOpF32 ? 4 : 2);
  uint64_t best = 0;
  for (int i = threadIdx.x; i < a.vocab; i += kThreads) best = max(best, rank_key(logit<TYPE>(x, i), i));
  best = block_max(best, red64);
  const float m = logit<TYPE>(x, (int)~(uint32_t)best);
  float cnt = 0.0f, s = 0.0f, sd = 0.0f;
  for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
    const float v = logit<TYPE>(x, i);
    const float d = v - m, p = expf(d);
    if (v == m) {
      cnt += 1.0f;
    } else {
      s += p;
      sd += p == 0.0f ? 0.0f : p * d;
    }
  }
  cnt = block_sum<kThreads>(cnt, red);
  s = block_sum<kThreads>(s, red);
  sd = block_sum<kThreads>(sd, red);
  const bool none = m == -INFINITY && s == 0.0f;  // every token is masked: probability 0 for all
  const float lz = m == INFINITY ? NAN : log1pf(s + (cnt - 1.0f));
  auto log_prob = [&](float v) { return none ? -INFINITY : (v - m) - lz; };
  if (threadIdx.x == 0 && a.entropy) a.entropy[r] = none ? 0.0f : lz - sd / (cnt + s);
  for (int i = threadIdx.x; i < a.given; i += kThreads) {
    const int t = a.tokens[r * a.tok_row + i];
    a.log_probs[(int64_t)r * a.given + i] = t == -1 ? 0.0f : t < 0 || t >= a.vocab ? NAN : log_prob(logit<TYPE>(x, t));
  }
  for (int k = 0; k < a.top; k++) {
    if (threadIdx.x == 0) {
      const int t = (int)~(uint32_t)best;
      a.top_tokens[(int64_t)r * a.top + k] = t;
      a.top_log_probs[(int64_t)r * a.top + k] = log_prob(logit<TYPE>(x, t));
    }
    uint64_t next = 0;
    for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
      const uint64_t key = rank_key(logit<TYPE>(x, i), i);
      if (key < best) next = max(next, key);
    }
    best = block_max(next, red64);
  }
}

}  // namespace

size_t token_scores_ws(const TokenScores &, int) { return 0; }

hipError_t token_scores(const TokenScores &a, int, hipStream_t s) {
  if (a.rows <= 0) return hipSuccess;
  if (a.top > kScoresMaxTop || a.top > a.vocab) return hipErrorInvalidValue;
  switch (a.type) {
    case kOpF32: hipLaunchKernelGGL(token_scores_kernel<kOpF32>, dim3(a.rows), dim3(kThreads), 0, s, a); break;
    case kOpBf16: hipLaunchKernelGGL(token_scores_kernel<kOpBf16>, dim3(a.rows), dim3(kThreads), 0, s, a); break;
    case kOpF16: hipLaunchKernelGGL(token_scores_kernel<kOpF16>, dim3(a.rows), dim3(kThreads), 0, s, a); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace itts
