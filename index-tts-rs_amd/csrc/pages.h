// Sequences and pages as the kernels find them (gfx950, wave64).
#pragma once

#include "kernels.h"

namespace itts {
namespace {

// Small tables that a kernel only reads, at an address all lanes share: through the scalar cache.
__device__ __forceinline__ int32_t uniform_load(const int32_t *p) {
  using Const = const __attribute__((address_space(4))) int32_t;
  return *(Const *)(uintptr_t)p;
}

// The sequence b that holds a token, the same in all lanes of the wave: the last one that starts at or in front of it, found
// 64 starts at a time; -1 for a token in front of the first sequence.  Empty sequences start where the next one does.
__device__ __forceinline__ int sequence_of(const int32_t *starts, int batch, int token) {
  const int lane = threadIdx.x & 63;
  int b = 0, n = batch;
  bool any = false;
  while (n > 1 || !any) {
    const int step = (n + 63) >> 6, at = lane * step;
    const uint64_t in = __ballot(at < n && starts[b + min(at, n - 1)] <= token);
    if (in == 0) return -1;
    const int i = 63 - __builtin_clzll(in);
    b += i * step, n = min(step, n - i * step), any = true;
  }
  return __builtin_amdgcn_readfirstlane(b);
}

// Tokens first .. first + n - 1 of a sequence; n = 0 for starts that do not rise or leave the tensors.
struct Span {
  int first, n;
};
__device__ __forceinline__ Span span_of(int start, int end, int tokens) {
  const bool ok = start >= 0 && end >= start && end <= tokens;
  return Span{ok ? start : 0, ok ? end - start : 0};
}

// The page of a row (rows < 2^24, pages of multiples of 16 rows) by a product: mul = ceil(2^32 / (size / 16)), exact for
// rows / 16 < 2^20 and sizes up to 2^16.
__host__ __device__ inline uint64_t page_mul(int size) { return ((1ull << 32) + size / 16 - 1) / (size / 16); }
__device__ __forceinline__ int page_of(int row, uint64_t mul) { return (int)(((uint64_t)(uint32_t)(row >> 4) * mul) >> 32); }

}  // namespace
}  // namespace itts
