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

// What a search over more than 64 sequences found on its way: of each level the key it went by (the largest), and the keys of
// the lanes behind that.
struct Way {
  int b0, n;  // the sequences left, 64 at most; n = 0: `at` lies in front of them all
  int own, later[2];
  // whether every place from `first` to `last` leads here too: places lead to rising sequences, whatever the keys are
  __device__ __forceinline__ bool leads(int first, int last) const {
    return own <= first && __ballot(later[0] <= last || later[1] <= last) == 0;
  }
};
// The group of sequences that place `at` leads to: at each of two levels at most the last of 64 whose key is not above it.
template <class F>
__device__ __forceinline__ Way way_to(int batch, int at, F key) {
  const int lane = threadIdx.x & 63;
  Way w{0, batch, -0x7fffffff - 1, {0x7fffffff, 0x7fffffff}};
#pragma unroll
  for (int level = 0; level < 2; level++) {  // (65,535 sequences: groups of 1,024, of 16)
    if (w.n <= 64) break;
    const int step = (w.n + 63) >> 6, k = lane * step < w.n ? key(w.b0 + lane * step) : 0x7fffffff;
    const uint64_t in = __ballot(k <= at);
    if (in == 0) {
      w.n = 0;
      break;
    }
    const int i = 63 - __builtin_clzll(in);
    w.own = max(w.own, __builtin_amdgcn_readlane(k, i)), w.later[level] = lane > i ? k : 0x7fffffff;
    w.b0 = __builtin_amdgcn_readfirstlane(w.b0 + i * step), w.n = min(step, w.n - i * step);
  }
  return w;
}

// The sequence that holds a token, the same in all lanes of the wave; b = -1: none.  Starts should rise.  Where they do not, a
// sequence has its tokens, all of them, or none: not if its starts fall or leave the tensors, nor if it starts in
// front of where an earlier one ends.  Of more than 64 sequences those count that the token leads to, and a sequence has its
// tokens if all of them lead to it.
struct Owner {
  int b, first, n;
};
__device__ __forceinline__ Owner owner_of(const int32_t *starts, int batch, int tokens, int token) {
  const int lane = threadIdx.x & 63;
  const Way w = way_to(batch, token, [&](int b) { return starts[b]; });
  const bool in = lane < w.n;
  const int start = in ? starts[w.b0 + lane] : 0, end = in ? starts[w.b0 + lane + 1] : 0;
  const bool has = start >= 0 && end > start && end <= tokens;
  const uint64_t holds = __ballot(has && start <= token && token < end);
  if (holds == 0) return Owner{-1, 0, 0};
  const int i = __builtin_ctzll(holds), first = __builtin_amdgcn_readlane(start, i), stop = __builtin_amdgcn_readlane(end, i);
  if (__ballot(has && lane < i && end > first) != 0 || !w.leads(first, stop - 1)) return Owner{-1, 0, 0};
  return Owner{w.b0 + i, first, stop - first};
}

// The page of a row (rows < 2^24, pages of multiples of 16 rows) by a product: mul = ceil(2^32 / (size / 16)), exact for
// rows / 16 < 2^20 and sizes up to 2^16.
__host__ __device__ inline uint64_t page_mul(int size) { return ((1ull << 32) + size / 16 - 1) / (size / 16); }
__device__ __forceinline__ int page_of(int row, uint64_t mul) { return (int)(((uint64_t)(uint32_t)(row >> 4) * mul) >> 32); }

}  // namespace
}  // namespace itts
