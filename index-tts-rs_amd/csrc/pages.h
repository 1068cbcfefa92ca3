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

// Tokens first .. first + n - 1 of a sequence; n = 0 for starts that do not rise or leave the tensors.
struct Span {
  int first, n;
};
__device__ __forceinline__ Span span_of(int start, int end, int tokens) {
  const bool ok = start >= 0 && end >= start && end <= tokens;
  return Span{ok ? start : 0, ok ? end - start : 0};
}

// What a search over more than 64 sequences found on its way.  A sequence has two keys, its first token (x) and another (y); of each
// level those it went by (the largest), and those of the lanes behind them.
struct Way {
  int b0, n;  // the sequences left, 64 at most; n = 0: the place lies in front of them all
  int2 own, later[2];
  // Whether all places from `first` to `last` lead here too: they lead to rising sequences, whatever the keys are.
  __device__ __forceinline__ bool leads_x(int first, int last) const {
    return own.x <= first && __ballot(later[0].x <= last || later[1].x <= last) == 0;
  }
  __device__ __forceinline__ bool leads_y(int first, int last) const {
    return own.y <= first && __ballot(later[0].y <= last || later[1].y <= last) == 0;
  }
};
// The group of sequences that a place leads to: at each of two levels at most the last of 64 whose key (BY_Y: y) is not above it.
template <bool BY_Y, class F>
__device__ __forceinline__ Way way_to(int batch, int place, F keys) {
  constexpr int kMost = 0x7fffffff;
  const int lane = threadIdx.x & 63;
  Way w{0, batch, make_int2(-kMost, -kMost), {make_int2(kMost, kMost), make_int2(kMost, kMost)}};
#pragma unroll
  for (int level = 0; level < 2; level++) {  // (65,535 sequences: groups of 1,024, of 16)
    if (w.n <= 64) break;
    const int step = (w.n + 63) >> 6;
    const int2 k = lane * step < w.n ? keys(w.b0 + lane * step) : make_int2(kMost, kMost);
    const uint64_t in = __ballot((BY_Y ? k.y : k.x) <= place);
    if (in == 0) {
      w.n = 0;
      break;
    }
    const int i = 63 - __builtin_clzll(in);
    w.own.x = max(w.own.x, __builtin_amdgcn_readlane(k.x, i)), w.own.y = max(w.own.y, __builtin_amdgcn_readlane(k.y, i));
    w.later[level] = lane > i ? k : make_int2(kMost, kMost);
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
  const Way w = way_to<false>(batch, token, [&](int b) { return make_int2(starts[b], 0); });
  const bool in = lane < w.n;
  const int start = in ? starts[w.b0 + lane] : 0, end = in ? starts[w.b0 + lane + 1] : 0;
  const bool has = start >= 0 && end > start && end <= tokens;
  const uint64_t holds = __ballot(has && start <= token && token < end);
  if (holds == 0) return Owner{-1, 0, 0};
  const int i = __builtin_ctzll(holds), first = __builtin_amdgcn_readlane(start, i), stop = __builtin_amdgcn_readlane(end, i);
  if (__ballot(has && lane < i && end > first) != 0 || !w.leads_x(first, stop - 1)) return Owner{-1, 0, 0};
  return Owner{w.b0 + i, first, stop - first};
}

// The page of a row (rows < 2^24, pages of multiples of 16 rows) by a product: mul = ceil(2^32 / (size / 16)), exact for
// rows / 16 < 2^20 and sizes up to 2^16.
__host__ __device__ inline uint64_t page_mul(int size) { return ((1ull << 32) + size / 16 - 1) / (size / 16); }
__device__ __forceinline__ int page_of(int row, uint64_t mul) { return (int)(((uint64_t)(uint32_t)(row >> 4) * mul) >> 32); }

}  // namespace
}  // namespace itts
