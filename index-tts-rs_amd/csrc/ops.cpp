// The operators on device memory of include/itts_hip.h (decoding with drafted trees): argument
// checks and launches.  Nothing here allocates, waits or throws.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <array>
#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>

#include "../../include/itts_hip.h"
#include "kernels.h"

namespace itts {
itts_status set_error_text(itts_status st, const char *msg);  // runtime.cpp
}

namespace {

using namespace itts;

itts_status fail(itts_status st, const char *fmt, ...) {
  char buf[256];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  return set_error_text(st, buf);
}
itts_status hip_fail(hipError_t e, const char *what) {
  (void)hipGetLastError();  // reported here, not by the program's next HIP call
  return fail(ITTS_E_DEVICE, "HIP error %s: %s", hipGetErrorName(e), what);
}

constexpr int kMaxGridYZ = 65535;

int op_type(itts_dtype t) { return t == ITTS_F32 ? kOpF32 : t == ITTS_BF16 ? kOpBf16 : t == ITTS_F16 ? kOpF16 : -1; }
int op_size(int t) { return t == kOpF32 ? 4 : 2; }

// Compute units of the current device (read once a device).
itts_status compute_units(int *dev, int *n_cu) {
  static std::atomic<int> known[kMaxDevices];
  if (hipError_t e = hipGetDevice(dev); e != hipSuccess) return hip_fail(e, "no device");
  if (*dev < 0 || *dev >= kMaxDevices) return fail(ITTS_E_DEVICE, "device %d: out of range", *dev);
  int n = known[*dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (hipError_t e = hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, *dev); e != hipSuccess)
      return hip_fail(e, "compute units");
    known[*dev].store(n, std::memory_order_relaxed);
  }
  *n_cu = n;
  return ITTS_OK;
}

// Whether the stream and the pointers belong to the current device: a host pointer, or memory of
// another device, would fault in the kernel.
struct NamedPtr {
  const void *p;
  const char *name;
};
template <int N>
itts_status check_device(int dev, void *stream, const NamedPtr (&ps)[N]) {
  if (stream) {
    hipDevice_t sd = -1;
    if (hipError_t e = hipStreamGetDevice(static_cast<hipStream_t>(stream), &sd); e != hipSuccess)
      return hip_fail(e, "stream");
    if (sd != dev) return fail(ITTS_E_VALIDATION, "stream: belongs to device %d, the current one is %d", (int)sd, dev);
  }
  for (const NamedPtr &q : ps) {
    if (!q.p) continue;
    hipPointerAttribute_t at{};
    if (hipPointerGetAttributes(&at, q.p) != hipSuccess) {
      (void)hipGetLastError();
      return fail(ITTS_E_VALIDATION, "%s: not device memory", q.name);
    }
    if (at.type != hipMemoryTypeDevice && at.type != hipMemoryTypeManaged)
      return fail(ITTS_E_VALIDATION, "%s: not device memory", q.name);
    if (at.type == hipMemoryTypeDevice && at.device != dev)
      return fail(ITTS_E_VALIDATION, "%s: memory of device %d, the current one is %d", q.name, at.device, dev);
  }
  return ITTS_OK;
}

bool aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
// A stride between rows that start at multiples of 16 bytes (of no account along an axis of one).
bool row_stride(int64_t stride, int extent, int size) {
  return extent <= 1 || (stride >= 0 && stride <= INT64_MAX / (16ll * extent) && stride * size % 16 == 0);
}

// Whether two rows of `row` elements share one, rows starting wherever multiples of the axes' strides add up to.
// Strides that each step over all that the smaller ones reach keep rows apart.  Others may (0, 2 | 0, 3): then
// differences of two rows' indices are tried, all axes but the longest one, which follows from the others; more
// than a million of them count as an overlap.
struct Axis {
  int64_t stride, extent;
};
template <int N>
bool rows_overlap(std::array<Axis, N> axes, int64_t row) {
  std::sort(axes.begin(), axes.end(), [](const Axis &x, const Axis &y) { return x.extent <= 1 ? y.extent > 1 : y.extent > 1 && x.stride < y.stride; });
  int64_t span = row;
  bool nested = true;
  for (const Axis &x : axes) {
    if (x.extent <= 1) continue;
    if (x.stride < row) return true;
    nested = nested && x.stride >= span;
    span += (x.extent - 1) * x.stride;
  }
  if (nested) return false;
  std::sort(axes.begin(), axes.end(), [](const Axis &x, const Axis &y) { return x.extent < y.extent; });
  double tries = 1;
  for (int i = 0; i + 1 < N; i++) tries *= 2.0 * std::max<int64_t>(1, axes[i].extent) - 1;
  if (tries > 1e6) return true;
  const Axis last = axes[N - 1];
  int64_t d[N] = {};
  for (int i = 0; i + 1 < N; i++) d[i] = 1 - std::max<int64_t>(1, axes[i].extent);
  for (;;) {
    int64_t at = 0;
    bool zero = true;
    for (int i = 0; i + 1 < N; i++) at += d[i] * axes[i].stride, zero = zero && d[i] == 0;
    const int64_t near = -at / last.stride;
    for (int64_t e = near - 1; e <= near + 1; e++) {
      const int64_t apart = at + e * last.stride;
      if (e > -last.extent && e < last.extent && apart > -row && apart < row && !(zero && e == 0)) return true;
    }
    int i = 0;
    while (i + 1 < N && d[i] + 1 >= std::max<int64_t>(1, axes[i].extent)) d[i] = 1 - std::max<int64_t>(1, axes[i].extent), i++;
    if (i + 1 >= N) return false;
    d[i]++;
  }
}

itts_status tree_args(const itts_tree_attention_args *a, TreeAttn *o) {
  if (!a) return fail(ITTS_E_VALIDATION, "args: null");
  if (a->batch < 0 || a->batch > kMaxGridYZ) return fail(ITTS_E_VALIDATION, "batch: must be in 0..=%d, got %d", kMaxGridYZ, a->batch);
  if (a->n_nodes < 0 || a->n_nodes > kTreeMaxNodes)
    return fail(ITTS_E_VALIDATION, "n_nodes: must be in 0..=%d, got %d", kTreeMaxNodes, a->n_nodes);
  if (a->n_head < 1 || a->n_head > 1024 || a->n_kv_head < 1 || a->n_head % a->n_kv_head != 0)
    return fail(ITTS_E_VALIDATION, "n_kv_head: %d key heads do not divide %d query heads (1..=1024)", a->n_kv_head, a->n_head);
  if (a->head_dim != 64 && a->head_dim != 128)
    return fail(ITTS_E_VALIDATION, "head_dim: must be 64 or 128, got %d", a->head_dim);
  if (a->max_seq < 1 || a->max_seq > 1 << 30)
    return fail(ITTS_E_VALIDATION, "max_seq: must be in 1..=2^30, got %d", a->max_seq);
  if (!(a->scale - a->scale == 0.0f)) return fail(ITTS_E_VALIDATION, "scale: must be finite");
  const int qt = op_type(a->q_dtype), kvt = op_type(a->kv_dtype);
  if (qt < 0 || kvt < 0 || !(qt == kvt || (qt == kOpF32 && kvt == kOpBf16)))
    return fail(ITTS_E_VALIDATION, "kv_dtype: queries and caches must be of one type (F32, BF16, F16), or F32 and BF16");
  const int qs = op_size(qt), ks = op_size(kvt), b = a->batch, n = a->n_nodes, h = a->n_head, hk = a->n_kv_head;
  if (!row_stride(a->q_batch, b, qs) || !row_stride(a->q_node, n, qs) || !row_stride(a->q_head, h, qs) || !aligned16(a->q))
    return fail(ITTS_E_VALIDATION, "q: rows must start at multiples of 16 bytes");
  if (!row_stride(a->out_batch, b, qs) || !row_stride(a->out_node, n, qs) || !row_stride(a->out_head, h, qs) || !aligned16(a->out))
    return fail(ITTS_E_VALIDATION, "out: rows must start at multiples of 16 bytes");
  if (rows_overlap<3>({{{a->out_batch, b}, {a->out_node, n}, {a->out_head, h}}}, a->head_dim))
    return fail(ITTS_E_VALIDATION, "out: rows must not overlap");
  if (!row_stride(a->k_batch, b, ks) || !row_stride(a->k_head, hk, ks) || !row_stride(a->k_row, a->max_seq, ks) || !aligned16(a->k))
    return fail(ITTS_E_VALIDATION, "k: rows must start at multiples of 16 bytes");
  if (!row_stride(a->v_batch, b, ks) || !row_stride(a->v_head, hk, ks) || !row_stride(a->v_row, a->max_seq, ks) || !aligned16(a->v))
    return fail(ITTS_E_VALIDATION, "v: rows must start at multiples of 16 bytes");
  if (a->max_seq > 1 && (a->k_row * ks > kTreeMaxRowBytes || a->v_row * ks > kTreeMaxRowBytes))
    return fail(ITTS_E_VALIDATION, "k_row, v_row: rows must be at most %d bytes apart", kTreeMaxRowBytes);
  if (b > 1 && a->parents_batch < 0) return fail(ITTS_E_VALIDATION, "parents: negative stride");
  *o = TreeAttn{a->q, a->k, a->v, a->out, a->lengths, a->parents, b, n, h, hk, a->head_dim, a->max_seq, qt, kvt, a->scale,
                a->q_batch, a->q_node, a->q_head, a->out_batch, a->out_node, a->out_head, a->k_batch, a->k_head, a->k_row,
                a->v_batch, a->v_head, a->v_row, a->parents_batch, nullptr};
  return ITTS_OK;
}

itts_status scores_args(const itts_token_scores_args *a, TokenScores *o) {
  if (!a) return fail(ITTS_E_VALIDATION, "args: null");
  if (a->rows < 0 || a->rows > 1 << 23) return fail(ITTS_E_VALIDATION, "rows: must be in 0..=2^23, got %d", a->rows);
  if (a->vocab < 1 || a->vocab > 1 << 24) return fail(ITTS_E_VALIDATION, "vocab: must be in 1..=2^24, got %d", a->vocab);
  if (a->n_tokens < 0) return fail(ITTS_E_VALIDATION, "n_tokens: must be >= 0, got %d", a->n_tokens);
  if (a->top_n < 0 || a->top_n > kScoresMaxTop || a->top_n > a->vocab)
    return fail(ITTS_E_VALIDATION, "top_n: must be in 0..=%d and at most the vocabulary of %d, got %d", kScoresMaxTop, a->vocab, a->top_n);
  const int t = op_type(a->dtype);
  if (t < 0) return fail(ITTS_E_VALIDATION, "dtype: must be F32, BF16 or F16");
  if (reinterpret_cast<uintptr_t>(a->logits) % op_size(t)) return fail(ITTS_E_VALIDATION, "logits: misaligned");
  if (a->rows > 1 && (a->logits_row < 0 || a->logits_row > INT64_MAX / 4 / a->rows || a->tokens_row < 0 || a->tokens_row > INT64_MAX / 4 / a->rows))
    return fail(ITTS_E_VALIDATION, "logits_row: rows must ascend");
  *o = TokenScores{a->logits, a->tokens, a->log_probs, a->entropy, a->top_tokens, a->top_log_probs, a->rows, a->vocab,
                   a->n_tokens, a->top_n, t, a->logits_row, a->tokens_row, nullptr};
  return ITTS_OK;
}

itts_status check_workspace(const void *ws, uint64_t have, uint64_t need) {
  if (need && (!ws || have < need))
    return fail(ITTS_E_VALIDATION, "workspace: %llu bytes needed, got %llu", (unsigned long long)need,
                (unsigned long long)(ws ? have : 0));
  if (need && !aligned16(ws)) return fail(ITTS_E_VALIDATION, "workspace: must start at a multiple of 16 bytes");
  return ITTS_OK;
}

}  // namespace

extern "C" {

itts_status itts_tree_attention_workspace(const itts_tree_attention_args *args, uint64_t *bytes) {
  TreeAttn a;
  int dev = 0, n_cu = 0;
  if (itts_status st = tree_args(args, &a)) return st;
  if (!bytes) return fail(ITTS_E_VALIDATION, "bytes: null");
  *bytes = 0;
  if (a.batch == 0 || a.n == 0) return ITTS_OK;
  if (itts_status st = compute_units(&dev, &n_cu)) return st;
  *bytes = sizeof(float) * tree_attn_ws(a, n_cu);
  return ITTS_OK;
}

itts_status itts_tree_attention(const itts_tree_attention_args *args, void *workspace, uint64_t workspace_bytes,
                                void *stream) {
  TreeAttn a;
  int dev = 0, n_cu = 0;
  if (itts_status st = tree_args(args, &a)) return st;
  if (a.batch == 0 || a.n == 0) return ITTS_OK;
  if (!a.q || !a.k || !a.v || !a.out || !a.lengths || !a.parents) return fail(ITTS_E_VALIDATION, "q, k, v, out, lengths, parents: null");
  if (itts_status st = compute_units(&dev, &n_cu)) return st;
  const uint64_t need = sizeof(float) * tree_attn_ws(a, n_cu);
  if (itts_status st = check_workspace(workspace, workspace_bytes, need)) return st;
  if (itts_status st = check_device(dev, stream, {{a.q, "q"}, {a.k, "k"}, {a.v, "v"}, {a.out, "out"}, {a.lengths, "lengths"},
                                                  {a.parents, "parents"}, {need ? workspace : nullptr, "workspace"}}))
    return st;
  a.part = static_cast<float *>(workspace);
  if (hipError_t e = tree_attn(a, n_cu, static_cast<hipStream_t>(stream)); e != hipSuccess) return hip_fail(e, "tree attention");
  return ITTS_OK;
}

itts_status itts_token_scores_workspace(const itts_token_scores_args *args, uint64_t *bytes) {
  TokenScores a;
  int dev = 0, n_cu = 0;
  if (itts_status st = scores_args(args, &a)) return st;
  if (!bytes) return fail(ITTS_E_VALIDATION, "bytes: null");
  *bytes = 0;
  if (a.rows == 0) return ITTS_OK;
  if (itts_status st = compute_units(&dev, &n_cu)) return st;
  *bytes = token_scores_ws(a, n_cu);
  return ITTS_OK;
}

itts_status itts_token_scores(const itts_token_scores_args *args, void *workspace, uint64_t workspace_bytes, void *stream) {
  TokenScores a;
  int dev = 0, n_cu = 0;
  if (itts_status st = scores_args(args, &a)) return st;
  if (a.rows == 0) return ITTS_OK;
  if (!a.x || (a.given && (!a.tokens || !a.log_probs)) || (a.top && (!a.top_tokens || !a.top_log_probs)))
    return fail(ITTS_E_VALIDATION, "logits, tokens, log_probs, top_tokens, top_log_probs: null");
  if (itts_status st = compute_units(&dev, &n_cu)) return st;
  const uint64_t need = token_scores_ws(a, n_cu);
  if (itts_status st = check_workspace(workspace, workspace_bytes, need)) return st;
  if (itts_status st = check_device(
          dev, stream, {{a.x, "logits"}, {a.given ? a.tokens : nullptr, "tokens"}, {a.given ? a.log_probs : nullptr, "log_probs"},
                        {a.entropy, "entropy"}, {a.top ? a.top_tokens : nullptr, "top_tokens"},
                        {a.top ? a.top_log_probs : nullptr, "top_log_probs"}, {need ? workspace : nullptr, "workspace"}}))
    return st;
  a.ws = workspace;
  if (hipError_t e = token_scores(a, n_cu, static_cast<hipStream_t>(stream)); e != hipSuccess) return hip_fail(e, "token scores");
  return ITTS_OK;
}

itts_status itts_cache_keep(const itts_cache_keep_args *a, void *stream) {
  if (!a) return fail(ITTS_E_VALIDATION, "args: null");
  if (a->batch < 0 || a->batch > kMaxGridYZ) return fail(ITTS_E_VALIDATION, "batch: must be in 0..=%d, got %d", kMaxGridYZ, a->batch);
  if (a->n_layer < 0 || a->n_head < 0 || a->max_seq < 1 || a->head_dim < 1 || a->n_path < 0)
    return fail(ITTS_E_VALIDATION, "n_layer, n_head, max_seq, head_dim, n_path: must not be negative, nor 0 for a row");
  const int t = op_type(a->dtype);
  if (t < 0) return fail(ITTS_E_VALIDATION, "dtype: must be F32, BF16 or F16");
  const int es = op_size(t);
  if ((int64_t)a->head_dim * es % 16 != 0) return fail(ITTS_E_VALIDATION, "head_dim: rows must be multiples of 16 bytes");
  const int64_t items = (int64_t)a->head_dim * es / 16 * 2;
  if ((double)items * a->n_layer * a->n_head > 4e9) return fail(ITTS_E_VALIDATION, "n_layer: caches too large");
  const int64_t ks[4] = {a->k_layer, a->k_batch, a->k_head, a->k_row}, vs[4] = {a->v_layer, a->v_batch, a->v_head, a->v_row};
  const int ext[4] = {a->n_layer, a->batch, a->n_head, a->max_seq};
  for (int i = 0; i < 4; i++) {
    if (!row_stride(ks[i], ext[i], es) || !aligned16(a->k)) return fail(ITTS_E_VALIDATION, "k: rows must start at multiples of 16 bytes");
    if (!row_stride(vs[i], ext[i], es) || !aligned16(a->v)) return fail(ITTS_E_VALIDATION, "v: rows must start at multiples of 16 bytes");
  }
  if (a->batch > 1 && a->path_batch < 0) return fail(ITTS_E_VALIDATION, "path: negative stride");
  if (a->batch == 0) return ITTS_OK;
  if (!a->lengths || !a->new_lengths || (a->n_path && !a->path) || ((int64_t)a->n_layer * a->n_head && (!a->k || !a->v)))
    return fail(ITTS_E_VALIDATION, "k, v, lengths, path, new_lengths: null");
  if (a->lengths == a->new_lengths) return fail(ITTS_E_VALIDATION, "new_lengths: must not be lengths");
  // Keys and values apart are one more axis where their strides are the same.
  bool alike = true;
  for (int i = 0; i < 4; i++) alike = alike && (ext[i] <= 1 || ks[i] == vs[i]);
  const int64_t from_k = std::llabs(reinterpret_cast<intptr_t>(a->v) - reinterpret_cast<intptr_t>(a->k)) / es;
  const bool rows = a->n_layer > 0 && a->n_head > 0;
  if (rows && (rows_overlap<4>({{{ks[0], ext[0]}, {ks[1], ext[1]}, {ks[2], ext[2]}, {ks[3], ext[3]}}}, a->head_dim) ||
               rows_overlap<4>({{{vs[0], ext[0]}, {vs[1], ext[1]}, {vs[2], ext[2]}, {vs[3], ext[3]}}}, a->head_dim) ||
               (alike && from_k > 0 && from_k < INT64_MAX / 16 &&
                rows_overlap<5>({{{ks[0], ext[0]}, {ks[1], ext[1]}, {ks[2], ext[2]}, {ks[3], ext[3]}, {from_k, 2}}}, a->head_dim))))
    return fail(ITTS_E_VALIDATION, "k, v: rows must not overlap");
  // One memory for both moves once: two would read rows that the other has moved.
  const bool same = a->k == a->v && rows;
  if (same && !alike) return fail(ITTS_E_VALIDATION, "k, v: rows must not overlap");
  int dev = 0, n_cu = 0;
  if (itts_status st = compute_units(&dev, &n_cu)) return st;
  if (itts_status st = check_device(dev, stream, {{a->k, "k"}, {a->v, "v"}, {a->lengths, "lengths"}, {a->n_path ? a->path : nullptr, "path"},
                                                  {a->new_lengths, "new_lengths"}}))
    return st;
  const int per = 16 / es;
  const CacheKeep c{a->k, a->v, a->lengths, a->path, a->new_lengths, a->n_layer, a->batch, a->n_head, a->max_seq,
                    a->head_dim / per, a->n_path, ks[0] / per, ks[1] / per, ks[2] / per, ks[3] / per, vs[0] / per, vs[1] / per,
                    vs[2] / per, vs[3] / per, a->path_batch, same ? 1 : 2};
  if (hipError_t e = cache_keep(c, static_cast<hipStream_t>(stream)); e != hipSuccess) return hip_fail(e, "kept rows");
  return ITTS_OK;
}

}  // extern "C"
