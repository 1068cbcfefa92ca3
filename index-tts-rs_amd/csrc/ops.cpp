// The operators on device memory of include/itts_hip.h (drafted trees, paged caches, logits): argument
// checks and launches.  Nothing here allocates, waits or throws.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <array>
#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <initializer_list>

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

// Whether rows of `row` bytes at x and at multiples of a tensor's strides from there meet rows of another one at y.  The axis with
// the longest stride goes first, index by index (of an axis of both: difference by difference) as far as what is left
// can meet at all; more than a million steps count as meeting.
struct Rows {
  Axis axes[3];  // bytes; the longest stride last
  int n;
  int64_t reach;  // bytes from the first row's start to the last one's end
};
Rows rows_of(std::initializer_list<Axis> axes, int size, int64_t row) {
  Rows r{{}, 0, row};
  for (const Axis &x : axes)
    if (x.extent > 1 && x.stride > 0) r.axes[r.n++] = Axis{x.stride * size, x.extent}, r.reach += (x.extent - 1) * x.stride * size;
  std::sort(r.axes, r.axes + r.n, [](const Axis &x, const Axis &y) { return x.stride < y.stride; });
  return r;
}
bool rows_meet(int64_t apart, Rows a, Rows b, int *left) {  // apart: y - x
  if (apart >= a.reach || -apart >= b.reach) return false;
  if ((a.n == 0 && b.n == 0) || --*left < 0) return true;
  const int64_t in_a = a.n > 0 ? a.axes[a.n - 1].stride : 0, in_b = b.n > 0 ? b.axes[b.n - 1].stride : 0, step = std::max(in_a, in_b);
  int64_t low = 0, high = 0;  // apart + step * (low .. high)
  if (in_a == step) a.n--, low = 1 - a.axes[a.n].extent, a.reach -= (a.axes[a.n].extent - 1) * step;
  if (in_b == step) b.n--, high = b.axes[b.n].extent - 1, b.reach -= (b.axes[b.n].extent - 1) * step;
  // -b.reach < apart + step i < a.reach (one more at either end: quotients round towards 0)
  low = std::max(low, (-b.reach - apart) / step - 1), high = std::min(high, (a.reach - apart) / step + 1);
  for (int64_t i = low; i <= high; i++)
    if (rows_meet(apart + step * i, a, b, left)) return true;
  return false;
}
bool rows_meet(const void *x, const Rows &a, const void *y, const Rows &b) {
  int left = 1000000;
  return rows_meet(reinterpret_cast<intptr_t>(y) - reinterpret_cast<intptr_t>(x), a, b, &left);
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

constexpr int kMaxTokens = 1 << 20;

// A cache's pages; `writes`: rows are written, so none may share memory with another.
itts_status pages_args(const itts_pages &g, bool writes, Pages *o) {
  const int t = g.dtype == ITTS_I4 ? kOpI4 : op_type(g.dtype);
  if (t < 0) return fail(ITTS_E_VALIDATION, "pages.dtype: must be F32, BF16, F16 or I4");
  if (g.head_dim != 64 && g.head_dim != 128) return fail(ITTS_E_VALIDATION, "pages.head_dim: must be 64 or 128, got %d", g.head_dim);
  if (g.n_kv_head < 1 || g.n_kv_head > 1024) return fail(ITTS_E_VALIDATION, "pages.n_kv_head: must be in 1..=1024, got %d", g.n_kv_head);
  if (g.page_size < 16 || g.page_size > 65536 || g.page_size % 16)
    return fail(ITTS_E_VALIDATION, "pages.page_size: must be a multiple of 16 in 16..=65536, got %d", g.page_size);
  if (g.n_pages < 1) return fail(ITTS_E_VALIDATION, "pages.n_pages: must be >= 1, got %d", g.n_pages);
  if (!g.k || !g.v || (t == kOpI4 && (!g.k_params || !g.v_params))) return fail(ITTS_E_VALIDATION, "pages: k, v or their params: null");
  const int es = t == kOpI4 ? 1 : op_size(t), row = t == kOpI4 ? g.head_dim / 2 : g.head_dim;
  const int64_t ks[3] = {g.k_page, g.k_head, g.k_row}, vs[3] = {g.v_page, g.v_head, g.v_row};
  const int64_t kps[3] = {g.k_params_page, g.k_params_head, g.k_params_row}, vps[3] = {g.v_params_page, g.v_params_head, g.v_params_row};
  const int ext[3] = {g.n_pages, g.n_kv_head, g.page_size};
  const int pair_row = 2 * (g.head_dim / 64);  // float16 of a row's pairs
  for (int i = 0; i < 3; i++) {
    if (!row_stride(ks[i], ext[i], es) || !aligned16(g.k)) return fail(ITTS_E_VALIDATION, "pages.k: rows must start at multiples of 16 bytes");
    if (!row_stride(vs[i], ext[i], es) || !aligned16(g.v)) return fail(ITTS_E_VALIDATION, "pages.v: rows must start at multiples of 16 bytes");
    if (t != kOpI4 || ext[i] <= 1) continue;
    for (int64_t s : {kps[i], vps[i]})
      if (s < 0 || s > INT64_MAX / (16ll * ext[i]) || s % pair_row)
        return fail(ITTS_E_VALIDATION, "pages.k_params, v_params: rows must start at multiples of %d bytes", 2 * pair_row);
  }
  if (t == kOpI4 && (reinterpret_cast<uintptr_t>(g.k_params) % (2 * pair_row) || reinterpret_cast<uintptr_t>(g.v_params) % (2 * pair_row)))
    return fail(ITTS_E_VALIDATION, "pages.k_params, v_params: rows must start at multiples of %d bytes", 2 * pair_row);
  if (g.k_row * es > kTreeMaxRowBytes || g.v_row * es > kTreeMaxRowBytes ||
      (t == kOpI4 && (g.k_params_row * 2 > kTreeMaxRowBytes || g.v_params_row * 2 > kTreeMaxRowBytes)))
    return fail(ITTS_E_VALIDATION, "pages.k_row, v_row: rows must be at most %d bytes apart", kTreeMaxRowBytes);
  if (g.n_pages > 1 && (g.k_page * es > UINT32_MAX || g.v_page * es > UINT32_MAX ||
                        (t == kOpI4 && (g.k_params_page * 2 > UINT32_MAX || g.v_params_page * 2 > UINT32_MAX))))
    return fail(ITTS_E_VALIDATION, "pages.k_page, v_page: pages must be less than 2^32 bytes apart");
  if (writes) {
    auto rows = [&](const int64_t(&s)[3], int size, int n) { return rows_of({{s[0], ext[0]}, {s[1], ext[1]}, {s[2], ext[2]}}, size, (int64_t)n * size); };
    auto meet = [&](const int64_t(&a)[3], const int64_t(&b)[3], const void *x, const void *y, int size, int n) {
      return rows_overlap<3>({{{a[0], ext[0]}, {a[1], ext[1]}, {a[2], ext[2]}}}, n) || rows_overlap<3>({{{b[0], ext[0]}, {b[1], ext[1]}, {b[2], ext[2]}}}, n) ||
             rows_meet(x, rows(a, size, n), y, rows(b, size, n));
    };
    if (meet(ks, vs, g.k, g.v, es, row)) return fail(ITTS_E_VALIDATION, "pages.k, v: rows must not overlap");
    if (t == kOpI4) {
      if (meet(kps, vps, g.k_params, g.v_params, 2, pair_row)) return fail(ITTS_E_VALIDATION, "pages.k_params, v_params: rows must not overlap");
      const Rows k = rows(ks, es, row), v = rows(vs, es, row), kp = rows(kps, 2, pair_row), vp = rows(vps, 2, pair_row);
      if (rows_meet(g.k, k, g.k_params, kp) || rows_meet(g.k, k, g.v_params, vp) || rows_meet(g.v, v, g.k_params, kp) || rows_meet(g.v, v, g.v_params, vp))
        return fail(ITTS_E_VALIDATION, "pages.k, v: rows must not overlap those of k_params, v_params");
    }
  }
  *o = Pages{static_cast<char *>(g.k), static_cast<char *>(g.v), static_cast<char *>(g.k_params), static_cast<char *>(g.v_params),
             g.n_pages, g.page_size, g.n_kv_head, g.head_dim, t, ks[0] * es, ks[1] * es, ks[2] * es, vs[0] * es, vs[1] * es, vs[2] * es,
             kps[0] * 2, kps[1] * 2, kps[2] * 2, vps[0] * 2, vps[1] * 2, vps[2] * 2};
  return ITTS_OK;
}
// The type of tensors beside the pages.
bool goes_with(int type, int pages) { return type >= 0 && (type == pages || pages == kOpI4 || (type == kOpF32 && pages == kOpBf16)); }
itts_status batch_args(int batch, int tokens, int n_table, int64_t table_batch, bool ragged) {
  if (batch < 0 || batch > kMaxGridYZ) return fail(ITTS_E_VALIDATION, "batch: must be in 0..=%d, got %d", kMaxGridYZ, batch);
  if (tokens < 0 || tokens > kMaxTokens) return fail(ITTS_E_VALIDATION, "n_tokens: must be in 0..=2^20, got %d", tokens);
  if (ragged && batch == 0 && tokens > 0) return fail(ITTS_E_VALIDATION, "batch: %d tokens of no sequence", tokens);
  if (n_table < 0 || (batch > 1 && (table_batch < 0 || table_batch > INT64_MAX / 16 / batch))) return fail(ITTS_E_VALIDATION, "table: negative size or stride");
  return ITTS_OK;
}
itts_status heads_args(int n_head, int n_kv_head) {
  if (n_head < 1 || n_head > 1024 || n_head % n_kv_head)
    return fail(ITTS_E_VALIDATION, "n_head: %d key heads do not divide %d query heads (1..=1024)", n_kv_head, n_head);
  return ITTS_OK;
}
// Rows [tokens][heads] of a tensor.
bool token_rows(const void *p, int64_t token, int64_t head, int tokens, int heads, int size) {
  return row_stride(token, tokens, size) && row_stride(head, heads, size) && aligned16(p);
}

// Whether rows [tokens][heads] are written to where others of their size are read without one meeting another's: all in the same
// places, or none.
bool in_place(const void *in, int64_t in_token, int64_t in_head, const void *out, int64_t out_token, int64_t out_head, int tokens, int heads,
              int size, int dim) {
  if (in == out && (tokens <= 1 || in_token == out_token) && (heads <= 1 || in_head == out_head)) return true;
  return tokens == 0 || !rows_meet(in, rows_of({{in_token, tokens}, {in_head, heads}}, size, dim * size), out,
                                   rows_of({{out_token, tokens}, {out_head, heads}}, size, dim * size));
}

itts_status append_args(const itts_paged_append_args *a, PagedAppend *o) {
  if (!a) return fail(ITTS_E_VALIDATION, "args: null");
  Pages g;
  if (itts_status st = batch_args(a->batch, a->n_tokens, a->n_table, a->table_batch, true)) return st;
  if (itts_status st = pages_args(a->pages, true, &g)) return st;
  if (a->n_head != 0)
    if (itts_status st = heads_args(a->n_head, g.Hk)) return st;
  const int t = op_type(a->dtype), n = a->n_tokens;
  if (!goes_with(t, g.type)) return fail(ITTS_E_VALIDATION, "dtype: must be the pages', F32 over BF16, or any over I4");
  const int es = op_size(t);
  if (!token_rows(a->k, a->k_token, a->k_head, n, g.Hk, es)) return fail(ITTS_E_VALIDATION, "k: rows must start at multiples of 16 bytes");
  if (!token_rows(a->v, a->v_token, a->v_head, n, g.Hk, es)) return fail(ITTS_E_VALIDATION, "v: rows must start at multiples of 16 bytes");
  if (a->n_head > 0) {
    if (!token_rows(a->q, a->q_token, a->q_head, n, a->n_head, es)) return fail(ITTS_E_VALIDATION, "q: rows must start at multiples of 16 bytes");
    if (!token_rows(a->q_out, a->q_out_token, a->q_out_head, n, a->n_head, es))
      return fail(ITTS_E_VALIDATION, "q_out: rows must start at multiples of 16 bytes");
    if (rows_overlap<2>({{{a->q_out_token, n}, {a->q_out_head, a->n_head}}}, g.D)) return fail(ITTS_E_VALIDATION, "q_out: rows must not overlap");
    if (!in_place(a->q, a->q_token, a->q_head, a->q_out, a->q_out_token, a->q_out_head, n, a->n_head, es, g.D))
      return fail(ITTS_E_VALIDATION, "q_out: may be q with the same strides, but must not share memory with it otherwise");
  }
  int rot = 0;
  if (a->rotation) {
    rot = a->n_rotated;
    if (rot < 16 || rot > g.D || rot % 16) return fail(ITTS_E_VALIDATION, "n_rotated: must be a multiple of 16 in 16..=%d, got %d", g.D, rot);
    // (positions that are not in the table read its first row)
    if (a->n_positions < 1) return fail(ITTS_E_VALIDATION, "n_positions: a rotation needs one at least, got %d", a->n_positions);
    if (!row_stride(a->rotation_row, a->n_positions, 4) || !aligned16(a->rotation))
      return fail(ITTS_E_VALIDATION, "rotation: rows must start at multiples of 16 bytes");
  }
  *o = PagedAppend{g, a->k, a->v, a->q, a->q_out, a->rotation, a->starts, a->lengths, a->table, a->positions, a->new_lengths, a->batch, n,
                   a->n_head, a->n_table, rot, a->rotation ? a->n_positions : 0, a->interleaved != 0, t, a->k_token, a->k_head, a->v_token,
                   a->v_head, a->q_token, a->q_head, a->q_out_token, a->q_out_head, a->rotation_row, a->table_batch};
  return ITTS_OK;
}

itts_status paged_args(const itts_paged_attention_args *a, PagedAttn *o) {
  if (!a) return fail(ITTS_E_VALIDATION, "args: null");
  Pages g;
  if (itts_status st = batch_args(a->batch, a->n_tokens, a->n_table, a->table_batch, true)) return st;
  if (itts_status st = pages_args(a->pages, false, &g)) return st;
  if (itts_status st = heads_args(a->n_head, g.Hk)) return st;
  if ((int64_t)a->n_tokens * a->n_head > 1 << 29) return fail(ITTS_E_VALIDATION, "n_tokens: at most 2^29 rows, got %d of %d heads", a->n_tokens, a->n_head);
  const int t = op_type(a->q_dtype), n = a->n_tokens;
  if (!goes_with(t, g.type)) return fail(ITTS_E_VALIDATION, "q_dtype: must be the pages', F32 over BF16, or any over I4");
  const int es = op_size(t);
  if (!token_rows(a->q, a->q_token, a->q_head, n, a->n_head, es)) return fail(ITTS_E_VALIDATION, "q: rows must start at multiples of 16 bytes");
  if (!token_rows(a->out, a->out_token, a->out_head, n, a->n_head, es)) return fail(ITTS_E_VALIDATION, "out: rows must start at multiples of 16 bytes");
  if (rows_overlap<2>({{{a->out_token, n}, {a->out_head, a->n_head}}}, g.D)) return fail(ITTS_E_VALIDATION, "out: rows must not overlap");
  if (!in_place(a->q, a->q_token, a->q_head, a->out, a->out_token, a->out_head, n, a->n_head, es, g.D))
    return fail(ITTS_E_VALIDATION, "out: may be q with the same strides, but must not share memory with it otherwise");
  if (a->max_rows < 0 || a->max_rows > (int64_t)a->n_table * g.size || a->max_rows > kPagesMaxRows)
    return fail(ITTS_E_VALIDATION, "max_rows: must be in 0..=%d pages of %d rows and at most 2^24, got %d", a->n_table, g.size, a->max_rows);
  if (a->window < 0 || a->sinks < 0) return fail(ITTS_E_VALIDATION, "window, sinks: must be >= 0, got %d and %d", a->window, a->sinks);
  if (!(a->scale - a->scale == 0.0f)) return fail(ITTS_E_VALIDATION, "scale: must be finite");
  // (longer than any sequence is as good as no bound, and leaves room for sums)
  constexpr int kFar = 2 * kPagesMaxRows;
  *o = PagedAttn{g, a->q, a->out, a->starts, a->lengths, a->table, a->batch, n, a->n_head, a->n_table, a->max_rows, t,
                 std::min(a->window, kFar), std::min(a->sinks, kFar), a->scale, a->q_token, a->q_head, a->out_token, a->out_head,
                 a->table_batch, nullptr};
  if (!paged_attn_fits(*o))
    return fail(ITTS_E_VALIDATION, "n_tokens: too many of %d sequences and %d key heads for one launch, got %d", a->batch, g.Hk, n);
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

itts_status itts_paged_append(const itts_paged_append_args *args, void *stream) {
  PagedAppend a;
  int dev = 0, n_cu = 0;
  if (itts_status st = append_args(args, &a)) return st;
  if (a.batch == 0) return ITTS_OK;
  if (!a.starts || !a.lengths || !a.new_lengths || (a.n_table && !a.table) || (a.tokens && (!a.k || !a.v || (a.H && (!a.q || !a.q_out)))))
    return fail(ITTS_E_VALIDATION, "k, v, q, q_out, starts, lengths, table, new_lengths: null");
  if (a.lengths == a.new_lengths) return fail(ITTS_E_VALIDATION, "new_lengths: must not be lengths");
  if (itts_status st = compute_units(&dev, &n_cu)) return st;
  const bool any = a.tokens > 0, turn = any && a.H > 0;
  if (itts_status st = check_device(
          dev, stream, {{a.pages.k, "pages.k"}, {a.pages.v, "pages.v"}, {a.pages.type == kOpI4 ? a.pages.kp : nullptr, "pages.k_params"},
                        {a.pages.type == kOpI4 ? a.pages.vp : nullptr, "pages.v_params"}, {any ? a.k : nullptr, "k"}, {any ? a.v : nullptr, "v"},
                        {turn ? a.q : nullptr, "q"}, {turn ? a.q_out : nullptr, "q_out"}, {a.rotation, "rotation"},
                        {a.starts, "starts"}, {a.lengths, "lengths"}, {a.n_table ? a.table : nullptr, "table"},
                        {any ? a.positions : nullptr, "positions"}, {a.new_lengths, "new_lengths"}}))
    return st;
  if (hipError_t e = paged_append(a, n_cu, static_cast<hipStream_t>(stream)); e != hipSuccess) return hip_fail(e, "paged append");
  return ITTS_OK;
}

itts_status itts_paged_attention_workspace(const itts_paged_attention_args *args, uint64_t *bytes) {
  PagedAttn a;
  int dev = 0, n_cu = 0;
  if (itts_status st = paged_args(args, &a)) return st;
  if (!bytes) return fail(ITTS_E_VALIDATION, "bytes: null");
  *bytes = 0;
  if (a.tokens == 0) return ITTS_OK;
  if (itts_status st = compute_units(&dev, &n_cu)) return st;
  *bytes = sizeof(float) * paged_attn_ws(a, n_cu);
  return ITTS_OK;
}

itts_status itts_paged_attention(const itts_paged_attention_args *args, void *workspace, uint64_t workspace_bytes, void *stream) {
  PagedAttn a;
  int dev = 0, n_cu = 0;
  if (itts_status st = paged_args(args, &a)) return st;
  if (a.tokens == 0) return ITTS_OK;
  if (!a.q || !a.out || !a.starts || !a.lengths || (a.n_table && !a.table)) return fail(ITTS_E_VALIDATION, "q, out, starts, lengths, table: null");
  if (itts_status st = compute_units(&dev, &n_cu)) return st;
  const uint64_t need = sizeof(float) * paged_attn_ws(a, n_cu);
  if (itts_status st = check_workspace(workspace, workspace_bytes, need)) return st;
  if (itts_status st = check_device(
          dev, stream, {{a.pages.k, "pages.k"}, {a.pages.v, "pages.v"}, {a.pages.type == kOpI4 ? a.pages.kp : nullptr, "pages.k_params"},
                        {a.pages.type == kOpI4 ? a.pages.vp : nullptr, "pages.v_params"}, {a.q, "q"}, {a.out, "out"}, {a.starts, "starts"},
                        {a.lengths, "lengths"}, {a.n_table ? a.table : nullptr, "table"}, {need ? workspace : nullptr, "workspace"}}))
    return st;
  a.part = static_cast<float *>(workspace);
  if (hipError_t e = paged_attn(a, n_cu, static_cast<hipStream_t>(stream)); e != hipSuccess) return hip_fail(e, "paged attention");
  return ITTS_OK;
}

itts_status itts_paged_gather(const itts_paged_gather_args *a, void *stream) {
  if (!a) return fail(ITTS_E_VALIDATION, "args: null");
  Pages g;
  if (itts_status st = batch_args(a->batch, 0, a->n_table, a->table_batch, false)) return st;
  if (itts_status st = pages_args(a->pages, false, &g)) return st;
  if (a->n_rows < 0 || a->n_rows > kPagesMaxRows) return fail(ITTS_E_VALIDATION, "n_rows: must be in 0..=2^24, got %d", a->n_rows);
  const int t = op_type(a->dtype);
  if (t < 0 || (t != g.type && g.type != kOpI4)) return fail(ITTS_E_VALIDATION, "dtype: must be the pages', or any over I4");
  const int es = op_size(t);
  const int64_t ks[3] = {a->k_batch, a->k_head, a->k_row}, vs[3] = {a->v_batch, a->v_head, a->v_row};
  const int ext[3] = {a->batch, g.Hk, a->n_rows};
  for (int i = 0; i < 3; i++) {
    if (!row_stride(ks[i], ext[i], es) || !aligned16(a->k)) return fail(ITTS_E_VALIDATION, "k: rows must start at multiples of 16 bytes");
    if (!row_stride(vs[i], ext[i], es) || !aligned16(a->v)) return fail(ITTS_E_VALIDATION, "v: rows must start at multiples of 16 bytes");
  }
  if (a->batch == 0 || a->n_rows == 0) return ITTS_OK;
  if (!a->k || !a->v || !a->lengths || (a->n_table && !a->table)) return fail(ITTS_E_VALIDATION, "k, v, lengths, table: null");
  auto rows = [&](const int64_t(&s)[3]) { return rows_of({{s[0], ext[0]}, {s[1], ext[1]}, {s[2], ext[2]}}, es, g.D * es); };
  if (rows_overlap<3>({{{ks[0], ext[0]}, {ks[1], ext[1]}, {ks[2], ext[2]}}}, g.D) ||
      rows_overlap<3>({{{vs[0], ext[0]}, {vs[1], ext[1]}, {vs[2], ext[2]}}}, g.D) || rows_meet(a->k, rows(ks), a->v, rows(vs)))
    return fail(ITTS_E_VALIDATION, "k, v: rows must not overlap");
  int dev = 0, n_cu = 0;
  if (itts_status st = compute_units(&dev, &n_cu)) return st;
  if (itts_status st = check_device(
          dev, stream, {{g.k, "pages.k"}, {g.v, "pages.v"}, {g.type == kOpI4 ? g.kp : nullptr, "pages.k_params"},
                        {g.type == kOpI4 ? g.vp : nullptr, "pages.v_params"}, {a->k, "k"}, {a->v, "v"}, {a->lengths, "lengths"},
                        {a->n_table ? a->table : nullptr, "table"}}))
    return st;
  const PagedGather p{g, a->k, a->v, a->lengths, a->table, a->batch, a->n_rows, a->n_table, t, ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
                      a->table_batch};
  if (hipError_t e = paged_gather(p, static_cast<hipStream_t>(stream)); e != hipSuccess) return hip_fail(e, "paged gather");
  return ITTS_OK;
}

itts_status itts_adjust_logits(const itts_adjust_logits_args *a, void *stream) {
  if (!a) return fail(ITTS_E_VALIDATION, "args: null");
  if (a->rows < 0 || a->rows > 1 << 23) return fail(ITTS_E_VALIDATION, "rows: must be in 0..=2^23, got %d", a->rows);
  if (a->vocab < 1 || a->vocab > 1 << 24) return fail(ITTS_E_VALIDATION, "vocab: must be in 1..=2^24, got %d", a->vocab);
  if (!adjust_logits_fits(a->rows, a->vocab)) return fail(ITTS_E_VALIDATION, "rows: too many of %d logits, got %d", a->vocab, a->rows);
  if (a->n_history < 0 || a->n_history > kAdjustMaxList) return fail(ITTS_E_VALIDATION, "n_history: must be in 0..=%d, got %d", kAdjustMaxList, a->n_history);
  if (a->n_bias < 0 || a->n_bias > kAdjustMaxList) return fail(ITTS_E_VALIDATION, "n_bias: must be in 0..=%d, got %d", kAdjustMaxList, a->n_bias);
  const int t = op_type(a->dtype);
  if (t < 0) return fail(ITTS_E_VALIDATION, "dtype: must be F32, BF16 or F16");
  if (!a->repetition && !(a->repetition_all > 0.0f && a->repetition_all - a->repetition_all == 0.0f))
    return fail(ITTS_E_VALIDATION, "repetition: must be above 0 and finite");
  if ((!a->frequency && !(a->frequency_all - a->frequency_all == 0.0f)) || (!a->presence && !(a->presence_all - a->presence_all == 0.0f)))
    return fail(ITTS_E_VALIDATION, "frequency, presence: must be finite");
  if (reinterpret_cast<uintptr_t>(a->logits) % op_size(t) || reinterpret_cast<uintptr_t>(a->out) % op_size(t))
    return fail(ITTS_E_VALIDATION, "logits, out: misaligned");
  if (a->rows > 1) {
    for (int64_t s : {a->logits_row, a->out_row, a->history_row, a->bias_tokens_row, a->bias_row, a->allowed_row})
      if (s < 0 || s > INT64_MAX / 16 / a->rows) return fail(ITTS_E_VALIDATION, "logits_row, out_row, history_row, bias_row, allowed_row: rows must ascend");
    if (a->out_row < a->vocab) return fail(ITTS_E_VALIDATION, "out: rows must not overlap");
  }
  if (a->rows == 0) return ITTS_OK;
  if (!a->logits || !a->out || (a->n_history && !a->history) || (a->n_bias && (!a->bias_tokens || !a->bias)))
    return fail(ITTS_E_VALIDATION, "logits, out, history, bias_tokens, bias: null");
  // (a block reads what it has not written yet: its own tokens)
  const int es = op_size(t);
  if (!(a->logits == a->out && (a->rows == 1 || a->logits_row == a->out_row)) &&
      rows_meet(a->logits, rows_of({{a->logits_row, a->rows}}, es, (int64_t)a->vocab * es), a->out, rows_of({{a->out_row, a->rows}}, es, (int64_t)a->vocab * es)))
    return fail(ITTS_E_VALIDATION, "out: may be logits with the same stride, but must not share memory with them otherwise");
  int dev = 0, n_cu = 0;
  if (itts_status st = compute_units(&dev, &n_cu)) return st;
  if (itts_status st = check_device(
          dev, stream, {{a->logits, "logits"}, {a->out, "out"}, {a->n_history ? a->history : nullptr, "history"},
                        {a->n_bias ? a->bias_tokens : nullptr, "bias_tokens"}, {a->n_bias ? a->bias : nullptr, "bias"}, {a->allowed, "allowed"},
                        {a->repetition, "repetition"}, {a->frequency, "frequency"}, {a->presence, "presence"}}))
    return st;
  const AdjustLogits p{a->logits, a->out, a->history, a->bias_tokens, a->bias, a->allowed, a->repetition, a->frequency, a->presence,
                       a->repetition_all, a->frequency_all, a->presence_all, a->rows, a->vocab, a->n_history, a->n_bias, t, a->logits_row,
                       a->out_row, a->history_row, a->bias_tokens_row, a->bias_row, a->allowed_row};
  if (hipError_t e = adjust_logits(p, n_cu, static_cast<hipStream_t>(stream)); e != hipSuccess) return hip_fail(e, "adjusted logits");
  return ITTS_OK;
}

}  // extern "C"
