"""The library's operators on device tensors: decoding with drafted trees, and over paged caches.

    tree_attention   attention of every node of a tree of drafted tokens over its sequence's
                     cached rows and its own ancestors (one node: a decode step)
    token_scores     log-probabilities of given tokens, entropy, the most probable tokens
    cache_keep       the accepted nodes' key and value rows moved up in the caches
    paged_cache      memory for pages of keys and values, of 32 bits, 16 or 4 (PagedCache)
    paged_append     tokens' keys and values into their sequences' pages, rotated on the way
    paged_attention  attention of tokens (single ones, pieces of prompts) over their sequences' pages, with a
                     window and first rows that stay in sight
    paged_gather     sequences' rows out of their pages, as caches of one piece
    adjust_logits    penalties for tokens that were there, biases and a grammar's mask on rows of logits

They take torch tensors on one GPU and enqueue on that GPU's current stream: nothing waits, and
a call may be captured into a graph.  Outputs and workspaces come from torch's allocator, so that
calls on several streams, and captured ones, share nothing.  No gradients, in either mode: the tensors are
those of decoding.  Wrong arguments raise ``ValidationError`` naming the argument; what the operators do with
lengths, parents, paths, tables and tokens that are out of range (the host cannot see them) is written at
each function.

Import this module, or torch, before the library's first call (a decoder's, say): they have to share a HIP
runtime, and an ImportError says so when they do not.
"""
from __future__ import annotations

import ctypes as C
import functools
import os
import struct
from typing import NamedTuple, Optional, Tuple, Union

import torch
from torch.autograd import forward_ad

from . import (ITTS_BF16, ITTS_E_VALIDATION, ITTS_F16, ITTS_F32, ITTS_I4, ValidationError, _check, itts_adjust_logits_args,
               itts_cache_keep_args, itts_paged_append_args, itts_paged_attention_args, itts_paged_gather_args,
               itts_token_scores_args, itts_tree_attention_args, lib)



def _one_runtime():
    """Loads the library, and refuses a process with two HIP runtimes: the second one finds no GPU."""
    lib.load()
    try:
        with open("/proc/self/maps") as f:
            found = {os.path.realpath(line.split(maxsplit=5)[5].strip()) for line in f if "libamdhip64" in line}
    except OSError:
        return
    if len(found) > 1:
        raise ImportError(f"torch and libitts_hip use different HIP runtimes ({', '.join(sorted(found))}): import torch or "
                          "itts_hip.ops before the library's first call")


_one_runtime()

_DTYPES = {torch.float32: ITTS_F32, torch.bfloat16: ITTS_BF16, torch.float16: ITTS_F16}


def _refuse(message: str):
    raise ValidationError(ITTS_E_VALIDATION, message)


def _tensor(t, name: str, dims: int, device=None, dtype=None, last=False):
    """Checks a tensor; device: the others' index; last: its last dimension must be contiguous.  (A call of an
    operator is host time before all else: nothing is asked twice here, and strides are handed on.)"""
    if not isinstance(t, torch.Tensor):
        _refuse(f"{name}: a tensor is needed, got {type(t).__name__}")
    if t.dim() != dims:
        _refuse(f"{name}: {dims} dimensions expected, got {t.dim()}")
    if dtype is None:
        if t.dtype not in _DTYPES:
            _refuse(f"{name}: float32, bfloat16 or float16 expected, got {t.dtype}")
    elif t.dtype != dtype:
        _refuse(f"{name}: {dtype} expected, got {t.dtype}")
    if device is None or t.get_device() != device:
        if not t.is_cuda:
            _refuse(f"{name}: a GPU tensor is needed, got one on {t.device}")
        if device is not None:
            _refuse(f"{name}: on {t.device}, the other tensors on cuda:{device}")
    if dtype is not torch.int32:  # (what its memory does not show)
        if t.requires_grad and torch.is_grad_enabled():
            _refuse(f"{name}: requires a gradient, which this operator does not give")
        if t.is_neg():
            _refuse(f"{name}: is negated when it is read, its memory is not what it says (resolve_neg() gives one that is)")
        if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
            _refuse(f"{name}: has a forward-mode tangent, which this operator does not give")
    strides = t.stride()
    if last and strides[-1] != 1 and t.shape[-1] > 1:
        _refuse(f"{name}: the last dimension must be contiguous")
    return strides


# Host time is most of a small call.  The current stream's handle without a Stream object around it saves
# 2 us, a new tensor without torch.empty's reading of its arguments 0.5 to 0.9 (of 1.3 to 1.6).
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
try:
    from torch._C._dynamo.guards import _empty_strided_cuda as _empty
except ImportError:
    def _empty(shape, strides, dtype):
        return torch.empty_strided(shape, strides, dtype=dtype, device="cuda")


def _packer(args, layout: str):
    """Fills the C structure `args` as bytes (1 us less than filling the ctypes one)."""
    s = struct.Struct(layout)
    if s.size != C.sizeof(args):
        raise ImportError(f"{args.__name__}: {C.sizeof(args)} bytes, packed {s.size}")
    return s.pack


_tree_args = _packer(itts_tree_attention_args, "@6P6i2if13q")
_scores_args = _packer(itts_token_scores_args, "@6P4ii2q")
_keep_args = _packer(itts_cache_keep_args, "@5P6ii9q")
_append_args = _packer(itts_paged_append_args, "@4P5i12q10P8i10q")
_paged_args = _packer(itts_paged_attention_args, "@4P5i12q5P8if5q")
_gather_args = _packer(itts_paged_gather_args, "@4P5i12q4P4i7q")
_adjust_args = _packer(itts_adjust_logits_args, "@9P3f5i6q")


def _on_device(op):
    """Runs an operator with its first tensor's device (a cache's: that of its keys) as the current one."""
    name = op.__code__.co_varnames[0]

    @functools.wraps(op)
    def run(*args, **kwargs):
        t = args[0] if args else kwargs.get(name)
        if isinstance(t, PagedCache):
            t = t.k
        try:
            if isinstance(t, torch.Tensor) and t.is_cuda and t.get_device() != _current_device():
                with torch.cuda.device(t.device):
                    return op(*args, **kwargs)
            return op(*args, **kwargs)
        except (struct.error, OverflowError) as e:
            _refuse(f"an argument does not fit the library's types: {e}")
    return run


def _run(fn, need, args, device):
    """Enqueues on the current device's stream, with the workspace that the sizes need."""
    if need is None:
        return _check(fn(args, _stream(device)))
    size = C.c_uint64()
    _check(need(args, C.byref(size)))
    bytes_ = size.value
    if not bytes_:
        return _check(fn(args, None, 0, _stream(device)))
    ws = _empty((bytes_,), (1,), torch.uint8)
    _check(fn(args, ws.data_ptr(), bytes_, _stream(device)))


@_on_device
def tree_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor, parents: torch.Tensor, *,
                   scale: Optional[float] = None, max_length: Optional[int] = None,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the nodes of one tree of drafted tokens a sequence.

    q        [batch][nodes][heads][dim], dim 64 or 128, at most 256 nodes
    k, v     [batch][key heads][rows][dim]: the caches, node i's key and value in row lengths[b] + i.
             q's type, or bfloat16 under float32 queries.  Any strides whose rows start at multiples
             of 16 bytes (0 between sequences that share a cache)
    lengths  [batch] int32: rows in front of the tree, which every node sees
    parents  [batch][nodes] int32: -1 for a node that follows the sequence itself, j < i for a child
             of node j.  Anything else marks an unused slot (padding); it and slots below it get
             rows of zeros
    scale    of the scores (default dim ** -0.5)
    max_length  rows that a sequence with its nodes may use (default: the caches' rows); a tight one
             lets short sequences do with one launch
    out      where to write (default: a new tensor)

    A node sees its sequence's rows, its ancestors and itself.  A negative length, or one whose nodes do not
    fit, gives rows of NaN.  Returns out [batch][nodes][heads][dim] in q's type."""
    sq = _tensor(q, "q", 4, last=True)
    dev = q.get_device()
    sk = _tensor(k, "k", 4, dev, last=True)
    sv = _tensor(v, "v", 4, dev, last=True)
    sl = _tensor(lengths, "lengths", 1, dev, torch.int32)
    sp = _tensor(parents, "parents", 2, dev, torch.int32, last=True)
    b, n, h, d = q.shape
    kb, hk, rows, kd = shape = k.shape
    if shape != v.shape or k.dtype != v.dtype:
        _refuse(f"v: must be like k, {tuple(shape)} {k.dtype}, got {tuple(v.shape)} {v.dtype}")
    if kb != b or kd != d:
        _refuse(f"k: [{b}][heads][rows][{d}] expected, got {tuple(shape)}")
    if lengths.shape[0] != b or parents.shape != (b, n):
        _refuse(f"lengths, parents: [{b}] and [{b}][{n}] expected, got {tuple(lengths.shape)} and {tuple(parents.shape)}")
    if b > 1 and sl[0] != 1:
        _refuse("lengths: must be contiguous")
    if max_length is not None:
        if int(max_length) > rows:
            _refuse(f"max_length: the caches have {rows} rows, got {int(max_length)}")
        rows = int(max_length)
    if out is None:
        so = (n * h * d, h * d, d)
        out = _empty((b, n, h, d), (*so, 1), q.dtype)
    else:
        so = _tensor(out, "out", 4, dev, q.dtype, last=True)
        if out.shape != q.shape:
            _refuse(f"out: {tuple(q.shape)} expected, got {tuple(out.shape)}")
    a = _tree_args(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lengths.data_ptr(),
                   parents.data_ptr(), b, n, h, hk, d, rows, _DTYPES[q.dtype], _DTYPES[k.dtype],
                   d ** -0.5 if scale is None else scale, sq[0], sq[1], sq[2], so[0], so[1], so[2], sk[0], sk[1], sk[2],
                   sv[0], sv[1], sv[2], sp[0])
    _run(lib.itts_tree_attention, lib.itts_tree_attention_workspace, a, dev)
    return out


class TokenScores(NamedTuple):
    log_probs: Optional[torch.Tensor]      # [rows][given] float32 (None without tokens)
    entropy: torch.Tensor                  # [rows] float32, nats
    top_tokens: torch.Tensor               # [rows][top_n] int32
    top_log_probs: torch.Tensor            # [rows][top_n] float32


@_on_device
def token_scores(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, top_n: int = 0) -> TokenScores:
    """Scores of rows of logits [rows][vocab] (float32, bfloat16 or float16; rows any distance apart).

    tokens   [rows] or [rows][given] int32: tokens whose log-probabilities are wanted, -1 for none (0.0
             comes back); another that is outside the vocabulary gives NaN
    top_n    how many of the most probable tokens to return (at most 64), the most probable first and
             the lowest token first among equals

    A row of -inf alone gives every token -inf, and entropy 0.  A NaN or +inf makes its row's
    log-probabilities and entropy NaN; NaN counts as -inf in the order.  log_probs has tokens' shape."""
    sx = _tensor(logits, "logits", 2, last=True)
    dev = logits.get_device()
    r, vocab = logits.shape
    given, log_probs, tok, log_probs_at, tok_row = 0, None, 0, 0, 0
    if tokens is not None:
        one = isinstance(tokens, torch.Tensor) and tokens.dim() == 1
        st = _tensor(tokens, "tokens", 1 if one else 2, dev, torch.int32, last=not one)
        if tokens.shape[0] != r:
            _refuse(f"tokens: {r} rows expected, got {tokens.shape[0]}")
        given, tok_row = 1 if one else tokens.shape[1], st[0]
        log_probs = _empty((r,) if one else (r, given), (1,) if one else (given, 1), torch.float32)
        if given:
            tok, log_probs_at = tokens.data_ptr(), log_probs.data_ptr()
    top_n = int(top_n)
    if not 0 <= top_n <= min(64, vocab):
        _refuse(f"top_n: must be in 0..=64 and at most the vocabulary of {vocab}, got {top_n}")
    entropy = _empty((r,), (1,), torch.float32)
    top_tokens = _empty((r, top_n), (top_n, 1), torch.int32)
    top_log_probs = _empty((r, top_n), (top_n, 1), torch.float32)
    a = _scores_args(logits.data_ptr(), tok, log_probs_at, entropy.data_ptr(), top_tokens.data_ptr(),
                     top_log_probs.data_ptr(), r, vocab, given, top_n, _DTYPES[logits.dtype], sx[0], tok_row)
    _run(lib.itts_token_scores, lib.itts_token_scores_workspace, a, dev)
    return TokenScores(log_probs, entropy, top_tokens, top_log_probs)


@_on_device
def cache_keep(k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor, path: torch.Tensor) -> torch.Tensor:
    """Keeps the accepted nodes of a tree: rows lengths[b] + path[b][i] of k and v [layers][batch][heads][rows][dim]
    (or [batch][heads][rows][dim]) move, in place, to rows lengths[b] + i in every layer and head.

    lengths  [batch] int32
    path     [batch][n] int32: the kept nodes in rising order, ended by a negative entry

    Returns the new lengths [batch], lengths[b] + the nodes kept; -1, with nothing moved, for a path that does not rise or
    leaves the cache, or a negative length."""
    dims = 4 if isinstance(k, torch.Tensor) and k.dim() == 4 else 5
    sk = _tensor(k, "k", dims, last=True)
    dev = k.get_device()
    sv = _tensor(v, "v", dims, dev, k.dtype, last=True)
    sl = _tensor(lengths, "lengths", 1, dev, torch.int32)
    sp = _tensor(path, "path", 2, dev, torch.int32, last=True)
    if v.shape != k.shape:
        _refuse(f"v: must be like k, {tuple(k.shape)}, got {tuple(v.shape)}")
    if dims == 5:
        layers, b, h, rows, d = k.shape
    else:
        layers, (b, h, rows, d) = 1, k.shape
        sk, sv = (0, *sk), (0, *sv)
    if lengths.shape[0] != b or path.shape[0] != b:
        _refuse(f"lengths, path: {b} sequences expected, got {lengths.shape[0]} and {path.shape[0]}")
    if b > 1 and sl[0] != 1:
        _refuse("lengths: must be contiguous")
    new = _empty((b,), (1,), torch.int32)
    a = _keep_args(k.data_ptr(), v.data_ptr(), lengths.data_ptr(), path.data_ptr(), new.data_ptr(), layers, b, h,
                   rows, d, path.shape[1], _DTYPES[k.dtype], sk[0], sk[1], sk[2], sk[3], sv[0], sv[1], sv[2], sv[3], sp[0])
    _run(lib.itts_cache_keep, None, a, dev)
    return new


class PagedCache(NamedTuple):
    """Pages of keys and values that any sequence may own, k and v [pages][key heads][page size][dim], float32, bfloat16
    or float16; or uint8 [pages][key heads][page size][dim / 2], 4 bits: two codes a byte, the lower half first, and
    k_params, v_params float16 [pages][key heads][page size][dim / 64][2] with the (scale, base) of every 64 elements, a value
    being scale * code + base.  dim 64 or 128, page sizes multiples of 16; any strides whose rows start at multiples of 16
    bytes (pairs: dim / 16), pages less than 2^32 bytes apart, rows at most 2^26."""
    k: torch.Tensor
    v: torch.Tensor
    k_params: Optional[torch.Tensor] = None
    v_params: Optional[torch.Tensor] = None


def paged_cache(pages: int, heads: int, page_size: int, dim: int, dtype: torch.dtype = torch.bfloat16, *, bits: int = 16,
                device: Union[None, int, str, torch.device] = "cuda") -> PagedCache:
    """Memory for `pages` pages (what it holds is not set): of `dtype` (bits 32 with float32 alone, which may leave them out), or
    with bits 4 of codes and their pairs."""
    if bits == 4:
        k, v = (torch.empty((pages, heads, page_size, dim // 2), dtype=torch.uint8, device=device) for _ in range(2))
        kp, vp = (torch.empty((pages, heads, page_size, dim // 64, 2), dtype=torch.float16, device=device) for _ in range(2))
        return PagedCache(k, v, kp, vp)
    if bits not in (16, 32) or dtype not in _DTYPES or (bits == 32 and dtype != torch.float32):
        _refuse(f"bits, dtype: float32, bfloat16 or float16, or 4 bits expected, got {bits} and {dtype}")
    k, v = (torch.empty((pages, heads, page_size, dim), dtype=dtype, device=device) for _ in range(2))
    return PagedCache(k, v)


def _cache(cache, device=None):
    """A cache's part of a packed structure, its key heads, page size, dim and device."""
    if not isinstance(cache, tuple) or len(cache) != 4:
        _refuse(f"cache: a PagedCache is needed, got {type(cache).__name__}")
    k, v, kp, vp = cache
    codes = isinstance(k, torch.Tensor) and k.dtype == torch.uint8
    sk = _tensor(k, "cache.k", 4, device, torch.uint8 if codes else None, last=True)
    device = k.get_device()
    sv = _tensor(v, "cache.v", 4, device, k.dtype, last=True)
    shape = k.shape
    n, h, size, d = shape
    if v.shape != shape:
        _refuse(f"cache.v: must be like k, {tuple(shape)}, got {tuple(v.shape)}")
    if not codes:
        if kp is not None or vp is not None:
            _refuse("cache.k_params, v_params: for 4 bits alone")
        return (k.data_ptr(), v.data_ptr(), 0, 0, n, size, h, d, _DTYPES[k.dtype], sk[0], sk[1], sk[2], sv[0], sv[1], sv[2],
                0, 0, 0, 0, 0, 0), h, size, d, device
    d *= 2
    skp = _tensor(kp, "cache.k_params", 5, device, torch.float16)
    svp = _tensor(vp, "cache.v_params", 5, device, torch.float16)
    want = (n, h, size, d // 64, 2)
    if kp.shape != want or vp.shape != want:
        _refuse(f"cache.k_params, v_params: {want} expected, got {tuple(kp.shape)} and {tuple(vp.shape)}")
    for s in (skp, svp):
        if s[4] != 1 or (d > 64 and s[3] != 2):
            _refuse("cache.k_params, v_params: the last two dimensions must be contiguous")
    return (k.data_ptr(), v.data_ptr(), kp.data_ptr(), vp.data_ptr(), n, size, h, d, ITTS_I4, sk[0], sk[1], sk[2], sv[0], sv[1],
            sv[2], skp[0], skp[1], skp[2], svp[0], svp[1], svp[2]), h, size, d, device


def _sequences(lengths, table, device, starts=None):
    """Checks what says where sequences are: (batch, pages of a row of the table, its stride)."""
    sl = _tensor(lengths, "lengths", 1, device, torch.int32)
    st = _tensor(table, "table", 2, device, torch.int32, last=True)
    b = lengths.shape[0]
    tb, pages = table.shape
    if tb != b:
        _refuse(f"table: {b} sequences expected, got {tb}")
    if b > 1 and sl[0] != 1:
        _refuse("lengths: must be contiguous")
    if starts is not None:
        ss = _tensor(starts, "starts", 1, device, torch.int32)
        if starts.shape[0] != b + 1:
            _refuse(f"starts: [{b + 1}] expected, got {tuple(starts.shape)}")
        if b > 0 and ss[0] != 1:
            _refuse("starts: must be contiguous")
    return b, pages, st[0]


class PagedAppend(NamedTuple):
    lengths: torch.Tensor                  # [batch] int32: the new ones
    q: Optional[torch.Tensor]              # the rotated queries (None without queries)


@_on_device
def paged_append(cache: PagedCache, k: torch.Tensor, v: torch.Tensor, starts: torch.Tensor, lengths: torch.Tensor,
                 table: torch.Tensor, *, q: Optional[torch.Tensor] = None, rotation: Optional[torch.Tensor] = None,
                 positions: Optional[torch.Tensor] = None, interleaved: bool = False,
                 q_out: Optional[torch.Tensor] = None) -> PagedAppend:
    """Appends tokens' keys and values to their sequences, in the cache's pages, rotated by their positions on the way.

    k, v     [tokens][key heads][dim]: the cache's type, float32 over bfloat16, or any over 4 bits.  Any strides whose
             rows start at multiples of 16 bytes (parts of one product's result)
    starts   [batch + 1] int32, rising: sequence b's tokens are starts[b] .. starts[b + 1] - 1
    lengths  [batch] int32: rows that the sequences have; token i becomes row lengths[b] + i
    table    [batch][pages] int32: the pages of a sequence's rows in their order
    rotation [positions][n] float32, n a multiple of 16 up to dim: n / 2 cosines, then the sines of a position's angles.
             The first n elements of each key turn by them, elements i and i + n / 2 together, or with `interleaved` 2 i
             and 2 i + 1.  Worked out in 64 bits, rounded once
    positions  [tokens] int32: rows of `rotation` (default: the tokens' rows)
    q        [tokens][heads][dim] of k's type: queries that turn the same way, into q_out (default: a new tensor; q
             itself is fine)

    4 bits: of every 64 elements base = min, scale = (max - min) / 15, both as float16, and codes to the nearest.  64 elements of
    which one is no finite number, or too large for float16, read back as NaN.
    Returns the new lengths and the queries.  A sequence with a negative length, or without room in its table, is not written, nor
    is a row whose table entry is no page of the cache: its new length is -1 (and its queries NaN in the first case).  So it is, too,
    for a sequence whose starts fall, leave the tensors or lie in front of where an earlier one ends (of more than 64 perhaps for its
    neighbours): it has no tokens.  A position outside `rotation` makes its rows NaN.  Queries of tokens that belong to no sequence
    become zeros.  Two sequences must not be given the same row of a page to write."""
    pages, hk, size, d, dev = _cache(cache)
    sk = _tensor(k, "k", 3, dev, last=True)
    sv = _tensor(v, "v", 3, dev, k.dtype, last=True)
    b, n_table, table_b = _sequences(lengths, table, dev, starts)
    shape = k.shape
    n = shape[0]
    if shape[1] != hk or shape[2] != d or v.shape != shape:
        _refuse(f"k, v: [tokens][{hk}][{d}] expected, got {tuple(shape)} and {tuple(v.shape)}")
    heads, sq, so, q_at, out_at = 0, (0, 0), (0, 0), 0, 0
    if q is not None:
        sq = _tensor(q, "q", 3, dev, k.dtype, last=True)
        heads = q.shape[1]
        if q.shape[0] != n or q.shape[2] != d:
            _refuse(f"q: [{n}][heads][{d}] expected, got {tuple(q.shape)}")
        if heads == 0:
            _refuse("q: no heads")
        if q_out is None:
            so = (heads * d, d)
            q_out = _empty((n, heads, d), (*so, 1), q.dtype)
        else:
            so = _tensor(q_out, "q_out", 3, dev, q.dtype, last=True)
            if q_out.shape != q.shape:
                _refuse(f"q_out: {tuple(q.shape)} expected, got {tuple(q_out.shape)}")
        q_at, out_at = q.data_ptr(), q_out.data_ptr()
    elif q_out is not None:
        _refuse("q_out: without q")
    rot_at, n_rot, n_pos, rot_row, pos_at = 0, 0, 0, 0, 0
    if rotation is not None:
        sr = _tensor(rotation, "rotation", 2, dev, torch.float32, last=True)
        rot_at, rot_row = rotation.data_ptr(), sr[0]
        n_pos, n_rot = rotation.shape
        if n_pos == 0:
            _refuse("rotation: no positions")
    if positions is not None:
        sp = _tensor(positions, "positions", 1, dev, torch.int32)
        if positions.shape[0] != n or (n > 1 and sp[0] != 1):
            _refuse(f"positions: [{n}], contiguous, expected, got {tuple(positions.shape)}")
        pos_at = positions.data_ptr()
    new = _empty((b,), (1,), torch.int32)
    a = _append_args(*pages, k.data_ptr(), v.data_ptr(), q_at, out_at, rot_at, starts.data_ptr(), lengths.data_ptr(),
                     table.data_ptr(), pos_at, new.data_ptr(), b, n, heads, n_table, n_rot, n_pos, bool(interleaved),
                     _DTYPES[k.dtype], sk[0], sk[1], sv[0], sv[1], sq[0], sq[1], so[0], so[1], rot_row, table_b)
    _run(lib.itts_paged_append, None, a, dev)
    return PagedAppend(new, q_out)


@_on_device
def paged_attention(q: torch.Tensor, cache: PagedCache, starts: torch.Tensor, lengths: torch.Tensor, table: torch.Tensor, *,
                    scale: Optional[float] = None, window: int = 0, sinks: int = 0, max_length: Optional[int] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of tokens over their sequences' rows in a paged cache: decode steps, prompts and pieces of them together.

    q        [tokens][heads][dim]: the cache's type, float32 over bfloat16, or any over 4 bits.  Any strides whose rows
             start at multiples of 16 bytes
    starts   [batch + 1] int32, rising: sequence b's tokens are starts[b] .. starts[b + 1] - 1
    lengths  [batch] int32: rows of the sequences, their tokens' own among them (as paged_append returns them): a
             sequence's n tokens are its last n rows, and each sees the rows up to its own
    table    [batch][pages] int32: the pages of a sequence's rows in their order
    scale    of the scores (default dim ** -0.5)
    window   rows that a token sees, its own the last of them (0: all); pages in front of every token's window may have been
             given to other sequences, their entries in the table are not used
    sinks    first rows of a sequence that stay in sight of every token beside the window
    max_length  the longest length that may come (default: the table's pages); a tight one lets short sequences do
             with one launch
    out      where to write (default: a new tensor; q itself is fine)

    A token at a position below 0 (more tokens than rows) gets zeros, as do tokens that belong to no sequence (starts that do not
    rise: as paged_append has it).  A length that is
    negative or too long, and a row in sight whose table entry is no page of the cache, gives NaN.  Returns out
    [tokens][heads][dim] in q's type."""
    sq = _tensor(q, "q", 3, last=True)
    dev = q.get_device()
    pages, hk, size, d, _ = _cache(cache, dev)
    b, n_table, table_b = _sequences(lengths, table, dev, starts)
    n, h, qd = shape = q.shape
    if qd != d:
        _refuse(f"q: [tokens][heads][{d}] expected, got {tuple(shape)}")
    rows = min(n_table * size, 1 << 24)
    if max_length is not None:
        if not 0 <= int(max_length) <= rows:
            _refuse(f"max_length: the table has room for {rows} rows, got {int(max_length)}")
        rows = int(max_length)
    if out is None:
        so = (h * d, d)
        out = _empty((n, h, d), (*so, 1), q.dtype)
    else:
        so = _tensor(out, "out", 3, dev, q.dtype, last=True)
        if out.shape != shape:
            _refuse(f"out: {tuple(shape)} expected, got {tuple(out.shape)}")
    a = _paged_args(*pages, q.data_ptr(), out.data_ptr(), starts.data_ptr(), lengths.data_ptr(), table.data_ptr(), b, n, h,
                    n_table, rows, window, sinks, _DTYPES[q.dtype], d ** -0.5 if scale is None else scale, sq[0], sq[1], so[0],
                    so[1], table_b)
    _run(lib.itts_paged_attention, lib.itts_paged_attention_workspace, a, dev)
    return out


@_on_device
def paged_gather(cache: PagedCache, lengths: torch.Tensor, table: torch.Tensor, rows: int, *,
                 dtype: Optional[torch.dtype] = None, k_out: Optional[torch.Tensor] = None,
                 v_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The first `rows` rows of every sequence out of its pages, as caches of one piece (tree_attention's): k, v
    [batch][key heads][rows][dim], zeros from lengths[b] on.

    lengths, table  as paged_attention takes them
    dtype    of the results over 4 bits (default float32); otherwise it is the cache's
    k_out, v_out  where to write (default: new tensors)

    Rows of a sequence whose length is negative or longer than its table, and rows whose table entry is no page of the cache, are
    NaN.  Returns (k, v)."""
    pages, hk, size, d, dev = _cache(cache)
    b, n_table, table_b = _sequences(lengths, table, dev)
    own = cache.k.dtype if cache.k_params is None else None
    dtype = dtype or (k_out.dtype if isinstance(k_out, torch.Tensor) else own or torch.float32)
    if dtype not in _DTYPES or (own is not None and dtype != own):
        _refuse(f"dtype: {own or 'float32, bfloat16 or float16'} expected, got {dtype}")
    rows = int(rows)
    if rows < 0:
        _refuse(f"rows: must be >= 0, got {rows}")
    outs, strides = [], []
    for t, name in ((k_out, "k_out"), (v_out, "v_out")):
        if t is None:
            s = (hk * rows * d, rows * d, d, 1)
            t = _empty((b, hk, rows, d), s, dtype)
        else:
            s = _tensor(t, name, 4, dev, dtype, last=True)
            if t.shape != (b, hk, rows, d):
                _refuse(f"{name}: {(b, hk, rows, d)} expected, got {tuple(t.shape)}")
        outs.append(t)
        strides.extend(s[:3])
    a = _gather_args(*pages, outs[0].data_ptr(), outs[1].data_ptr(), lengths.data_ptr(), table.data_ptr(), b, rows, n_table,
                     _DTYPES[dtype], *strides, table_b)
    _run(lib.itts_paged_gather, None, a, dev)
    return outs[0], outs[1]


def _per_row(x, name, rows, device):
    """A number for every row, or one a row: (address, number)."""
    if not isinstance(x, torch.Tensor):
        return 0, float(x)
    s = _tensor(x, name, 1, device, torch.float32)
    if x.shape[0] != rows or (rows > 1 and s[0] != 1):
        _refuse(f"{name}: a number or [{rows}], contiguous, expected, got {tuple(x.shape)}")
    return x.data_ptr(), 0.0


@_on_device
def adjust_logits(logits: torch.Tensor, *, history: Optional[torch.Tensor] = None,
                  repetition: Union[float, torch.Tensor] = 1.0, frequency: Union[float, torch.Tensor] = 0.0,
                  presence: Union[float, torch.Tensor] = 0.0, bias_tokens: Optional[torch.Tensor] = None,
                  bias: Optional[torch.Tensor] = None, allowed: Optional[torch.Tensor] = None,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rows of logits [rows][vocab] (float32, bfloat16 or float16; rows any distance apart) as the next token is to be
    chosen from them.

    history  [rows][n] int32, n <= 65535: the tokens that were there, -1 (or any number outside the vocabulary) in places
             that are not used
    repetition, frequency, presence  a number, or float32 [rows]: a token that stands c > 0 times in its row's history gets
             (x < 0 ? x * repetition : x / repetition) - (frequency * c + presence)
    bias_tokens, bias  [rows][n] int32 and float32: added to those tokens' logits (where one stands twice, the last one's)
    allowed  [rows][(vocab + 31) // 32] int32: bit t % 32 of word t // 32 says whether token t may follow; the others
             become -inf
    out      where to write (default: a new tensor; logits itself is fine, but not its memory shifted)

    Rows of lists and masks may be one for all (expand()).  Worked out in float32, rounded once.  Returns out."""
    sx = _tensor(logits, "logits", 2, last=True)
    dev = logits.get_device()
    r, vocab = logits.shape
    hist, n_hist, hist_row = 0, 0, 0
    if history is not None:
        s = _tensor(history, "history", 2, dev, torch.int32, last=True)
        if history.shape[0] != r:
            _refuse(f"history: {r} rows expected, got {history.shape[0]}")
        hist, n_hist, hist_row = history.data_ptr(), history.shape[1], s[0]
    rep, rep_all = _per_row(repetition, "repetition", r, dev)
    freq, freq_all = _per_row(frequency, "frequency", r, dev)
    pres, pres_all = _per_row(presence, "presence", r, dev)
    tok, n_bias, tok_row, add, add_row = 0, 0, 0, 0, 0
    if bias_tokens is not None or bias is not None:
        st = _tensor(bias_tokens, "bias_tokens", 2, dev, torch.int32, last=True)
        sb = _tensor(bias, "bias", 2, dev, torch.float32, last=True)
        if bias_tokens.shape[0] != r or bias.shape != bias_tokens.shape:
            _refuse(f"bias_tokens, bias: {r} rows of one length expected, got {tuple(bias_tokens.shape)} and {tuple(bias.shape)}")
        tok, n_bias, tok_row, add, add_row = bias_tokens.data_ptr(), bias.shape[1], st[0], bias.data_ptr(), sb[0]
    mask, mask_row = 0, 0
    if allowed is not None:
        sm = _tensor(allowed, "allowed", 2, dev, torch.int32, last=True)
        if allowed.shape != (r, (vocab + 31) // 32):
            _refuse(f"allowed: {(r, (vocab + 31) // 32)} expected, got {tuple(allowed.shape)}")
        mask, mask_row = allowed.data_ptr(), sm[0]
    if out is None:
        out = _empty((r, vocab), (vocab, 1), logits.dtype)
        out_row = vocab
    else:
        out_row = _tensor(out, "out", 2, dev, logits.dtype, last=True)[0]
        if out.shape != logits.shape:
            _refuse(f"out: {tuple(logits.shape)} expected, got {tuple(out.shape)}")
    a = _adjust_args(logits.data_ptr(), out.data_ptr(), hist, tok, add, mask, rep, freq, pres, rep_all, freq_all, pres_all, r,
                     vocab, n_hist, n_bias, _DTYPES[logits.dtype], sx[0], out_row, hist_row, tok_row, add_row, mask_row)
    _run(lib.itts_adjust_logits, None, a, dev)
    return out
