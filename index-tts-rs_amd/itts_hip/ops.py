"""The library's operators on device tensors: decoding with drafted trees.

    tree_attention   attention of every node of a tree of drafted tokens over its sequence's
                     cached rows and its own ancestors (one node: a decode step)
    token_scores     log-probabilities of given tokens, entropy, the most probable tokens
    cache_keep       the accepted nodes' key and value rows moved up in the caches

They take torch tensors on one GPU and enqueue on that GPU's current stream: nothing waits, and
a call may be captured into a graph.  Outputs and workspaces come from torch's allocator, so that
calls on several streams, and captured ones, share nothing.  No gradients, in either mode: the tensors are
those of decoding.  Wrong arguments raise ``ValidationError`` naming the argument; what the operators do with
lengths, parents, paths and tokens that are out of range (the host cannot see them) is written at
each function.

Import this module, or torch, before the library's first call (a decoder's, say): they have to share a HIP
runtime, and an ImportError says so when they do not.
"""
from __future__ import annotations

import ctypes as C
import functools
import os
import struct
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import (ITTS_BF16, ITTS_E_VALIDATION, ITTS_F16, ITTS_F32, ValidationError, _check, itts_cache_keep_args,
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
    if t.requires_grad and torch.is_grad_enabled():
        _refuse(f"{name}: requires a gradient, which this operator does not give")
    if dtype is not torch.int32:  # (what its memory does not show)
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


def _on_device(op):
    """Runs an operator with its first tensor's device as the current one."""
    name = op.__code__.co_varnames[0]

    @functools.wraps(op)
    def run(*args, **kwargs):
        t = args[0] if args else kwargs.get(name)
        try:
            if isinstance(t, torch.Tensor) and t.is_cuda and t.device.index != torch.cuda.current_device():
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
