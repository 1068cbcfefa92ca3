"""Refusals of the operators over paged caches and on logits, without a GPU: wrong sizes, types, strides and alignments at the
C entries, and wrong tensors at the Python ones."""
import ctypes as C
import random

import pytest
import torch

import itts_hip as H
from itts_hip import ops

P = 1 << 20  # an address that nothing reads: every call below is refused before its memory matters
PAGES = dict(k=P, v=9 * P, k_params=None, v_params=None, n_pages=10, page_size=32, n_kv_head=4, head_dim=64, dtype=H.ITTS_BF16,
             k_page=4 * 32 * 64, k_head=32 * 64, k_row=64, v_page=4 * 32 * 64, v_head=32 * 64, v_row=64)
CODES = dict(dtype=H.ITTS_I4, k_params=17 * P, v_params=25 * P, k_page=4 * 32 * 32, k_head=32 * 32, k_row=32, v_page=4 * 32 * 32,
             v_head=32 * 32, v_row=32, k_params_page=4 * 32 * 2, k_params_head=32 * 2, k_params_row=2, v_params_page=4 * 32 * 2,
             v_params_head=32 * 2, v_params_row=2)


def pages(over):
    return H.itts_pages(**dict(PAGES, **{k[6:]: over.pop(k) for k in list(over) if k.startswith("pages_")}))


def append(**over):
    f = dict(k=P, v=P, q=P, q_out=2 * P, rotation=P, starts=P, lengths=P, table=P, positions=None, new_lengths=2 * P, batch=3, n_tokens=7,
             n_head=8, n_table=5, n_rotated=64, n_positions=160, interleaved=0, dtype=H.ITTS_F32, k_token=256, k_head=64, v_token=256,
             v_head=64, q_token=512, q_head=64, q_out_token=512, q_out_head=64, rotation_row=64, table_batch=5)
    g = pages(over)
    f.update(over)
    return H.itts_paged_append_args(pages=g, **f)


def attention(**over):
    f = dict(q=P, out=2 * P, starts=P, lengths=P, table=P, batch=3, n_tokens=7, n_head=8, n_table=5, max_rows=160, window=0, sinks=0,
             q_dtype=H.ITTS_F32, scale=0.125, q_token=512, q_head=64, out_token=512, out_head=64, table_batch=5)
    g = pages(over)
    f.update(over)
    return H.itts_paged_attention_args(pages=g, **f)


def gather(**over):
    f = dict(k=P, v=2 * P, lengths=P, table=P, batch=3, n_rows=100, n_table=5, dtype=H.ITTS_BF16, k_batch=25600, k_head=6400, k_row=64,
             v_batch=25600, v_head=6400, v_row=64, table_batch=5)
    g = pages(over)
    f.update(over)
    return H.itts_paged_gather_args(pages=g, **f)


def adjust(**over):
    f = dict(logits=P, out=2 * P, history=P, bias_tokens=P, bias=P, allowed=P, repetition=None, frequency=None, presence=None,
             repetition_all=1.5, frequency_all=0.5, presence_all=0.5, rows=3, vocab=100, n_history=4, n_bias=2, dtype=H.ITTS_F32,
             logits_row=100, out_row=100, history_row=4, bias_tokens_row=2, bias_row=2, allowed_row=4)
    f.update(over)
    return H.itts_adjust_logits_args(**f)


def call(kind, a):
    if kind is attention:
        return H._check(H.lib.itts_paged_attention(C.byref(a), None, 0, None))
    entry = {append: H.lib.itts_paged_append, gather: H.lib.itts_paged_gather, adjust: H.lib.itts_adjust_logits}[kind]
    return H._check(entry(C.byref(a), None))


NAN, INF = float("nan"), float("inf")
SHARED = [("batch", dict(batch=-1)), ("batch", dict(batch=65536)), ("table", dict(n_table=-1)), ("table", dict(table_batch=-5)),
          ("pages.dtype", dict(pages_dtype=0)), ("pages.dtype", dict(pages_dtype=5)), ("pages.head_dim", dict(pages_head_dim=80)),
          ("pages.n_kv_head", dict(pages_n_kv_head=0)), ("pages.page_size", dict(pages_page_size=0)),
          ("pages.page_size", dict(pages_page_size=24)), ("pages.page_size", dict(pages_page_size=65552)),
          ("pages.n_pages", dict(pages_n_pages=0)), ("pages: k", dict(pages_k=None)), ("pages.k", dict(pages_k=P + 8)),
          ("pages.k", dict(pages_k_row=60)), ("pages.v", dict(pages_v_head=-2048)), ("pages.v", dict(pages_v=9 * P + 4)),
          ("pages.k_row", dict(pages_k_row=1 << 27)), ("pages.k_page", dict(pages_k_page=1 << 31)),
          ("pages.k_page", dict(pages_v_page=1 << 31)), ("pages: k", dict(pages_dtype=H.ITTS_I4)),
          ("pages.k_params", dict({"pages_" + k: v for k, v in CODES.items()}, pages_k_params=17 * P + 2)),
          ("pages.k_params", dict({"pages_" + k: v for k, v in CODES.items()}, pages_v_params_row=3)),
          ("pages.k", dict({"pages_" + k: v for k, v in CODES.items()}, pages_k_row=24))]
REFUSED = ([(kind, field, over) for kind in (append, attention, gather) for field, over in SHARED] + [
    (append, "n_tokens", dict(n_tokens=-1)), (append, "n_tokens", dict(n_tokens=(1 << 20) + 1)), (append, "batch", dict(batch=0)),
    (append, "n_head", dict(n_head=6)), (append, "n_head", dict(n_head=-4)), (append, "n_head", dict(n_head=1028)),
    (append, "dtype", dict(dtype=H.ITTS_F16)), (append, "dtype", dict(dtype=0)), (append, "dtype", dict(dtype=H.ITTS_I4)),
    (append, "k", dict(k_token=257)), (append, "v", dict(v=P + 4)), (append, "q", dict(q_head=-64)), (append, "q_out", dict(q_out_head=2)),
    (append, "q_out", dict(q_out_token=0)), (append, "q_out", dict(q_out=P, q_token=1024)),
    (append, "n_rotated", dict(n_rotated=0)), (append, "n_rotated", dict(n_rotated=40)), (append, "n_rotated", dict(n_rotated=80)),
    (append, "n_positions", dict(n_positions=-1)), (append, "rotation", dict(rotation_row=66)), (append, "rotation", dict(rotation=P + 4)),
    (append, "new_lengths", dict(new_lengths=P)), (append, "k, v", dict(starts=None)), (append, "k, v", dict(q=None)),
    (append, "k, v", dict(table=None)), (append, "pages.k, v", dict(pages_v=P)), (append, "pages.k, v", dict(pages_v=P + 2 * 64)),
    (append, "pages.k, v", dict(pages_k_row=32)), (append, "pages.k, v", dict(pages_k_page=0)),
    (append, "pages.k_params, v", dict({"pages_" + k: v for k, v in CODES.items()}, pages_v_params=17 * P)),
    (attention, "n_tokens", dict(n_tokens=-1)), (attention, "n_tokens", dict(n_tokens=1 << 20, n_head=1024)),
    (attention, "batch", dict(batch=0)), (attention, "n_head", dict(n_head=6)), (attention, "n_head", dict(n_head=0)),
    (attention, "q_dtype", dict(q_dtype=H.ITTS_F16)), (attention, "q_dtype", dict(q_dtype=7)), (attention, "q", dict(q=P + 8)),
    (attention, "out", dict(out_head=32)), (attention, "out", dict(out_token=64)), (attention, "max_rows", dict(max_rows=161)),
    (attention, "max_rows", dict(max_rows=-1)), (attention, "max_rows", dict(n_table=1 << 20, max_rows=(1 << 24) + 1)),
    (attention, "window", dict(window=-1)), (attention, "window", dict(sinks=-1)), (attention, "scale", dict(scale=NAN)),
    (attention, "scale", dict(scale=INF)), (attention, "q, out", dict(lengths=None)), (attention, "q, out", dict(out=None)),
    (gather, "n_rows", dict(n_rows=-1)), (gather, "n_rows", dict(n_rows=(1 << 24) + 1)), (gather, "dtype", dict(dtype=H.ITTS_F32)),
    (gather, "dtype", dict(dtype=H.ITTS_I4)), (gather, "k", dict(k_row=60)), (gather, "v", dict(v=P + 2)), (gather, "k, v", dict(v=P)),
    (gather, "k, v", dict(k_row=32)), (gather, "k, v", dict(k_batch=0)), (gather, "k, v", dict(lengths=None)),
    (adjust, "rows", dict(rows=-1)), (adjust, "rows", dict(rows=1 << 23, vocab=1 << 24)), (adjust, "vocab", dict(vocab=0)),
    (adjust, "vocab", dict(vocab=(1 << 24) + 1)), (adjust, "n_history", dict(n_history=65536)), (adjust, "n_bias", dict(n_bias=-1)),
    (adjust, "dtype", dict(dtype=H.ITTS_I4)), (adjust, "logits", dict(logits=P + 2)), (adjust, "logits_row", dict(logits_row=-100)),
    (adjust, "logits_row", dict(allowed_row=-1)), (adjust, "out", dict(out_row=99)), (adjust, "out", dict(out=P, logits_row=200)),
    (adjust, "repetition", dict(repetition_all=0.0)), (adjust, "repetition", dict(repetition_all=INF)),
    (adjust, "frequency", dict(presence_all=NAN)), (adjust, "logits", dict(logits=None)), (adjust, "logits", dict(history=None)),
    (adjust, "logits", dict(bias=None)),
])


@pytest.mark.parametrize("kind,field,over", REFUSED, ids=lambda x: getattr(x, "__name__", str(x))[:60])
def test_c_entries_refuse(kind, field, over):
    with pytest.raises(H.ValidationError) as e:
        call(kind, kind(**dict(over)))
    assert e.value.message.startswith(field), e.value.message


def test_null_arguments():
    n = C.c_uint64()
    for f in (H.lib.itts_paged_append, H.lib.itts_paged_gather, H.lib.itts_adjust_logits):
        with pytest.raises(H.ValidationError, match="args"):
            H._check(f(None, None))
    with pytest.raises(H.ValidationError, match="args"):
        H._check(H.lib.itts_paged_attention(None, None, 0, None))
    with pytest.raises(H.ValidationError, match="args"):
        H._check(H.lib.itts_paged_attention_workspace(None, C.byref(n)))
    with pytest.raises(H.ValidationError, match="bytes"):
        H._check(H.lib.itts_paged_attention_workspace(C.byref(attention()), None))


def test_empty_calls_do_nothing():
    call(append, append(batch=0, n_tokens=0, starts=None, lengths=None))
    call(attention, attention(n_tokens=0, q=None, starts=None))
    call(gather, gather(batch=0, lengths=None))
    call(gather, gather(n_rows=0, k=None))
    call(adjust, adjust(rows=0, logits=None))


def takes(kind, **over):
    """Whether the sizes pass: without a GPU the call then fails for that."""
    try:
        call(kind, kind(**over))
    except H.ValidationError as e:
        return "not device memory" in e.message or "workspace" in e.message
    except H.IttsError:
        pass
    return True


def test_layouts_that_are_taken():
    """Rows of all heads beside each other, keys beside values, one page, one head; 4 bits; q turned in place."""
    rows = dict(pages_k_page=32 * 256, pages_k_head=64, pages_k_row=256, pages_v_page=32 * 256, pages_v_head=64, pages_v_row=256)
    both = dict(pages_v=P + 2 * 32 * 256, pages_k_page=2 * 32 * 256, pages_k_head=64, pages_k_row=256, pages_v_page=2 * 32 * 256,
                pages_v_head=64, pages_v_row=256)
    for kind in (append, attention, gather):
        assert takes(kind, **rows) and takes(kind, **both) and takes(kind, pages_n_pages=1, pages_k_page=0, pages_v_page=0)
        assert takes(kind, **dict({"pages_" + k: v for k, v in CODES.items()}, **({"dtype": H.ITTS_F16} if kind is gather else {})))
    assert takes(append, q_out=P) and takes(append, n_head=0, q=None, q_out=None) and takes(append, rotation=None)
    assert takes(attention, pages_v=P)  # (keys that are values, read alone)
    assert takes(adjust, out=P) and takes(adjust, logits_row=0, history_row=0, allowed_row=0)


def test_python_entries_refuse():
    i = torch.zeros(2, dtype=torch.int32)
    x = torch.zeros(1, 4, 64)
    cache = ops.paged_cache(3, 4, 16, 64, device="cpu")
    for call_, match in ((lambda: ops.paged_attention(x, cache, i, i[:1], i.view(1, 2)), "q: a GPU tensor"),
                         (lambda: ops.paged_append(cache, x, x, i, i[:1], i.view(1, 2)), "cache.k: a GPU tensor"),
                         (lambda: ops.paged_append(x, x, x, i, i[:1], i.view(1, 2)), "cache: a PagedCache"),
                         (lambda: ops.paged_gather(cache, i[:1], i.view(1, 2), 5), "cache.k: a GPU tensor"),
                         (lambda: ops.adjust_logits(torch.zeros(2, 5)), "logits: a GPU tensor"),
                         (lambda: ops.adjust_logits("x"), "logits: a tensor"),
                         (lambda: ops.paged_cache(3, 4, 16, 64, torch.float32, bits=8, device="cpu"), "bits")):
        with pytest.raises(H.ValidationError, match=match):
            call_()


def test_cache_memory():
    c = ops.paged_cache(3, 4, 16, 128, bits=4, device="cpu")
    assert c.k.shape == (3, 4, 16, 64) and c.k.dtype == torch.uint8 and c.v_params.shape == (3, 4, 16, 2, 2)
    c = ops.paged_cache(3, 4, 16, 128, torch.float32, bits=32, device="cpu")
    assert c.k.shape == (3, 4, 16, 128) and c.k.dtype == torch.float32 and c.k_params is None


def test_a_rotation_has_positions():
    """Without one a token's row of the table, which is read before anything says that its position is not there, would lie outside it."""
    with pytest.raises(H.ValidationError) as e:
        call(append, append(n_positions=0))
    assert e.value.message.startswith("n_positions"), e.value.message
    assert takes(append, n_positions=0, rotation=None) and takes(append, n_positions=1)


@pytest.mark.parametrize("over,fine", [
    (dict(out=P + 4), False), (dict(out=P - 4), False), (dict(out=P + 4 * 99), False), (dict(out=P + 4 * 100), False), (dict(out=P + 4 * 300), True),
    (dict(out=P - 4 * 300), True), (dict(out=P, logits_row=200, out_row=200), True), (dict(out=P, logits_row=200), False),
    (dict(out=P + 400, logits_row=200, out_row=200), True), (dict(out=P + 396, logits_row=200, out_row=200), False),
    (dict(out=P + 404, logits_row=200, out_row=200), False), (dict(out=P, logits_row=0, out_row=100), False), (dict(out=P, rows=1, out_row=0), True),
    (dict(out=P + 4, rows=1), False), (dict(out=P + 400, logits_row=0), True), (dict(out=P + 200, dtype=H.ITTS_BF16), False),
    (dict(out=P + 600, dtype=H.ITTS_BF16), True)], ids=str)
def test_adjusted_logits_in_the_memory_of_logits(over, fine):
    """Rows of 100 logits, 400 bytes: in place with the same stride, beside each other, but not shifted against each other."""
    if fine:
        assert takes(adjust, **over)
    else:
        with pytest.raises(H.ValidationError) as e:
            call(adjust, adjust(**over))
        assert e.value.message.startswith("out: "), e.value.message


def gathered(rng, es):
    """Strides of [batch][heads][rows] rows of 64 elements: nested in any order, or rows of two axes that interleave, in some places
    a little too close."""
    ext, order, strides, at = [rng.randint(1, 3) for _ in range(3)], rng.sample(range(3), 3), [0, 0, 0], 64
    for axis in order:
        strides[axis] = at + rng.choice([0, 0, 8, 64, 96])
        at = strides[axis] * rng.choice([ext[axis], ext[axis], 1, 2])
    return ext, strides


def taken(at, strides, ext, es):
    """The pieces of 16 bytes of all rows, in their order."""
    return [at // 16 + (b * strides[0] + h * strides[1] + r * strides[2]) * es // 16 + i
            for b in range(ext[0]) for h in range(ext[1]) for r in range(ext[2]) for i in range(64 * es // 16)]


@pytest.mark.parametrize("seed", range(400))
def test_gathered_rows_that_meet(seed):
    """Keys and values of any strides and distance: taken exactly where no two rows share memory."""
    rng = random.Random(seed)
    ext, ks = gathered(rng, 2)
    vs = list(ks)
    if rng.random() < 0.7:
        rng2 = random.Random(seed + 10 ** 6)
        _, vs = gathered(rng2, 2)
    v = P + 16 * rng.randint(-600, 600)
    pieces = taken(P, ks, ext, 2) + taken(v, vs, ext, 2)
    over = dict(k=P, v=v, batch=ext[0], pages_n_kv_head=ext[1], n_rows=ext[2], k_batch=ks[0], k_head=ks[1], k_row=ks[2], v_batch=vs[0],
                v_head=vs[1], v_row=vs[2])
    if len(set(pieces)) == len(pieces):
        assert takes(gather, **over)
    else:
        with pytest.raises(H.ValidationError) as e:
            call(gather, gather(**over))
        assert e.value.message.startswith("k, v: rows must not overlap"), e.value.message


I4 = {"pages_" + k: v for k, v in CODES.items()}


@pytest.mark.parametrize("over,match", [
    # keys [page][head][row], values [page][row][head] in one memory, a page's keys in front of its values
    (dict(pages_v=P + 2 * 8192, pages_k_page=16384, pages_v_page=16384, pages_v_head=64, pages_v_row=256), None),
    (dict(pages_v=P + 2 * 8064, pages_k_page=16384, pages_v_page=16384, pages_v_head=64, pages_v_row=256), "pages.k, v"),
    (dict(pages_v=P + 2 * 8192, pages_k_page=16384, pages_v_page=16256, pages_v_head=64, pages_v_row=256), "pages.k, v"),
    # one page: its stride is of no account
    (dict(pages_n_pages=1, pages_v=P + 128, pages_v_page=0), "pages.k, v"),
    # values inside the keys' range, their rows between the keys'
    (dict(pages_v=P + 128, pages_k_row=128, pages_k_head=4096, pages_k_page=16384, pages_v_row=128, pages_v_head=4096, pages_v_page=32768), None),
    (dict(pages_v=P + 128, pages_k_row=128, pages_k_head=4096, pages_k_page=16384, pages_v_row=64, pages_v_head=4096, pages_v_page=16384), "pages.k, v"),
    (dict(pages_v=P + 1000 * 16384, pages_n_pages=4000, pages_v_page=32768), "pages.k, v"),
    (dict(pages_v=P + 4000 * 16384, pages_n_pages=4000, pages_v_page=32768), None),
    # pairs behind a page's codes, and over them
    (dict(I4, pages_v=P + 4096, pages_k_page=8192 + 1024, pages_v_page=8192 + 1024, pages_k_params=P + 8192, pages_v_params=P + 8704,
          pages_k_params_page=4608, pages_v_params_page=4608), None),
    (dict(I4, pages_v=P + 4096, pages_k_page=8192 + 1024, pages_v_page=8192 + 1024, pages_k_params=P + 8192, pages_v_params=P + 8704,
          pages_k_params_page=4608, pages_v_params_page=4096), "pages.k"),
    (dict(I4, pages_v_params=P + 40), "pages.k, v: rows must not overlap those"), (dict(I4, pages_k_params=9 * P + 40900), "pages.k, v: rows must not overlap those"),
], ids=lambda x: str(x)[-70:])
def test_pages_that_meet(over, match):
    """Keys, values and pairs of any strides are written where none meets another; they may all be read."""
    assert takes(attention, **over) and takes(gather, **dict(over, **({"dtype": H.ITTS_F16} if over.get("pages_dtype") == H.ITTS_I4 else {})))
    if match is None:
        assert takes(append, **over)
    else:
        with pytest.raises(H.ValidationError) as e:
            call(append, append(**dict(over)))
        assert e.value.message.startswith(match), e.value.message


@pytest.mark.parametrize("kind,out", [(append, "q_out"), (attention, "out")])
@pytest.mark.parametrize("at,strides,fine", [(0, {}, True), (16, {}, False), (-256, {}, False), (2048, {}, False), (7 * 2048, {}, True), (-7 * 2048, {}, True),
                                             (0, dict(token=1024), False), (2048, dict(token=1024, q_token=1024), True),
                                             (2032, dict(token=1024, q_token=1024), False), (0, dict(n_tokens=1, token=4096), True),
                                             (256, dict(n_tokens=1), False)])
def test_queries_and_results_in_one_memory(kind, out, at, strides, fine):
    """7 tokens of 8 heads of 64, 2,048 bytes: in place with the same strides, or beside each other."""
    over = {out: P + at, **{f"{out}_token" if k == "token" else k: v for k, v in strides.items()}}
    if fine:
        assert takes(kind, **over)
    else:
        with pytest.raises(H.ValidationError) as e:
            call(kind, kind(**over))
        assert e.value.message.startswith(f"{out}: "), e.value.message


@pytest.mark.parametrize("kind,field,over", [
    (adjust, "rows", dict(rows=1 << 22, vocab=2049)), (adjust, "rows", dict(rows=1 << 22, vocab=16384)), (adjust, "rows", dict(rows=1 << 21, vocab=16385)),
    (adjust, None, dict(rows=(1 << 22) - 1, vocab=2049)), (adjust, None, dict(rows=(1 << 22) - 1, vocab=16384)), (adjust, None, dict(rows=1 << 23, vocab=2048)),
    (adjust, None, dict(rows=4095, vocab=1 << 24)), (adjust, "rows", dict(rows=4096, vocab=1 << 24)),
    (attention, "n_tokens", dict(n_tokens=1 << 20, batch=65535, n_head=512, n_kv_head=512)),
    (attention, "n_tokens", dict(n_tokens=1 << 19, batch=65535, n_head=1024, n_kv_head=512)),
    (attention, None, dict(n_tokens=1 << 20, batch=65535, n_head=100, n_kv_head=100)),
    (attention, None, dict(n_tokens=1 << 20, batch=1, n_head=512, n_kv_head=512))], ids=str)
def test_more_threads_than_a_launch_has(kind, field, over):
    """Sizes that are fine one by one, at and past what one launch holds."""
    over = dict(over)
    if kind is adjust:
        v = over["vocab"]
        over.update(logits=1 << 40, out=1 << 50, logits_row=v, out_row=v, allowed_row=0, history_row=0, bias_tokens_row=0, bias_row=0)
    else:
        h, hk = over["n_head"], over.pop("n_kv_head")
        over.update(q=1 << 40, out=1 << 50, q_token=64 * h, out_token=64 * h, pages_n_kv_head=hk)
    if field is None:
        assert takes(kind, **over)
    else:
        with pytest.raises(H.ValidationError) as e:
            call(kind, kind(**over))
        assert e.value.message.startswith(field), e.value.message


def test_cache_of_32_bits_is_float32():
    """32 bits of a type of 16 were given as 16; float32 need not say its bits."""
    for dtype in (torch.bfloat16, torch.float16):
        with pytest.raises(H.ValidationError, match="bits"):
            ops.paged_cache(3, 4, 16, 128, dtype, bits=32, device="cpu")
    with pytest.raises(H.ValidationError, match="bits"):
        ops.paged_cache(3, 4, 16, 128, bits=32, device="cpu")
    assert ops.paged_cache(3, 4, 16, 128, torch.float32, device="cpu").k.dtype == torch.float32
    assert ops.paged_cache(3, 4, 16, 128, torch.float16, device="cpu").k.dtype == torch.float16
