"""The operators of decoding over a paged cache, as cases that can be timed and checked.

A program that serves many sequences keeps their keys and values in pages that any sequence may
own, a table a sequence naming them in order.  The operators, through ``itts_hip.ops`` on device
tensors:

  append     new tokens' keys and values into their sequences' pages, rotated by their positions on
             the way, and their queries beside them (``ops.paged_append``); into a cache of 4 bits
             they are quantised, and read back as values (``ops.paged_gather``)
  attention  single tokens or whole pieces of prompts over the pages, all rows or a window and the
             first rows, over 16 and 32 bits or 4 (``ops.paged_attention``)
  gather     sequences' rows out of their pages into caches of one piece (``ops.paged_gather``)
  adjust     the step's logits under penalties for tokens that were there, biases and a grammar's
             mask (``ops.adjust_logits``)

``run`` computes them from elementary torch operations in 32 bits (64 where values are quantised),
or, with ``own`` set, through the framework; ``exact`` evaluates the definitions in 64 bits.

A cache of 4 bits holds each run of 64 elements of a row as codes c (two a byte, the lower half
first) and a pair (s, b) of float16: the values s c + b.
"""
import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "index-tts-rs_amd")
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_GROUP = 64  # elements that share a scale in 4 bits


def listed():
    return [
        # ---- append: q / kv are the types of tensors and cache; a sequence's new tokens new_lo..new_hi behind lo..hi rows;
        # rot: elements of a row that are rotated (0: none) ----
        # one sentence's next token, the speech decoder's heads and default cache, which knows positions: latency
        dict(name="append_step", op="append", q="f32", kv="bf16", batch=1, heads=20, kv_heads=20, dim=64, page=64,
             new_lo=1, new_hi=1, lo=234, hi=234, rot=0, interleaved=False),
        # prompts' pieces of many sequences at once into 4 bits, query heads sharing key heads
        dict(name="append_prompts", op="append", q="bf16", kv="int4", batch=12, heads=32, kv_heads=8, dim=128, page=32,
             new_lo=37, new_hi=1201, lo=0, hi=900, rot=128, interleaved=False),
        # ---- attention: lengths lo..hi count the new tokens; window 0: all rows ----
        # one token early in a sentence: latency
        dict(name="attn_step", op="attention", q="f32", kv="bf16", batch=1, heads=20, kv_heads=20, dim=64, page=64,
             new_lo=1, new_hi=1, lo=235, hi=235, window=0, sinks=0),
        # a decode step of many sequences, grouped heads, small pages
        dict(name="attn_batch", op="attention", q="bf16", kv="bf16", batch=64, heads=32, kv_heads=8, dim=128, page=16,
             new_lo=1, new_hi=1, lo=501, hi=6001, window=0, sinks=0),
        # the same over long sequences in 4 bits: the most rows
        dict(name="attn_4bit", op="attention", q="bf16", kv="int4", batch=16, heads=32, kv_heads=8, dim=128, page=64,
             new_lo=1, new_hi=1, lo=8191, hi=32768, window=0, sinks=0),
        # endless streams: the last rows and the first four, pages between given back
        dict(name="attn_stream", op="attention", q="f16", kv="f16", batch=24, heads=16, kv_heads=16, dim=64, page=32,
             new_lo=1, new_hi=3, lo=30011, hi=60000, window=4000, sinks=4),
        # pieces of prompts beside single tokens: the most arithmetic
        dict(name="attn_prompts", op="attention", q="bf16", kv="bf16", batch=6, heads=32, kv_heads=8, dim=128, page=64,
             new_lo=1, new_hi=2400, lo=1700, hi=6100, window=0, sinks=0),
        # four long utterances replayed in the reference's cache type, the conditioning and text rows in front staying in sight of
        # a window over the codes
        dict(name="attn_replay", op="attention", q="f32", kv="f32", batch=4, heads=20, kv_heads=20, dim=64, page=16,
             new_lo=547, new_hi=547, lo=547, hi=1200, window=256, sinks=232),
        # ---- gather: rows of a sequence ----
        # sequences that leave the batch for a cache of their own
        dict(name="gather_rows", op="gather", kv="bf16", batch=8, kv_heads=8, dim=128, page=16, lo=300, hi=2900),
        # a long sequence kept in 4 bits, as values
        dict(name="gather_4bit", op="gather", kv="int4", batch=1, kv_heads=8, dim=128, page=64, lo=9001, hi=9001),
        # ---- adjust: rows of logits, the tokens that were there, biases, a mask ----
        # the speech decoder's step late in an utterance
        dict(name="adjust_step", op="adjust", type="f32", rows=1, vocab=8194, history=1500, biases=0, masked=False),
        # a batch of constrained text
        dict(name="adjust_batch", op="adjust", type="bf16", rows=256, vocab=60510, history=2000, biases=50, masked=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


_HEADS = [(20, 20, 64), (16, 16, 64), (12, 4, 64), (32, 8, 128), (32, 4, 128), (8, 8, 128), (5, 5, 64), (6, 1, 128), (28, 4, 128)]
_PAIRS = [("f32", "bf16"), ("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "int4"), ("f16", "int4"), ("f32", "int4")]
_BYTES = {"f32": 4.0, "bf16": 2.0, "f16": 2.0, "int4": 0.5 + 4.0 / _GROUP}


def draw(rng):
    op = rng.choice(["append", "append", "attention", "attention", "attention", "attention", "gather", "adjust", "adjust"])
    page = rng.choice([16, 16, 32, 48, 64, 128, 256])
    heads, kv_heads, dim = rng.choice(_HEADS)
    q, kv = rng.choice(_PAIRS)
    batch = _log(rng, 1, 64)
    if op == "append":
        # within the largest listed case's elements
        most = 2.9e7 / (batch * (heads + 2 * kv_heads) * dim)
        new_hi = 1 if rng.random() < 0.4 else _log(rng, 1, max(1, int(most)))
        # (in 4 bits all rows come back as values)
        hi = _log(rng, 1, max(1, min(4000, int(1.4e7 / (batch * kv_heads * dim)) - new_hi)))
        return dict(op=op, q=q, kv=kv, batch=batch, heads=rng.choice([0, heads, heads]), kv_heads=kv_heads, dim=dim, page=page,
                    new_lo=rng.randint(0, new_hi), new_hi=new_hi, lo=rng.randint(0, hi), hi=hi,
                    rot=rng.choice([0, dim, dim, dim // 2, 48]), interleaved=rng.random() < 0.4)
    if op == "attention":
        window, sinks = rng.choice([(0, 0), (0, 0), (_log(rng, 1, 8000), rng.choice([0, 1, 4, _log(rng, 1, 300)]))])
        new_hi = 1 if rng.random() < 0.5 else _log(rng, 1, 2400)
        # within the largest listed cases' bytes of cache and arithmetic
        rate = 1.0 if q != "f32" else 0.25 if kv != "f32" else 0.08
        pairs = rate * 2.2e11 / (4.0 * batch * heads * dim)
        new_hi = max(1, min(new_hi, int(math.sqrt(pairs))))
        seen = max(1.0, min(6e8 / (batch * kv_heads * dim * 2 * _BYTES[kv]), pairs / new_hi))
        hi = _log(rng, 1, 60000 if window and seen > window + sinks + new_hi else max(1, min(60000, int(seen))))
        return dict(op=op, q=q, kv=kv, batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, page=page,
                    new_lo=rng.choice([new_hi, rng.randint(0, new_hi)]), new_hi=new_hi,
                    lo=rng.choice([hi, rng.randint(0, hi)]), hi=hi, window=window, sinks=sinks)
    if op == "gather":
        kv = rng.choice(["f32", "bf16", "f16", "int4"])
        hi = _log(rng, 1, max(1, min(20000, int(2.4e7 / (batch * kv_heads * dim)))))
        return dict(op=op, kv=kv, batch=batch, kv_heads=kv_heads, dim=dim, page=page, lo=rng.randint(0, hi), hi=hi)
    vocab = _log(rng, 70, 131072)
    return dict(op=op, type=rng.choice(["f32", "bf16", "f16"]), rows=_log(rng, 1, max(1, min(512, 15_000_000 // vocab))),
                vocab=vocab, history=rng.choice([0, _log(rng, 1, 8000), _log(rng, 1, 8000)]),
                biases=rng.choice([0, 0, _log(rng, 1, 300)]), masked=rng.random() < 0.5)


# ---- inputs ---------------------------------------------------------------------------------
def _gen(seed, device="cuda"):
    return torch.Generator(device=device).manual_seed(seed)


def _normal(g, shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _lengths(case):
    """The sequences' lengths: spread evenly from lo to hi, the longest first."""
    b, lo, hi = case["batch"], case["lo"], case["hi"]
    return [hi - (hi - lo) * i // max(1, b - 1) for i in range(b)]


def _new(case):
    """The sequences' new tokens: new_lo to new_hi, in another order than the lengths."""
    b, lo, hi = case["batch"], case["new_lo"], case["new_hi"]
    new = [hi - (hi - lo) * ((i * 5 + 1) % b if b % 5 else (i * 7 + 1) % b) // max(1, b - 1) for i in range(b)]
    return new if case["op"] == "append" else [min(n, length) for n, length in zip(new, _lengths(case))]


def _starts(case):
    starts = [0]
    for n in _new(case):
        starts.append(starts[-1] + n)
    return starts


def _seen_from(case, length, new):
    """The first row behind the sinks that any of a sequence's new tokens sees."""
    return max(0, length - new - case["window"] + 1) if case.get("window") else 0


def _table(case, rows, seed):
    """(table, pages): a table [batch][most pages] of pages in no order; -1 for those that hold no row that is seen."""
    size, table = case["page"], []
    new = _new(case) if case["op"] == "attention" else [0] * case["batch"]
    for length, n in zip(rows, new):
        first, sinks = _seen_from(case, length, n), case.get("sinks", 0)
        table.append([i * size < min(sinks, length) or (i + 1) * size > first for i in range(-(-length // size))])
    count = sum(map(sum, table)) + 3
    order = iter(torch.randperm(count, generator=_gen(seed, "cpu")).tolist())
    wide = max(1, max(map(len, table)))
    table = [[next(order) if used else -1 for used in row] + [-1] * (wide - len(row)) for row in table]
    return _ints(table), count


def _pages(case, count, g):
    """A cache's pages: (k, v, k's pairs, v's pairs), the pairs of a cache of 4 bits."""
    shape = (count, case["kv_heads"], case["page"], case["dim"])
    if case["kv"] != "int4":
        # keys share a direction (as after a layer norm's bias); values are centred
        k = _normal(g, shape)
        k += 0.5 * torch.randn((1, case["kv_heads"], 1, case["dim"]), generator=g, device="cuda")
        return k.to(_TYPES[case["kv"]]), _normal(g, shape, _TYPES[case["kv"]]), None, None
    out = []
    for _ in range(2):
        # codes with most in the middle, as bell-shaped values have
        a, b = (torch.randint(0, 256, (*shape[:3], shape[3] // 2), generator=g, device="cuda", dtype=torch.uint8) for _ in range(2))
        out.append(((a & 0x0f) + (b & 0x0f)) // 2 + (((a >> 4) + (b >> 4)) // 2 << 4))
        pair = torch.rand((*shape[:3], shape[3] // _GROUP, 2), generator=g, device="cuda")
        pair[..., 0] = 0.25 + 0.1 * pair[..., 0]
        pair[..., 1] = -2.4 + 0.8 * pair[..., 1]
        out.append(pair.half())
    return out[0], out[2], out[1], out[3]


def _rotation(case, rows):
    """[rows][rot]: the cosines, then the sines, of a row's rot / 2 angles."""
    n = case["rot"] // 2
    angle = torch.arange(rows, dtype=torch.float64).unsqueeze(1) * 10000.0 ** (-torch.arange(n, dtype=torch.float64) / n)
    return torch.cat([angle.cos(), angle.sin()], 1).float().cuda()


def prepare(case, seed):
    g = _gen(seed)
    if case["op"] == "adjust":
        r, v, n = case["rows"], case["vocab"], case["history"]
        x = 2.5 * _normal(g, (r, v))
        # some tokens come back often, places that are not used yet hold -1
        history = (v * torch.rand((r, n), generator=g, device="cuda") ** 2).int().clamp_(max=v - 1)
        history[:, 1::3] = history[:, :1] if n else 0
        used = torch.tensor([n - i * 7 % (n // 3 + 1) for i in range(r)], device="cuda").unsqueeze(1)
        history = history.masked_fill(torch.arange(n, device="cuda") >= used, -1)
        words = torch.randint(-2 ** 31, 2 ** 31, (r, (v + 31) // 32), generator=g, device="cuda") if case["masked"] else None
        biases = torch.stack([torch.randperm(v, generator=g, device="cuda")[:case["biases"]] for _ in range(r)]).int()
        return dict(case=case, logits=x.to(_TYPES[case["type"]]), history=history,
                    repetition=1.0 + torch.rand(r, generator=g, device="cuda"),
                    frequency=0.3 * torch.rand(r, generator=g, device="cuda"),
                    presence=0.5 * torch.rand(r, generator=g, device="cuda"), bias_tokens=biases,
                    bias=4.0 * _normal(g, biases.shape), allowed=None if words is None else words.int())
    lengths = _lengths(case)
    if case["op"] == "gather":
        table, count = _table(case, lengths, seed)
        return dict(case=case, cache=_pages(case, count, g), lengths=_ints(lengths), table=table)
    starts, d = _starts(case), case["dim"]
    state = dict(case=case, starts=_ints(starts), lengths=_ints(lengths))
    if case["op"] == "attention":
        state["table"], count = _table(case, lengths, seed)
        state["cache"] = _pages(case, count, g)
        state["q"] = (1.3 * _normal(g, (starts[-1], case["heads"], d))).to(_TYPES[case["q"]])
        return state
    rows = [length + n for length, n in zip(lengths, _new(case))]
    state["table"], count = _table(case, rows, seed)
    state["cache"] = _pages(case, count, g)
    # one product's result: queries, keys and values beside each other
    heads, hk, dtype = case["heads"], case["kv_heads"], _TYPES[case["q"]]
    x = _normal(g, (starts[-1], heads + 2 * hk, d))
    x[:, heads:heads + hk] += 0.5 * torch.randn((1, hk, d), generator=g, device="cuda")
    x = x.to(dtype)
    state["q"] = x[:, :heads] if heads else None
    state["k"], state["v"] = x[:, heads:heads + hk], x[:, heads + hk:]
    state["rotation"] = _rotation(case, max(rows) + 5) if case["rot"] else None
    return state


# ---- the plain forms ------------------------------------------------------------------------
def _values(codes, pairs):
    """The values of rows of 4 bits [..., dim / 2] with pairs [..., dim / 64, 2]."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()
    c = c.unflatten(-1, (-1, _GROUP))
    return (c * pairs[..., :1].float() + pairs[..., 1:].float()).flatten(-2)


def _rows(pages, pairs, ids):
    """A sequence's rows [heads][rows][dim] in 32 bits, from its pages' numbers."""
    x = pages.index_select(0, ids)
    x = _values(x, pairs.index_select(0, ids)) if pairs is not None else x.float()
    return x.transpose(0, 1).flatten(1, 2)


def _attention(s):
    case, starts, size = s["case"], _starts(s["case"]), s["case"]["page"]
    k_pages, v_pages, k_pairs, v_pairs = s["cache"]
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    window, sinks = case["window"], case["sinks"]
    out = torch.zeros_like(s["q"])
    for b, (length, n) in enumerate(zip(_lengths(case), _new(case))):
        if n == 0:
            continue
        first = _seen_from(case, length, n) // size
        front = min(-(-min(sinks, length) // size), first)  # pages with the first rows, then those of the window
        last = -(-length // size)
        ids = torch.cat([s["table"][b, :front], s["table"][b, first:last]]).long()
        at = torch.arange((front + last - first) * size, device=ids.device)
        at = torch.where(at < front * size, at, at + (first - front) * size)
        k, v = _rows(k_pages, k_pairs, ids), _rows(v_pages, v_pairs, ids)
        q = s["q"][starts[b]:starts[b + 1]].float().view(n, hk, h // hk, d).permute(1, 2, 0, 3).reshape(hk, -1, d)
        x = torch.matmul(q, k.transpose(1, 2).contiguous()) * (d ** -0.5)
        pos = torch.arange(length - n, length, device=ids.device).unsqueeze(1)
        sees = at <= pos
        if window:
            sees &= (at > pos - window) | (at < sinks)
        sees = sees.repeat(h // hk, 1)
        x = x.masked_fill(~sees, -math.inf)
        p = torch.exp(x - x.amax(-1, keepdim=True))
        o = torch.matmul(p, v.masked_fill((at >= length).unsqueeze(1), 0.0)) / p.sum(-1, keepdim=True)
        out[starts[b]:starts[b + 1]] = o.view(hk, h // hk, n, d).permute(2, 0, 1, 3).reshape(n, h, d).to(out.dtype)
    return out


def _places(s):
    """Each new token's (row in its sequence, page, row in the page)."""
    size, starts = s["case"]["page"], s["starts"].long()
    seq = torch.searchsorted(starts[1:].contiguous(), torch.arange(s["k"].shape[0], device=starts.device), right=True)
    row = s["lengths"].long()[seq] + torch.arange(s["k"].shape[0], device=starts.device) - starts[seq]
    return row, s["table"].long()[seq, row // size], row % size


def _rotate(x, table, row, interleaved):
    rot = table.shape[1]
    cos, sin = table[row].unsqueeze(1).to(x.dtype).chunk(2, -1)
    x, rest = x[..., :rot], x[..., rot:]
    a, b = (x[..., ::2], x[..., 1::2]) if interleaved else x.chunk(2, -1)
    turned = [a * cos - b * sin, b * cos + a * sin]
    return torch.cat([torch.stack(turned, -1).flatten(-2) if interleaved else torch.cat(turned, -1), rest], -1)


def _quantise(x):
    """Rows of values in 64 bits to (codes, pairs)."""
    x = x.unflatten(-1, (-1, _GROUP))
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale, base = ((hi - lo) / 15).half(), lo.half()
    step = torch.where(scale > 0, scale.double(), 1.0)
    c = ((x - base.double()) / step).round().clamp(0, 15)
    c = torch.where(scale > 0, c, 0.0).to(torch.uint8).flatten(-2)
    return c[..., ::2] | c[..., 1::2] << 4, torch.cat([scale, base], -1)


def _gather(s, lengths, rows):
    k_pages, v_pages, k_pairs, v_pairs = s["cache"]
    size, dtype = s["case"]["page"], torch.float32 if k_pairs is not None else k_pages.dtype
    at = torch.arange(rows, device=lengths.device)
    ids = s["table"].long()[:, at // size].clamp(min=0)                         # [batch][rows]
    live = (at < lengths.unsqueeze(1)).unsqueeze(1).unsqueeze(-1)
    out = []
    for pages, pairs in ((k_pages, k_pairs), (v_pages, v_pairs)):
        x = pages[ids, :, at % size]                                            # [batch][rows][heads][..]
        x = _values(x, pairs[ids, :, at % size]) if pairs is not None else x
        out.append(torch.where(live, x.transpose(1, 2), torch.zeros((), dtype=dtype, device=x.device)))
    return dict(k=out[0], v=out[1])


def _append(s):
    case, cache = s["case"], s["cache"]
    row, page, at = _places(s)
    wide = torch.float64 if case["kv"] == "int4" else torch.float32
    q, k, v = s["q"], s["k"].to(wide), s["v"].to(wide)
    if s["rotation"] is not None:
        k = _rotate(k, s["rotation"], row, case["interleaved"])
        q = None if q is None else _rotate(q.float(), s["rotation"], row, case["interleaved"]).to(q.dtype)
    for pages, pairs, x in ((cache[0], cache[2], k), (cache[1], cache[3], v)):
        if pairs is None:
            pages[page, :, at] = x.to(pages.dtype)
        else:
            pages[page, :, at], pairs[page, :, at] = _quantise(x)
    lengths = s["lengths"] + (s["starts"][1:] - s["starts"][:-1])
    out = dict(lengths=lengths) if q is None else dict(lengths=lengths, q=q)
    if case["kv"] != "int4":
        return dict(out, k=cache[0], v=cache[1])
    return dict(out, **_gather(s, lengths, _most_rows(case)))


def _most_rows(case):
    new = _new(case) if case["op"] == "append" else [0] * case["batch"]
    return max(1, max(length + n for length, n in zip(_lengths(case), new)))


def _adjust(s):
    x, v = s["logits"].float(), s["case"]["vocab"]
    h = s["history"].long()
    count = torch.zeros((x.shape[0], v + 1), device=x.device)
    count.scatter_add_(1, torch.where(h >= 0, h, v), torch.ones_like(h, dtype=torch.float32))
    count = count[:, :v]
    rep, freq, pres = (s[name].unsqueeze(1) for name in ("repetition", "frequency", "presence"))
    x = torch.where(count > 0, torch.where(x < 0, x * rep, x / rep) - (freq * count + pres), x)
    x = x.scatter_add(1, s["bias_tokens"].long(), s["bias"])
    if s["allowed"] is not None:
        bits = (s["allowed"].unsqueeze(-1) >> torch.arange(32, device=x.device, dtype=torch.int32)) & 1
        x = x.masked_fill(bits.flatten(1)[:, :v] == 0, -math.inf)
    return x.to(s["logits"].dtype)


def run(state):
    case, op = state["case"], state["case"]["op"]
    if not own:
        if op == "gather":
            return _gather(state, state["lengths"], _most_rows(case))
        return {"append": _append, "attention": _attention, "adjust": _adjust}[op](state)
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from itts_hip import ops

    if op == "adjust":
        biases = dict(bias_tokens=state["bias_tokens"], bias=state["bias"]) if case["biases"] else {}
        return ops.adjust_logits(state["logits"], history=state["history"], repetition=state["repetition"],
                                 frequency=state["frequency"], presence=state["presence"], allowed=state["allowed"], **biases)
    cache = ops.PagedCache(*state["cache"])
    if op == "attention":
        return ops.paged_attention(state["q"], cache, state["starts"], state["lengths"], state["table"],
                                   window=case["window"], sinks=case["sinks"])
    if op == "gather":
        k, v = ops.paged_gather(cache, state["lengths"], state["table"], _most_rows(case))
        return dict(k=k, v=v)
    lengths, q = ops.paged_append(cache, state["k"], state["v"], state["starts"], state["lengths"], state["table"],
                                  q=state["q"] if case["rot"] else None, rotation=state["rotation"],
                                  interleaved=case["interleaved"])
    q = state["q"] if q is None else q
    out = dict(lengths=lengths) if q is None else dict(lengths=lengths, q=q)
    if case["kv"] != "int4":
        return dict(out, k=cache.k, v=cache.v)
    k, v = ops.paged_gather(cache, lengths, state["table"], _most_rows(case))
    return dict(out, k=k, v=v)


def _pairs(case, length, n):
    """(query and row pairs of n tokens at the end of length rows, rows that any of them sees)."""
    window, sinks = case["window"] or length, case["sinks"]
    pairs = 0
    for pos in range(length - n, length):
        first = max(0, pos - window + 1)
        pairs += pos + 1 - first + min(sinks, first)
    first = max(0, length - n - window + 1)
    return pairs, length - first + min(sinks, first) if n else 0


def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}
    if case["op"] == "adjust":
        r, v = case["rows"], case["vocab"]
        each = 2 * v * size[case["type"]] + 4 * case["history"] + 8 * case["biases"] + 12 + (v // 8 if case["masked"] else 0)
        return dict(bytes=r * each, flops=2 * r * v)
    row = case["kv_heads"] * case["dim"] * 2  # elements of a row of keys and of values
    if case["op"] == "gather":
        rows = sum(_lengths(case))
        out = 4 if case["kv"] == "int4" else size[case["kv"]]
        return dict(bytes=int(rows * row * _BYTES[case["kv"]] + case["batch"] * _most_rows(case) * row * out),
                    flops=2 * rows * row if case["kv"] == "int4" else rows)
    if case["op"] == "append":
        new = sum(_new(case))
        q = case["heads"] * case["dim"] if case["rot"] else 0
        total = new * (size[case["q"]] * (2 * q + row) + _BYTES[case["kv"]] * row) + 4 * _most_rows(case) * case["rot"]
        if case["kv"] == "int4":
            total += sum(_lengths(case), new) * row * _BYTES["int4"] + case["batch"] * _most_rows(case) * row * 4
        return dict(bytes=int(total), flops=max(1, new * (3 * q + 2 * row)))
    h, d = case["heads"], case["dim"]
    pairs = rows = 0
    for length, n in zip(_lengths(case), _new(case)):
        p, seen = _pairs(case, length, n)
        pairs, rows = pairs + p, rows + seen
    return dict(bytes=int(rows * row * _BYTES[case["kv"]]) + 2 * sum(_new(case)) * h * d * size[case["q"]],
                flops=max(1, 4 * pairs * h * d))


# ---- the definitions in 64 bits -----------------------------------------------------------------
def _exact_rows(s, b, which, rows):
    """Rows `rows` of sequence b's keys (0) or values (1): [heads][rows][dim]."""
    size = s["case"]["page"]
    pages, pairs = s["cache"][which], s["cache"][2 + which]
    rows = torch.as_tensor(rows, dtype=torch.long, device=pages.device)
    page, at = s["table"][b].long()[rows // size], rows % size
    x = pages[page, :, at]
    if pairs is not None:
        c = torch.empty((*x.shape[:2], s["case"]["dim"]), dtype=torch.float64, device=x.device)
        c[..., 0::2], c[..., 1::2] = (x % 16).double(), (x // 16).double()
        pair = pairs[page, :, at].double().repeat_interleave(_GROUP, dim=2)
        x = pair[..., 0] * c + pair[..., 1]
    return x.double().permute(1, 0, 2)


def _exact_attention(s):
    case, q, starts = s["case"], s["q"], _starts(s["case"])
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for b, (length, n) in enumerate(zip(_lengths(case), _new(case))):
        if n == 0:
            continue
        first = _seen_from(case, length, n)
        rows = list(range(min(case["sinks"], first))) + list(range(first, length))
        at, pos = torch.tensor(rows, device=q.device), torch.arange(length - n, length, device=q.device).unsqueeze(1)
        hidden = at > pos
        if case["window"]:
            hidden |= (pos - at >= case["window"]) & (at >= case["sinks"])
        k, v = _exact_rows(s, b, 0, at), _exact_rows(s, b, 1, at)
        for head in range(case["heads"]):
            x = q[starts[b]:starts[b + 1], head].double() @ k[head // group].T / math.sqrt(case["dim"])
            out[starts[b]:starts[b + 1], head] = torch.softmax(x.masked_fill(hidden, -math.inf), -1) @ v[head // group]
    return out


def _exact_turn(x, s, rows):
    """x [tokens][heads][dim] rotated, element pair by element pair."""
    case, x = s["case"], x.double().clone()
    if s["rotation"] is None:
        return x
    n = case["rot"] // 2
    t = s["rotation"].double()[rows]
    for i in range(n):
        a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + n)
        xa, xb = x[..., a].clone(), x[..., b].clone()
        c, sn = t[:, i:i + 1], t[:, n + i:n + i + 1]
        x[..., a], x[..., b] = xa * c - xb * sn, xa * sn + xb * c
    return x


def _exact_append(s):
    case, starts, lengths = s["case"], _starts(s["case"]), _lengths(s["case"])
    new = _new(case)
    rows = torch.tensor([length + i for length, n in zip(lengths, new) for i in range(n)], dtype=torch.long, device="cuda")
    out = dict(lengths=torch.tensor([length + n for length, n in zip(lengths, new)], dtype=torch.int32))
    if s["q"] is not None:
        out["q"] = _exact_turn(s["q"], s, rows)
    size, table = case["page"], s["table"].cpu()
    for name, which in (("k", 0), ("v", 1)):
        x = _exact_turn(s[name], s, rows) if name == "k" else s[name].double()
        if case["kv"] == "int4":
            whole = torch.zeros((case["batch"], case["kv_heads"], _most_rows(case), case["dim"]), dtype=torch.float64, device="cuda")
            for b, (length, n) in enumerate(zip(lengths, new)):
                whole[b, :, :length] = _exact_rows(s, b, which, range(length))
                fresh = x[starts[b]:starts[b + 1]].reshape(n, case["kv_heads"], case["dim"] // _GROUP, _GROUP)
                lo, hi = fresh.min(-1, keepdim=True)[0], fresh.max(-1, keepdim=True)[0]
                scale, base = ((hi - lo) / 15).half().double(), lo.half().double()
                c = torch.clamp(torch.round((fresh - base) / scale), 0, 15)
                fresh = torch.where(scale == 0, base, scale * c + base)
                whole[b, :, length:length + n] = fresh.reshape(n, case["kv_heads"], case["dim"]).permute(1, 0, 2)
            out[name] = whole
        else:
            pages = s["cache"][which].double()
            for b, (length, n) in enumerate(zip(lengths, new)):
                for at in range(length, length + n, 1):
                    pages[int(table[b, at // size]), :, at % size] = x[starts[b] + at - length]
            out[name] = pages
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(s)
    if case["op"] == "append":
        return _exact_append(s)
    if case["op"] == "gather":
        out = {}
        for name, which in (("k", 0), ("v", 1)):
            x = torch.zeros((case["batch"], case["kv_heads"], _most_rows(case), case["dim"]), dtype=torch.float64, device="cuda")
            for b, length in enumerate(_lengths(case)):
                x[b, :, :length] = _exact_rows(s, b, which, range(length))
            out[name] = x
        return out
    out = []
    for i in range(case["rows"]):
        x = s["logits"][i].double()
        tokens = s["history"][i]
        count = torch.bincount(tokens[tokens >= 0].long(), minlength=case["vocab"]).double()
        rep, freq, pres = (float(s[name][i]) for name in ("repetition", "frequency", "presence"))
        there = count > 0
        x = torch.where(there & (x < 0), x * rep, torch.where(there, x / rep, x))
        x = x - freq * count - pres * there.double()
        for token, bias in zip(s["bias_tokens"][i].tolist(), s["bias"][i].tolist()):
            x[token] += bias
        if s["allowed"] is not None:
            t = torch.arange(case["vocab"], device=x.device)
            x[(s["allowed"][i].long()[t // 32] & 0xffffffff) >> t % 32 & 1 == 0] = -math.inf
        out.append(x)
    return torch.stack(out)
