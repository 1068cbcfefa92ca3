"""The operators of drafted decoding, as cases that can be timed and checked.

A program that decodes with drafts proposes a tree of tokens after a sequence, has the model
score every node of it in one pass over the cached keys and values, and keeps the path that it
accepts.  The operators, through ``itts_hip.ops`` on device tensors:

  attention  attention of every node over its sequence's cached rows and its own ancestors
             (``ops.tree_attention``)
  scores     log-probabilities of given tokens, entropy and the most probable alternatives of
             rows of logits (``ops.token_scores``): what drafts are made from and judged by
  keep       the accepted nodes' key and value rows moved up behind the sequence's own, in every
             layer (``ops.cache_keep``)

``run`` computes them from elementary torch operations in 32 bits, or, with ``own`` set, through
the framework; ``exact`` evaluates the definitions in 64 bits.
"""
import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "index-tts-rs_amd")
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # ---- attention: q / kv are the types of queries and cache, lo..hi the lengths ----
        # a small draft early in a sentence, the speech decoder's heads and default cache: latency
        dict(name="attn_start", op="attention", q="f32", kv="bf16", batch=1, heads=20, kv_heads=20, dim=64,
             nodes=8, lo=235, hi=235, rows=2048, pad=False),
        # a wide draft at the end of a long utterance, the reference's cache type
        dict(name="attn_late", op="attention", q="f32", kv="f32", batch=1, heads=20, kv_heads=20, dim=64,
             nodes=33, lo=1734, hi=1734, rows=2048, pad=False),
        # eight sentences of different lengths, drafts of different sizes padded to the largest
        dict(name="attn_batch8", op="attention", q="f32", kv="bf16", batch=8, heads=20, kv_heads=20, dim=64,
             nodes=27, lo=250, hi=1400, rows=2048, pad=True),
        # single tokens of many sequences, query heads sharing key heads: no draft at all
        dict(name="attn_single", op="attention", q="bf16", kv="bf16", batch=32, heads=32, kv_heads=4, dim=128,
             nodes=1, lo=513, hi=4097, rows=4200, pad=False),
        # large drafts over ordinary contexts, grouped heads: the most arithmetic
        dict(name="attn_grouped", op="attention", q="bf16", kv="bf16", batch=12, heads=32, kv_heads=8, dim=128,
             nodes=64, lo=1000, hi=8191, rows=8320, pad=True),
        # few sequences with long contexts: the most bytes, split over the keys
        dict(name="attn_long", op="attention", q="f16", kv="f16", batch=2, heads=16, kv_heads=16, dim=64,
             nodes=61, lo=40001, hi=65500, rows=65600, pad=False),
        # ---- scores: rows of logits, given tokens per row, alternatives ----
        # one step of the speech decoder
        dict(name="scores_step", op="scores", type="f32", rows=1, vocab=8194, given=1, top=10, masked=False),
        # the nodes of a draft: every child's probability at its parent, the next draft's candidates
        dict(name="scores_draft", op="scores", type="f32", rows=64, vocab=8194, given=7, top=8, masked=True),
        # a replay of four prompts, each row's next code judged
        dict(name="scores_replay", op="scores", type="f32", rows=2188, vocab=8194, given=1, top=5, masked=False),
        # a text-sized vocabulary in 16 bits
        dict(name="scores_text", op="scores", type="bf16", rows=1000, vocab=60510, given=1, top=20, masked=False),
        # ---- keep: layers, sequences and heads of a cache, accepted nodes of a draft ----
        # one sentence's cache, the speech decoder's 24 layers
        dict(name="keep_one", op="keep", kv="bf16", layers=24, batch=1, kv_heads=20, dim=64, rows=2048,
             nodes=33, keep=5, lo=1200, hi=1200),
        # a batch of short ones with larger drafts
        dict(name="keep_batch", op="keep", kv="f32", layers=24, batch=8, kv_heads=8, dim=128, rows=300,
             nodes=64, keep=11, lo=17, hi=230),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "scores", "scores", "keep"])
    if op == "attention":
        q, kv = rng.choice([("f32", "bf16"), ("f32", "f32"), ("bf16", "bf16"), ("f16", "f16")])
        heads, kv_heads, dim = rng.choice([(20, 20, 64), (16, 16, 64), (12, 4, 64), (32, 8, 128), (32, 4, 128),
                                           (8, 8, 128), (5, 5, 64), (6, 1, 128)])
        nodes, batch = _log(rng, 1, 256), _log(rng, 1, 32)
        # within the largest listed cases' bytes of cache and arithmetic
        size = 4 if kv == "f32" else 2
        most = min(65000.0, 5e8 / (batch * kv_heads * dim * 2 * size),
                   (1.0 if q != "f32" else 0.25) * 4.5e10 / (4.0 * batch * heads * dim * nodes))
        hi = _log(rng, 1, max(1, int(most)))
        lo = max(0, hi - rng.choice([0, 0, rng.randint(0, hi)]))
        return dict(op=op, q=q, kv=kv, batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, nodes=nodes, lo=lo, hi=hi,
                    rows=hi + nodes + rng.randint(0, 100), pad=rng.random() < 0.5)
    if op == "scores":
        vocab = _log(rng, 70, 131072)
        rows = _log(rng, 1, max(1, min(4000, 60_000_000 // vocab)))
        return dict(op=op, type=rng.choice(["f32", "bf16", "f16"]), rows=rows, vocab=vocab, given=_log(rng, 1, 16),
                    top=rng.choice([0, 1, rng.randint(2, 20), rng.randint(21, 64)]), masked=rng.random() < 0.3)
    nodes = _log(rng, 2, 256)
    kv = rng.choice(["bf16", "f16", "f32"])
    hi = _log(rng, 1, 500)
    layers, batch, (kv_heads, dim) = _log(rng, 1, 32), _log(rng, 1, 8), rng.choice([(20, 64), (8, 128), (5, 64), (2, 128)])
    return dict(op="keep", kv=kv, layers=layers, batch=batch, kv_heads=kv_heads, dim=dim, nodes=nodes,
                keep=rng.randint(1, max(1, min(nodes // 2, 16))), lo=rng.randint(0, hi), hi=hi,
                rows=hi + nodes + rng.randint(0, 50))


# ---- inputs ---------------------------------------------------------------------------------
def _gen(seed, device="cuda"):
    return torch.Generator(device=device).manual_seed(seed)


def _normal(g, shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _lengths(case):
    """The sequences' lengths: spread evenly from lo to hi, the longest first."""
    b, lo, hi = case["batch"], case["lo"], case["hi"]
    return [hi - (hi - lo) * i // max(1, b - 1) for i in range(b)]


def _used(case):
    """The drafts' sizes: all nodes, or with padding down to about half of them."""
    n = case["nodes"]
    return [n - (i * 5) % (n // 2 + 1) if case["pad"] else n for i in range(case["batch"])]


def _tree(case, seed):
    """Parents [batch][nodes]: node 0 follows the sequence, every other one an earlier node (near
    ones more often); slots past a draft's size are marked unused (-2)."""
    g = _gen(seed, "cpu")
    n, batch = case["nodes"], case["batch"]
    par = torch.full((batch, n), -2, dtype=torch.int32)
    r = torch.rand((batch, n), generator=g)
    for b, used in enumerate(_used(case)):
        for i in range(used):
            par[b, i] = -1 if i == 0 else i - 1 - int(min(i, 12) * float(r[b, i]) ** 2)
    return par


def _accepted(case, seed):
    """Accepted paths [batch][keep], -1 past a path's end.  Kept nodes that move come from behind
    the kept ones' places, so that keeping once more changes nothing."""
    g = _gen(seed, "cpu")
    n, keep = case["nodes"], case["keep"]
    path = torch.full((case["batch"], keep), -1, dtype=torch.int32)
    for b in range(case["batch"]):
        m = keep - (b * 3) % keep
        free = torch.randperm(n - m, generator=g)[: m - 1] + m if n > m else torch.empty(0, dtype=torch.long)
        rows = [0] + sorted(free.tolist())
        path[b, : len(rows)] = torch.tensor(rows[:keep], dtype=torch.int32)
    return path


def prepare(case, seed):
    g = _gen(seed)
    if case["op"] == "attention":
        q, kv = _TYPES[case["q"]], _TYPES[case["kv"]]
        b, n, rows, d = case["batch"], case["nodes"], case["rows"], case["dim"]
        # keys share a direction (as after a layer norm's bias), some stand out; values are centred
        k = _normal(g, (b, case["kv_heads"], rows, d))
        k += 0.5 * torch.randn((1, case["kv_heads"], 1, d), generator=g, device="cuda")
        k[:, :, 0] *= 2.0
        return dict(case=case, k=k.to(kv), v=_normal(g, (b, case["kv_heads"], rows, d), kv),
                    q=(1.3 * _normal(g, (b, n, case["heads"], d))).to(q),
                    lengths=torch.tensor(_lengths(case), dtype=torch.int32, device="cuda"),
                    parents=_tree(case, seed).cuda())
    if case["op"] == "scores":
        r, v = case["rows"], case["vocab"]
        x = 2.5 * _normal(g, (r, v))
        # a few likely tokens a row
        like = torch.randint(0, v, (r, 6), generator=g, device="cuda")
        x.scatter_add_(1, like, 9.0 * torch.rand((r, 6), generator=g, device="cuda"))
        if case["masked"]:  # tokens that may not follow, the last one among them
            x[torch.rand((r, v), generator=g, device="cuda") < 0.3] = -math.inf
            x[:, -1] = -math.inf
        tokens = torch.randint(0, v, (r, case["given"]), generator=g, device="cuda")
        tokens[:, 0] = like[:, 0]
        return dict(case=case, logits=x.to(_TYPES[case["type"]]), tokens=tokens.int())
    b, rows, d = case["batch"], case["rows"], case["dim"]
    shape = (case["layers"], b, case["kv_heads"], rows, d)
    return dict(case=case, k=_normal(g, shape, _TYPES[case["kv"]]), v=_normal(g, shape, _TYPES[case["kv"]]),
                lengths=torch.tensor(_lengths(case), dtype=torch.int32, device="cuda"), path=_accepted(case, seed).cuda())


# ---- the plain forms ------------------------------------------------------------------------
def _ancestors(parents):
    """[batch][nodes][nodes]: whether node j is node i or one of its ancestors."""
    n = parents.shape[1]
    at = torch.arange(n, device=parents.device)
    one = (parents.unsqueeze(-1) == at).float() + torch.diag_embed((parents >= -1).float())
    steps = 1
    while steps < n:  # every product doubles the steps up the tree
        one = torch.matmul(one, one).clamp(max=1.0)
        steps *= 2
    return one > 0


def _attention(s):
    case, q, k, v = s["case"], s["q"].float(), s["k"], s["v"]
    b, n, h, d = q.shape
    hk, top = k.shape[1], case["hi"] + n
    k, v = k[:, :, :top].float(), v[:, :, :top].float()
    # query heads of one key head together: [batch][key head][group * nodes][dim]
    q = q.view(b, n, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)
    x = torch.matmul(q, k.transpose(2, 3).contiguous()) * (d ** -0.5)
    row = torch.arange(top, device=q.device)
    node = row.view(1, 1, -1) - s["lengths"].view(b, 1, 1)                     # [b][1][top]
    mask = _ancestors(s["parents"]).gather(2, node.clamp(0, n - 1).expand(b, n, top))
    mask = (mask & (node >= 0) & (node < n)) | ((node < 0) & (s["parents"] >= -1).unsqueeze(-1))
    mask = mask.repeat(1, h // hk, 1).unsqueeze(1)                             # [b][1][group * nodes][top]
    x = x.masked_fill(~mask, -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-3e38))
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    o = torch.where(mask.any(-1, keepdim=True), o, torch.zeros_like(o))
    return o.view(b, hk, h // hk, n, d).permute(0, 3, 1, 2, 4).reshape(b, n, h, d).to(s["q"].dtype)


def _scores(s):
    x, n = s["logits"].float(), s["case"]["top"]
    z = x - x.amax(-1, keepdim=True)
    e = torch.exp(z)
    lp = z - torch.log(e.sum(-1, keepdim=True))
    ent = -torch.where(e > 0, e * lp, torch.zeros_like(e)).sum(-1) / e.sum(-1)
    ids = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :n]  # ties: the lowest token first
    return dict(log_probs=lp.gather(1, s["tokens"].long()), entropy=ent, top_tokens=ids.int(),
                top_log_probs=lp.gather(1, ids))


def _keep(s):
    k, v, path, lengths = s["k"], s["v"], s["path"].long(), s["lengths"].long()
    live = path >= 0
    seq = torch.arange(path.shape[0], device=path.device).unsqueeze(1).expand_as(path)
    # slots past a path's end rewrite a row with itself
    to = lengths.unsqueeze(1) + torch.where(live, torch.arange(path.shape[1], device=path.device), 0)
    src = lengths.unsqueeze(1) + torch.where(live, path, path[:, :1])
    for t in (k, v):
        rows = t.permute(1, 3, 0, 2, 4)[seq, src]
        t.permute(1, 3, 0, 2, 4)[seq, to] = rows
    return dict(k=k, v=v, lengths=(lengths + live.sum(1)).int())


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"attention": _attention, "scores": _scores, "keep": _keep}[op](state)
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from itts_hip import ops

    if op == "attention":
        return ops.tree_attention(state["q"], state["k"], state["v"], state["lengths"], state["parents"])
    if op == "scores":
        r = ops.token_scores(state["logits"], state["tokens"], top_n=state["case"]["top"])
        return dict(log_probs=r.log_probs, entropy=r.entropy, top_tokens=r.top_tokens, top_log_probs=r.top_log_probs)
    lengths = ops.cache_keep(state["k"], state["v"], state["lengths"], state["path"])
    return dict(k=state["k"], v=state["v"], lengths=lengths)


def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}
    if case["op"] == "attention":
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        cached, pairs, q = 0, 0, 0
        for length, n in zip(_lengths(case), _used(case)):
            cached += length + n
            pairs += n * length + n  # (a node's other ancestors: few)
            q += n
        return dict(bytes=2 * cached * hk * d * size[case["kv"]] + 2 * q * h * d * size[case["q"]],
                    flops=4 * pairs * h * d)
    if case["op"] == "scores":
        r, v = case["rows"], case["vocab"]
        return dict(bytes=r * (v * size[case["type"]] + 8 * case["given"] + 4 + 8 * case["top"]), flops=6 * r * v)
    kept = int((_accepted(case, 0) >= 0).sum())
    row = case["layers"] * case["kv_heads"] * case["dim"] * size[case["kv"]] * 2
    return dict(bytes=2 * kept * row, flops=kept)


# ---- the definitions in 64 bits -----------------------------------------------------------------
def _exact_attention(s):
    q, k, v = s["q"], s["k"], s["v"]
    b, n, h, d = q.shape
    group = h // k.shape[1]
    out = torch.zeros((b, n, h, d), dtype=torch.float64, device=q.device)
    for i, length in enumerate(s["lengths"].tolist()):
        par = s["parents"][i].tolist()
        chain = torch.zeros((n, n), dtype=torch.bool)
        for j in range(n):
            if par[j] >= -1:
                chain[j, j] = True
                if par[j] >= 0:
                    chain[j] |= chain[par[j]]
        live = [j for j in range(n) if par[j] >= -1]
        sees = torch.cat([torch.ones((n, length), dtype=torch.bool), chain], 1)[live].to(q.device)
        for head in range(h):
            kk = k[i, head // group, : length + n].double()
            vv = v[i, head // group, : length + n].double()
            w = torch.softmax(((q[i, live, head].double() @ kk.T) / math.sqrt(d)).masked_fill(~sees, -math.inf), -1)
            out[i, live, head] = w @ vv
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(s)
    if case["op"] == "scores":
        out = dict(log_probs=[], entropy=[], top_tokens=[], top_log_probs=[])
        for x, t in zip(s["logits"].split(256), s["tokens"].split(256)):
            x = x.double()
            lse = torch.logsumexp(x, -1, keepdim=True)
            p = torch.exp(x - lse)
            order = torch.argsort(x, dim=-1, descending=True, stable=True)[:, : case["top"]]
            out["log_probs"].append(x.gather(1, t.long()) - lse)
            out["entropy"].append((p * torch.where(p > 0, lse - x, 0.0)).sum(-1))
            out["top_tokens"].append(order.int())
            out["top_log_probs"].append(x.gather(1, order) - lse)
        return {key: torch.cat(val) for key, val in out.items()}
    k, v = s["k"].clone(), s["v"].clone()
    lengths = s["lengths"].tolist()
    for b, path in enumerate(s["path"].tolist()):
        for i, j in enumerate(p for p in path if p >= 0):
            k[:, b, :, lengths[b] + i] = s["k"][:, b, :, lengths[b] + j]
            v[:, b, :, lengths[b] + i] = s["v"][:, b, :, lengths[b] + j]
        lengths[b] += sum(p >= 0 for p in path)
    return dict(k=k, v=v, lengths=torch.tensor(lengths, dtype=torch.int32))
