"""Decoding with drafts through the decoder: a tree of tokens in one step against the same tokens
stepped one by one (and the oracle), the rows that are kept, scores of codes, refusals."""
import sys

import numpy as np
import pytest

import ito
import itts_hip as H
from itts_hip import synth

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


_models = {}


def _model(bits=8, pd=H.ITTS_F16):
    if (bits, pd) not in _models:
        W = synth.make_weights(dict(synth.SMALL_CONFIG, quant_bits=bits, param_dtype=pd), seed=23, init="rich")
        _models[bits, pd] = (W, H.Gpt(W), ito.Model(W))
    return _models[bits, pd]


# as the prompts' tests: fp32 rows; bf16 rows round either way near the middle of two values
TOL = {H.ITTS_F32: 2e-5, H.ITTS_BF16: 2e-4}


def _tree(n, vocab, seed):
    r = np.random.default_rng(seed)
    return r.integers(0, vocab - 2, n).astype(np.int32), np.array([-1] + [int(r.integers(0, i)) for i in range(1, n)], np.int32)


def _path(parents, i):
    out = [i]
    while parents[out[0]] >= 0:
        out.insert(0, int(parents[out[0]]))
    return out


def _close(a, b, tol, what=""):
    d = np.abs(a - b).max()
    assert d < tol * max(1.0, np.abs(b).max()), f"{what}: {d:.2e} of {np.abs(b).max():.2f}"


# few-row products (up to 8 rows), LDS tiles (to 64, and past it)
@pytest.mark.parametrize("kv", [H.ITTS_F32, H.ITTS_BF16])
@pytest.mark.parametrize("bits,pd", [(8, H.ITTS_F16), (4, H.ITTS_F32)])
@pytest.mark.parametrize("n", [1, 5, 8, 9, 33, 64, 65, 256])
def test_tree_step_equals_single_steps(n, bits, pd, kv):
    say(f"[gpu] tree step n={n} bits={bits} pd={pd} kv={kv}")
    W, g, M = _model(bits, pd)
    pr = synth.make_prompt(W.cfg, 3, 20, seed=n)
    tokens, parents = _tree(n, W.cfg["mel_vocab"], n)
    cache, okv = g.kv_cache(420, kv), M.kv(420, kv_bf16=kv == H.ITTS_BF16)
    g.prefill(pr.text_tokens, pr.conds, pr.lang_id, cache)
    base = cache.valid_len()
    logits, r = g.step_tree(cache, tokens, parents, 2, scores=True, top_n=3)
    assert cache.valid_len() == base and logits.shape == (n, W.cfg["mel_vocab"])
    for i in sorted({0, n // 3, n // 2, n - 1}):
        path = _path(parents, i)
        M.prefill_after(okv, pr.text_tokens, pr.conds, pr.lang_id)
        for j, node in enumerate(path):
            want = M.step(okv, int(tokens[node]), 2 + j)
        _close(logits[i], want, TOL[kv], f"node {i}")
    # scores are those of the logits
    x = logits.astype(np.float64)
    lse = np.log(np.exp(x - x.max(1, keepdims=True)).sum(1)) + x.max(1)
    lp = np.array([0.0 if parents[i] < 0 else x[parents[i], tokens[i]] - lse[parents[i]] for i in range(n)])
    assert np.abs(r.log_probs - lp).max() < 1e-5
    assert np.array_equal(r.top_tokens, np.argsort(-logits, axis=1, kind="stable")[:, :3])
    assert np.abs(r.top_log_probs - (np.take_along_axis(x, r.top_tokens, 1) - lse[:, None])).max() < 1e-5
    p = np.exp(x - lse[:, None])
    assert np.abs(r.entropy - (p * (lse[:, None] - x)).sum(1)).max() < 1e-4
    # the deepest path kept: the cache then holds what single steps leave
    deep = max(range(n), key=lambda i: len(_path(parents, i)))
    path = _path(parents, deep)
    cache.keep(path)
    assert cache.valid_len() == base + len(path)
    single = g.kv_cache(420, kv)
    g.prefill(pr.text_tokens, pr.conds, pr.lang_id, single)
    for j, node in enumerate(path):
        g.step(single, int(tokens[node]), 2 + j, logits=False)
    for layer in (0, W.cfg["n_layer"] - 1):
        for is_v in (False, True):
            a, b = cache.read(layer, is_v), single.read(layer, is_v)
            # rows of a bf16 cache differ by a step at most where the values lie near a middle
            assert np.abs(a - b).max() <= (1e-4 if kv == H.ITTS_F32 else 2.0 ** -7) * max(1.0, np.abs(b).max())
    _close(g.step(cache, 7, 2 + len(path)), g.step(single, 7, 2 + len(path)), TOL[kv], "the next step")


def test_drafted_greedy_equals_greedy():
    """A whole decode with drafts (each step's best alternatives below the best token, some right and
    some wrong) gives the tokens of plain greedy steps."""
    say("[gpu] drafted greedy decoding")
    W, g, M = _model()
    pr = synth.make_prompt(W.cfg, 3, 15, seed=5)
    plain, cache = g.kv_cache(300, H.ITTS_F32), g.kv_cache(300, H.ITTS_F32)
    logits = g.prefill(pr.text_tokens, pr.conds, pr.lang_id, plain)
    want = []
    for i in range(60):
        want.append(int(np.argmax(logits)))
        logits = g.step(plain, want[-1], 2 + i)
    rng = np.random.default_rng(0)
    got, calls = [int(np.argmax(g.prefill(pr.text_tokens, pr.conds, pr.lang_id, cache)))], 0
    while len(got) < len(want):
        # the token just chosen, a guess of the next two (right every other time) and wrong siblings
        at = len(got)
        ahead = [want[at + j] if at + j < len(want) and rng.random() < 0.6 else int(rng.integers(0, 50)) for j in range(2)]
        tokens = [got[-1], ahead[0], (ahead[0] + 1) % 50, ahead[1], 3]
        parents = [-1, 0, 0, 1, 2]
        _, r = g.step_tree(cache, tokens, parents, 2 + at - 1, logits=False, top_n=1)
        calls += 1
        path = [0]
        while True:
            best = int(r.top_tokens[path[-1], 0])
            got.append(best)
            child = [i for i in range(5) if parents[i] == path[-1] and tokens[i] == best]
            if not child:
                break
            path.append(child[0])
        cache.keep(path)
    assert got[: len(want)] == want
    assert calls < len(want) - 5  # some drafts were accepted


def test_kept_nothing_and_dropped_trees():
    say("[gpu] dropped trees")
    W, g, M = _model()
    pr = synth.make_prompt(W.cfg, 3, 12, seed=6)
    a, b = g.kv_cache(200, H.ITTS_F32), g.kv_cache(200, H.ITTS_F32)
    for c in (a, b):
        g.prefill(pr.text_tokens, pr.conds, pr.lang_id, c)
    tokens, parents = _tree(12, W.cfg["mel_vocab"], 3)
    g.step_tree(a, tokens, parents, 2, logits=False)
    a.keep([])
    with pytest.raises(H.ValidationError, match="no drafted tree"):
        a.keep([0])
    assert np.array_equal(g.step(a, 9, 2), g.step(b, 9, 2))
    for drop in (lambda: g.step(a, 9, 3), lambda: H.step_batch(g, [a], [9], [3]), a.reset,
                 lambda: g.prefill(pr.text_tokens, pr.conds, pr.lang_id, a),
                 lambda: g.code_log_probs(pr.text_tokens, pr.conds, pr.lang_id, [1, 2], a),
                 lambda: H.generate_codes(g, pr.text_tokens, pr.conds, pr.lang_id, a,
                                          H.SamplingParams(greedy=True, max_mel_tokens=4), H.SamplerRng(0))):
        g.prefill(pr.text_tokens, pr.conds, pr.lang_id, a)
        g.step_tree(a, tokens, parents, 2, logits=False)
        drop()
        with pytest.raises(H.ValidationError, match="no drafted tree"):
            a.keep([0])


def test_code_scores():
    say("[gpu] code scores")
    W, g, M = _model()
    pr = synth.make_prompt(W.cfg, 3, 18, seed=8)
    codes = (np.arange(70, dtype=np.int32) * 37) % (W.cfg["mel_vocab"] - 2)
    cache = g.kv_cache(200, H.ITTS_F32)
    lp = g.code_log_probs(pr.text_tokens, pr.conds, pr.lang_id, codes, cache)
    r = g.code_scores(pr.text_tokens, pr.conds, pr.lang_id, codes, cache, top_n=4)
    assert cache.valid_len() == 0
    assert np.abs(r.log_probs - lp).max() < 4e-6
    x = g.forward_logits([H.CodePrompt(pr.text_tokens, pr.conds, pr.lang_id, codes[:-1])])[-len(codes):].astype(np.float64)
    lse = np.log(np.exp(x - x.max(1, keepdims=True)).sum(1, keepdims=True)) + x.max(1, keepdims=True)
    assert np.abs(r.entropy - (np.exp(x - lse) * (lse - x)).sum(1)).max() < 1e-4
    assert np.array_equal(r.top_tokens, np.argsort(-x, axis=1, kind="stable")[:, :4])
    assert np.abs(r.top_log_probs - (np.take_along_axis(x, r.top_tokens, 1) - lse)).max() < 1e-5
    few = g.code_scores(pr.text_tokens, pr.conds, pr.lang_id, codes[:1], cache)
    assert few.top_tokens.shape == (1, 0) and np.abs(few.log_probs - lp[:1]).max() < 4e-6


def test_refusals():
    say("[gpu] tree step refusals")
    W, g, M = _model()
    pr = synth.make_prompt(W.cfg, 3, 10, seed=9)
    cache, other = g.kv_cache(40, H.ITTS_F32), H.Gpt(synth.make_weights(synth.TINY_CONFIG, seed=3))
    g.prefill(pr.text_tokens, pr.conds, pr.lang_id, cache)
    V, P = W.cfg["mel_vocab"], W.cfg["mel_pos_len"]
    want = g.step_tree(cache, [1, 2], [-1, 0], 2)[0]

    def refuses(kind, match, tokens, parents, pos=2, **kw):
        with pytest.raises(kind, match=match):
            g.step_tree(cache, tokens, parents, pos, **kw)

    refuses(H.ValidationError, "n_nodes", [], [])
    refuses(H.ValidationError, "n_nodes", [1] * 257, [-1] * 257)
    refuses(H.ValidationError, "mel_token_id", [1, V], [-1, 0])
    refuses(H.ValidationError, "mel_token_id", [-1], [-1])
    refuses(H.ValidationError, "parents", [1, 2], [-1, 1])
    refuses(H.ValidationError, "parents", [1, 2], [-1, -2])
    refuses(H.ValidationError, "parents", [1, 2], [0, 0])
    refuses(H.ValidationError, "parents", [1, 2], [-1])
    refuses(H.ValidationError, "pos_idx", [1, 2], [-1, 0], P - 1)
    refuses(H.ValidationError, "pos_idx", [1], [-1], -1)
    refuses(H.ValidationError, "top_n", [1], [-1], top_n=65)
    refuses(H.ValidationError, "top_n", [1], [-1], top_n=-1)
    refuses(H.CapacityError, "kv_cache", [1] * 30, [-1] * 30)
    with pytest.raises(H.ValidationError, match="another decoder"):
        other.step_tree(cache, [1], [-1], 2)
    # refused calls leave the tree of the last good one
    for nodes, match in (([2], "out of range"), ([-1], "out of range"), ([1], "follows node 0"), ([0, 0], "follows"),
                         ([0, 1, 1], "follows")):
        with pytest.raises(H.ValidationError, match=match):
            cache.keep(nodes)
    base = cache.valid_len()
    cache.keep([0, 1])
    assert cache.valid_len() == base + 2
    again = g.kv_cache(40, H.ITTS_F32)
    g.prefill(pr.text_tokens, pr.conds, pr.lang_id, again)
    g.step(again, 1, 2)
    _close(g.step(again, 2, 3), want[1], 2e-5)
    other.close()


def test_tree_step_at_full_size(full_model):
    """The real shape late in an utterance: 24 layers, both cache types, against single steps."""
    W, g, M = full_model
    say("[gpu] tree step at full size")
    pr = synth.make_prompt(W.cfg, 32, 100, seed=31)
    prior = (np.arange(700, dtype=np.int32) * 11) % 8192
    tokens, parents = _tree(24, 8192, 4)
    for kv, tol in ((H.ITTS_F32, 1e-4), (H.ITTS_BF16, 5e-3)):
        cache = g.kv_cache(1024, kv)
        g.prefill_after(pr.text_tokens, pr.conds, pr.lang_id, prior, cache, logits=False)
        got, _ = g.step_tree(cache, tokens, parents, 702)
        for i in (0, 11, 23):
            path = _path(parents, i)
            g.prefill_after(pr.text_tokens, pr.conds, pr.lang_id, prior, cache, logits=False)
            for j, node in enumerate(path):
                want = g.step(cache, int(tokens[node]), 702 + j)
            assert np.abs(got[i] - want).max() < tol


def test_tree_step_of_many_heads():
    """A wide decoder's large tree: its attention's blocks share tiles and write the next product's operand themselves."""
    say("[gpu] tree step of 80 heads")
    W = synth.make_weights(dict(synth.SMALL_CONFIG, n_layer=1, n_head=80, d_model=5120, d_ffn=512), seed=29, init="rich")
    g = H.Gpt(W)
    pr = synth.make_prompt(W.cfg, 3, 20, seed=2)
    for n in (130, 256):
        cache = g.kv_cache(420, H.ITTS_BF16)
        tokens, parents = _tree(n, W.cfg["mel_vocab"], n)
        g.prefill(pr.text_tokens, pr.conds, pr.lang_id, cache)
        got, _ = g.step_tree(cache, tokens, parents, 2)
        for i in (0, n // 2, n - 1):
            g.prefill(pr.text_tokens, pr.conds, pr.lang_id, cache)
            for j, node in enumerate(_path(parents, i)):
                want = g.step(cache, int(tokens[node]), 2 + j)
            _close(got[i], want, TOL[H.ITTS_BF16], f"{n} nodes, node {i}")
    g.close()
