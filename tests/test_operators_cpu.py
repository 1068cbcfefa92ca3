"""Refusals of the operators on device memory, without a GPU: wrong sizes, types, strides and
alignments at the C entries, and wrong tensors at the Python ones."""
import ctypes as C
import os
import subprocess
import sys

import pytest
import torch

import itts_hip as H
from itts_hip import ops

PKG = os.path.dirname(os.path.dirname(H.__file__))
P = 1 << 20  # an address that nothing reads: every call below is refused before its memory matters


def tree(**over):
    f = dict(q=P, k=P, v=P, out=P, lengths=P, parents=P, batch=2, n_nodes=5, n_head=4, n_kv_head=2, head_dim=64, max_seq=100,
             q_dtype=H.ITTS_F32, kv_dtype=H.ITTS_BF16, scale=0.125, q_batch=5 * 256, q_node=256, q_head=64, out_batch=5 * 256,
             out_node=256, out_head=64, k_batch=12800, k_head=6400, k_row=64, v_batch=12800, v_head=6400, v_row=64,
             parents_batch=5)
    f.update(over)
    return H.itts_tree_attention_args(**f)


def scores(**over):
    f = dict(logits=P, tokens=P, log_probs=P, entropy=P, top_tokens=P, top_log_probs=P, rows=3, vocab=100, n_tokens=1, top_n=5,
             dtype=H.ITTS_F32, logits_row=100, tokens_row=1)
    f.update(over)
    return H.itts_token_scores_args(**f)


def keep(**over):
    f = dict(k=P, v=P, lengths=P, path=P, new_lengths=2 * P, n_layer=2, batch=3, n_head=4, max_seq=50, head_dim=64, n_path=4,
             dtype=H.ITTS_BF16, k_layer=38400, k_batch=12800, k_head=3200, k_row=64, v_layer=38400, v_batch=12800, v_head=3200,
             v_row=64, path_batch=4)
    f.update(over)
    return H.itts_cache_keep_args(**f)


def call(kind, a):
    if kind is tree:
        return H._check(H.lib.itts_tree_attention(C.byref(a), None, 0, None))
    if kind is scores:
        return H._check(H.lib.itts_token_scores(C.byref(a), None, 0, None))
    return H._check(H.lib.itts_cache_keep(C.byref(a), None))


REFUSED = [
    (tree, "batch", dict(batch=-1)), (tree, "batch", dict(batch=65536)), (tree, "n_nodes", dict(n_nodes=257)),
    (tree, "n_nodes", dict(n_nodes=-1)), (tree, "n_kv_head", dict(n_kv_head=3)), (tree, "n_kv_head", dict(n_kv_head=0)),
    (tree, "n_kv_head", dict(n_head=0)), (tree, "head_dim", dict(head_dim=80)), (tree, "max_seq", dict(max_seq=0)),
    (tree, "scale", dict(scale=float("nan"))), (tree, "scale", dict(scale=float("inf"))),
    (tree, "kv_dtype", dict(q_dtype=H.ITTS_BF16, kv_dtype=H.ITTS_F32)), (tree, "kv_dtype", dict(kv_dtype=H.ITTS_F16)),
    (tree, "kv_dtype", dict(kv_dtype=9)), (tree, "q", dict(q=P + 8)), (tree, "q", dict(q_node=257)), (tree, "q", dict(q_head=-64)),
    (tree, "k", dict(k_row=60)), (tree, "v", dict(v=P + 2)), (tree, "v", dict(v_head=6404)), (tree, "out", dict(out_head=0)),
    (tree, "out", dict(out_node=2)), (tree, "parents", dict(parents_batch=-5)), (tree, "q, k, v", dict(q=None)),
    (tree, "q, k, v", dict(lengths=None)), (tree, "k", dict(k_row=1 << 60)),
    (scores, "rows", dict(rows=-1)), (scores, "vocab", dict(vocab=0)), (scores, "vocab", dict(vocab=(1 << 24) + 1)),
    (scores, "n_tokens", dict(n_tokens=-1)), (scores, "top_n", dict(top_n=65)), (scores, "top_n", dict(top_n=4, vocab=3)),
    (scores, "top_n", dict(top_n=-1)), (scores, "dtype", dict(dtype=0)), (scores, "logits", dict(logits=P + 2)),
    (scores, "logits_row", dict(logits_row=-100)), (scores, "logits", dict(logits=None)), (scores, "logits", dict(tokens=None)),
    (scores, "logits", dict(top_tokens=None)),
    (keep, "batch", dict(batch=-1)), (keep, "n_layer", dict(n_layer=-1)), (keep, "n_layer", dict(max_seq=0)),
    (keep, "dtype", dict(dtype=0)), (keep, "head_dim", dict(head_dim=12)), (keep, "k", dict(k_row=4)), (keep, "v", dict(v=P + 4)),
    (keep, "k, v", dict(k_row=0)), (keep, "path", dict(path_batch=-1)), (keep, "k, v", dict(path=None)),
    (keep, "new_lengths", dict(new_lengths=P)),
]


@pytest.mark.parametrize("kind,field,over", REFUSED, ids=lambda x: getattr(x, "__name__", str(x)))
def test_c_entries_refuse(kind, field, over):
    with pytest.raises(H.ValidationError) as e:
        call(kind, kind(**over))
    assert e.value.message.split(":")[0].startswith(field), e.value.message


def test_null_arguments():
    n = C.c_uint64()
    for f in (H.lib.itts_tree_attention, H.lib.itts_token_scores):
        with pytest.raises(H.ValidationError, match="args"):
            H._check(f(None, None, 0, None))
    with pytest.raises(H.ValidationError, match="args"):
        H._check(H.lib.itts_cache_keep(None, None))
    for f, a in ((H.lib.itts_tree_attention_workspace, tree()), (H.lib.itts_token_scores_workspace, scores())):
        with pytest.raises(H.ValidationError, match="args"):
            H._check(f(None, C.byref(n)))
        with pytest.raises(H.ValidationError, match="bytes"):
            H._check(f(C.byref(a), None))


def test_empty_calls_do_nothing():
    for a in (tree(batch=0, q=None), tree(n_nodes=0, q=None)):
        call(tree, a)
    call(scores, scores(rows=0, logits=None))
    call(keep, keep(batch=0, k=None))


def test_python_entries_refuse():
    q = torch.zeros(1, 2, 4, 64)
    for bad in (q, q[0], "q"):
        with pytest.raises(H.ValidationError, match="^.*q:"):
            ops.tree_attention(bad, q, q, torch.zeros(1, dtype=torch.int32), torch.zeros(1, 2, dtype=torch.int32))
    with pytest.raises(H.ValidationError, match="logits: a GPU tensor"):
        ops.token_scores(torch.zeros(2, 5))
    with pytest.raises(H.ValidationError, match="logits: float32"):
        ops.token_scores(torch.zeros(2, 5, dtype=torch.float64))
    with pytest.raises(H.ValidationError, match="k: a GPU tensor"):
        ops.cache_keep(torch.zeros(2, 1, 4, 8, 64), torch.zeros(2, 1, 4, 8, 64), torch.zeros(1, dtype=torch.int32),
                       torch.zeros(1, 2, dtype=torch.int32))


@pytest.mark.parametrize("kind,field,over", [
    (keep, "k, v", dict(v_head=6400, v_batch=25600, v_layer=76800)), (keep, "k, v", dict(v_row=128, v_head=6400)),
    (keep, "n_layer", dict(n_layer=1 << 20, n_head=1 << 10)), (scores, "rows", dict(rows=(1 << 23) + 1)),
], ids=lambda x: getattr(x, "__name__", str(x)))
def test_c_entries_refuse_overlaps_and_sizes_past_a_grid(kind, field, over):
    """One memory as keys and as values under two layouts; more blocks than a launch has."""
    test_c_entries_refuse(kind, field, over)


@pytest.mark.parametrize("kind,field,over", [
    (tree, "out", dict(out_node=256, out_head=256)), (tree, "out", dict(out_batch=256, out_node=64, out_head=64)),
    (tree, "out", dict(out_batch=1216)), (tree, "out", dict(batch=4, out_batch=128, out_node=192, n_nodes=4, out_head=10 ** 6)),
    (keep, "k, v", dict(v=99 * P, k_batch=6400)), (keep, "k, v", dict(v=99 * P, v_head=64, v_row=64)), (keep, "k, v", dict(v=99 * P, k_layer=12800)),
    (keep, "k, v", dict(v=P + 2 * 64)), (keep, "k, v", dict(v=P - 2 * 12800)), (keep, "k, v", dict(v=P + 16)),
], ids=lambda x: getattr(x, "__name__", str(x)))
def test_c_entries_refuse_axes_that_meet(kind, field, over):
    """Strides that each step over a row, but together reach the same one twice; values one row behind the keys."""
    test_c_entries_refuse(kind, field, over)


def takes(a, kind):
    """Whether the sizes pass: without a GPU the call then fails for that."""
    try:
        call(kind, a)
    except H.ValidationError as e:
        return "must not overlap" not in e.message
    except H.IttsError:
        pass
    return True


def test_rows_that_interleave_are_taken():
    """Heads between rows, sequences between heads, keys beside values; steps of two and three rows that never meet."""
    assert takes(tree(out_batch=64, out_node=512, out_head=128), tree)
    assert not takes(tree(out_batch=192, out_node=128, n_nodes=2, parents_batch=2, out_head=320, n_head=4), tree)  # 320 = 192 + 128
    assert takes(tree(out_batch=192, out_node=128, n_nodes=3, parents_batch=3, out_head=1024), tree)   # 0 2 4 | 3 5 7
    assert takes(tree(out_batch=0, batch=1), tree) and takes(tree(out_head=0, n_head=1, n_kv_head=1), tree)
    assert takes(keep(k_row=2 * 256, k_head=64, k_batch=2 * 12800 * 2, k_layer=2 * 12800 * 2 * 3, v=P + 2 * 256, v_row=2 * 256, v_head=64,
                      v_batch=2 * 12800 * 2, v_layer=2 * 12800 * 2 * 3), keep)
    assert takes(keep(v=P + 2 * 76800), keep) and takes(keep(v=P), keep)


@pytest.mark.parametrize("seed", range(6))
def test_overlaps_as_counted(seed):
    """Random strides of three axes against a count of every element."""
    import itertools
    import random

    rng = random.Random(seed)
    for _ in range(150):
        b, n, h = rng.randint(1, 4), rng.randint(1, 5), rng.choice([1, 2, 3, 4])
        st = [64 * rng.choice([0, 1, 1, 2, 3, 4, 5, 7, 12, 20]) + rng.choice([0, 0, 16]) for _ in range(3)]
        starts = [sum(i * s for i, s in zip(ix, st)) for ix in itertools.product(range(b), range(n), range(h))]
        starts.sort()
        meets = any(y - x < 64 for x, y in zip(starts, starts[1:]))
        a = tree(batch=b, n_nodes=n, n_head=h, n_kv_head=1, out_batch=st[0], out_node=st[1], out_head=st[2])
        assert takes(a, tree) == (not meets), (b, n, h, st)


@pytest.mark.parametrize("first", ["from itts_hip import ops; H.version()", "H.version(); from itts_hip import ops"])
def test_one_hip_runtime_or_a_refusal(first):
    """The library loads with its first call and then shares torch's HIP runtime; called before torch is there it has
    its own, and the operators say so (unless that is torch's too)."""
    code = (f"import sys; sys.path.insert(0, {PKG!r})\nimport itts_hip as H\nassert 'amdhip64' not in open('/proc/self/maps').read()\n"
            f"{first}\n"
            "print(len({l.split()[5] for l in open('/proc/self/maps') if 'libamdhip64' in l}))")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    if first.startswith("from"):
        assert r.returncode == 0 and r.stdout.split()[-1] == "1", r.stdout + r.stderr
    else:
        assert (r.returncode == 0 and r.stdout.split()[-1] == "1") or "different HIP runtimes" in r.stderr, r.stdout + r.stderr
