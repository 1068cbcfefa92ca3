"""The operators on device tensors (itts_hip.ops) against their definitions in float64.

Tolerances.  Attention: a score is a sum of dim products in float32, off by at most about
2 sqrt(dim) roundings of its products' magnitudes (A = sum |q k| scale), and one or two roundings on
its way through the exponential; a probability is then off by twice that, relative, and a row of
n keys sums to within 2 sqrt(n) roundings.  Outputs of 16 bits add half a step of the result, and
half a step of the probabilities that enter the product in that type (P = sum p |v|).
Scores: log-probabilities are differences of float32 numbers up to the row's range."""
import math
import sys

import pytest
import torch

import itts_hip as H

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24  # half a step of float32
HALF = {torch.float32: EPS, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [(F32, BF16), (F32, F32), (BF16, BF16), (F16, F16)]
NAN, INF = float("nan"), float("inf")


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def ops():
    from itts_hip import ops as o

    return o


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=F32):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ---- trees -------------------------------------------------------------------------------
def shape_tree(kind, n, seed=0):
    if kind == "chain":
        return [i - 1 for i in range(n)]
    if kind == "star":
        return [-1] + [0] * (n - 1)
    if kind == "forest":
        return [-1 if i % 5 == 0 else i - 1 - i % 2 * (i > 1) for i in range(n)]
    g = torch.Generator().manual_seed(seed)
    r = torch.rand(n, generator=g).tolist()
    return [-1 if i == 0 else int(r[i] * i) for i in range(n)]


def paths(par):
    """Each slot's nodes on its path to the root, [] for a slot that is not in the tree."""
    out = []
    for i, p in enumerate(par):
        if p == -1:
            out.append([i])
        elif 0 <= p < i and out[p]:
            out.append(out[p] + [i])
        else:
            out.append([])
    return out


def attention_ref(q, k, v, lengths, parents, scale=None, max_rows=None):
    """(result, tolerance) in float64, row by row over the rows that a node sees."""
    b, n, h, d = q.shape
    group = h // k.shape[1]
    scale = d ** -0.5 if scale is None else scale
    ref = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(ref)
    for i in range(b):
        length, pt = int(lengths[i]), paths([int(p) for p in parents[i]])
        live = max([j + 1 for j in range(n) if pt[j]], default=0)
        if length < 0 or length + live > (k.shape[2] if max_rows is None else max_rows):
            ref[i] = NAN
            continue
        for j in range(n):
            if not pt[j]:
                continue
            rows = list(range(length)) + [length + a for a in pt[j]]
            kk = k[i][:, rows].double().repeat_interleave(group, 0)
            vv = v[i][:, rows].double().repeat_interleave(group, 0)
            qq = q[i, j].double().unsqueeze(1)
            p = torch.softmax((qq * kk).sum(-1) * scale, -1).unsqueeze(-1)
            mag = (qq * kk).abs().sum(-1).amax(-1, keepdim=True) * abs(scale)
            pv = (p * vv.abs()).sum(1)
            ref[i, j] = (p * vv).sum(1)
            tol[i, j] = pv * EPS * (2 * 2 * (math.sqrt(d) + 2) * mag + 2 * math.sqrt(len(rows)) + 8)
            if q.dtype != F32:
                tol[i, j] += HALF[q.dtype] * (ref[i, j].abs() + pv)
    return ref, tol + 1e-30


def check(got, ref, tol, what=""):
    bad_nan = torch.isnan(ref) != torch.isnan(got.double())
    assert not bad_nan.any(), f"{what}: NaN in other places ({int(bad_nan.sum())})"
    d = (got.double() - ref).abs().nan_to_num(0.0)
    assert (d <= tol).all(), f"{what}: off by {(d / tol).max().item():.2f} of the tolerance"


def attention_case(ops, types, b, n, h, hk, d, lengths, kind, rows=None, seed=0, par=None):
    g = gen(seed)
    rows = rows or max(lengths) + n
    q, kv = types
    args = (1.5 * randn(g, b, n, h, d)).to(q), randn(g, b, hk, rows, d, dtype=kv), randn(g, b, hk, rows, d, dtype=kv)
    par = par or [shape_tree(kind, n, seed + i) for i in range(b)]
    return args, ints(lengths), ints(par)


# tiles of 32 keys, of 16 query rows, lengths and trees at and around them
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("n,h,hk,d,lengths,kind", [
    (1, 4, 4, 64, [0, 1, 31, 32, 33, 700], "chain"),
    (1, 8, 2, 128, [5, 0, 1000], "chain"),
    (2, 5, 5, 64, [30, 31, 0], "star"),
    (7, 3, 1, 64, [64, 1, 250], "tree"),
    (16, 2, 2, 64, [127, 16], "forest"),
    (17, 2, 2, 128, [95, 0], "tree"),
    (33, 6, 2, 64, [200, 3], "tree"),
    (63, 2, 1, 128, [66, 1], "chain"),
    (64, 2, 2, 64, [512, 0], "tree"),
    (65, 1, 1, 64, [33, 2], "star"),
    (200, 3, 3, 64, [77], "tree"),
    (256, 2, 1, 64, [0, 1500], "tree"),
    (256, 1, 1, 128, [31], "chain"),
])
def test_attention_matches_float64(ops, types, n, h, hk, d, lengths, kind):
    say(f"[gpu] tree attention {types} n={n} h={h}/{hk} d={d} {lengths} {kind}")
    (q, k, v), ln, par = attention_case(ops, types, len(lengths), n, h, hk, d, lengths, kind)
    check(ops.tree_attention(q, k, v, ln, par), *attention_ref(q, k, v, ln, par))


# long caches, split over blocks: few rows and many
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("n,h,hk,d,lengths", [(1, 2, 1, 64, [20011, 5]), (9, 2, 2, 128, [6007]), (40, 1, 1, 64, [9001, 0, 300])])
def test_attention_split_over_keys(ops, types, n, h, hk, d, lengths):
    say(f"[gpu] tree attention split {types} n={n} h={h}/{hk} d={d} {lengths}")
    (q, k, v), ln, par = attention_case(ops, types, len(lengths), n, h, hk, d, lengths, "tree", rows=max(lengths) + n + 3)
    got = ops.tree_attention(q, k, v, ln, par)
    check(got, *attention_ref(q, k, v, ln, par))
    assert torch.equal(got, ops.tree_attention(q, k, v, ln, par))  # the same bits each time
    # a tight bound on the rows changes the split, not what is computed
    short = ops.tree_attention(q, k, v, ln, par, max_length=max(lengths) + n)
    check(short, *attention_ref(q, k, v, ln, par))


@pytest.mark.parametrize("types", TYPES)
def test_attention_unused_slots(ops, types):
    """Slots that are no nodes, in every form, and slots below them: rows of zeros, and nothing of
    what their cache rows hold reaches the others."""
    say(f"[gpu] tree attention unused slots {types}")
    par = [[-1, -2, 0, 1, 2, 3, 9, -2], [-2] * 8, [-1, 0, 1, -7, 4, 5, 6, 2], [-2, -2, -2, -1, 3, 3, 4, 2 ** 31 - 1]]
    (q, k, v), ln, _ = attention_case(ops, types, 4, 8, 4, 2, 64, [40, 40, 0, 700], "tree", rows=720)
    for i, p in enumerate(par):
        for j, pt in enumerate(paths(p)):
            if not pt:
                k[i, :, int(ln[i]) + j] = NAN
                v[i, :, int(ln[i]) + j] = INF if j % 2 else NAN
    v[0, :, 48:] = NAN
    k[2, :, 8:] = INF
    got = ops.tree_attention(q, k, v, ln, ints(par))
    check(got, *attention_ref(q, k, v, ln, par))
    assert (got[1] == 0).all() and (got[0, 1] == 0).all()


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("value", [NAN, INF, -INF])
def test_attention_odd_values_stay_where_they_are_seen(ops, types, value):
    """A node whose value row holds an infinity or NaN: it reaches the nodes below it alone."""
    say(f"[gpu] tree attention odd values {types} {value}")
    par = [[-1, 0, 0, 1, 2, 3, 4, 4]]
    (q, k, v), ln, _ = attention_case(ops, types, 1, 8, 4, 2, 64, [50], "tree")
    v[0, 1, 52, 7] = value
    k[0, 0, 51, 3] = value  # node 1: a score of either infinity (by the query's sign) or NaN; -inf weighs nothing
    got = ops.tree_attention(q, k, v, ln, ints(par))
    ref, tol = attention_ref(q, k, v, ln, par)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(torch.isinf(got), torch.isinf(ref))
    fin = torch.isfinite(ref)
    assert torch.equal(got[~fin & ~torch.isnan(ref)].double(), ref[~fin & ~torch.isnan(ref)])
    assert ((got.double() - ref).abs()[fin] <= tol[fin]).all()
    assert fin[0, 0].all() and fin[0, 4, 0].all() and not fin[0, 4, 2:].all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("b,n,h,hk,d,rows", [(3, 8, 4, 2, 64, 300), (12, 72, 8, 8, 64, 300), (12, 48, 16, 2, 128, 300), (3, 130, 20, 20, 128, 2000)])
def test_attention_of_16_bits_rounds_its_result_alone(ops, dtype, b, n, h, hk, d, rows):
    """Whatever a launch's layout: a probability's two planes are off by 2^-16 (bf16: 8 bits and a rounded 8; fp16 2^-21,
    and less than 2^-33 of the largest) of it at most, in the product and in the sum, so that half a step of the result is nearly all."""
    say(f"[gpu] tree attention's rounding {dtype} {b} x {n} h={h}/{hk} d={d} rows={rows}")
    (q, k, v), ln, par = attention_case(ops, (dtype, dtype), b, n, h, hk, d, [rows - n - 7 * i for i in range(b)], "tree", rows=rows, seed=rows + d)
    got = ops.tree_attention(q, k, v, ln, par)
    some, nodes = sorted({0, b // 2, b - 1}), sorted({0, 1, n // 2, n - 1})
    ref, tol = attention_ref(q[some], k[some], v[some], ln[some], par[some])
    pv = attention_ref(q[some], k[some], v[some].abs(), ln[some], par[some])[0]  # the probabilities with the values' sizes
    tol = tol - HALF[dtype] * (ref.abs() + pv)                                   # (the float32 part)
    tol += HALF[dtype] * (ref.abs() + tol) + 2 * pv * (2.0 ** -16 + 2.0 ** -23 if dtype == BF16 else 2.0 ** -21) + 2.0 ** -33 * rows * 8
    check(got[some][:, nodes], ref[:, nodes], tol[:, nodes])


# each kernel and the joining of blocks: few rows, few rows over dealt keys, shared tiles, shared tiles over dealt keys
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("b,n,h,hk,d,rows", [
    (3, 8, 4, 2, 64, 90), (2, 33, 2, 2, 128, 90), (2, 150, 2, 1, 64, 200), (2, 21, 2, 2, 64, 9000), (12, 72, 8, 8, 64, 300),
    (3, 130, 20, 20, 128, 2000),
])
def test_attention_large_values_stay_where_they_are_seen(ops, types, b, n, h, hk, d, rows):
    """Rows of unused slots, inside the tree and behind it, hold the type's largest values, leaves' rows large ones: nothing
    of them reaches a node that does not see them, whose own values are small."""
    say(f"[gpu] tree attention large values {types} {b} x {n} h={h}/{hk} d={d} rows={rows}")
    g = gen(n)
    q, kv = types
    (q, k, v), ln, par = attention_case(ops, types, b, n, h, hk, d, [rows - n - 3 - 5 * i for i in range(b)], "star", rows=rows, seed=n)
    v *= 2.0 ** -6
    top = torch.finfo(kv).max
    par[:, 1::3] = -2                                       # unused slots between the root's children
    large = 65504.0 if kv == F16 else 2.0 ** 120            # (a child's own result is that large too, and finite)
    for i in range(b):
        at = int(ln[i])
        v[i, :, at + 2:at + n] = large
        v[i, :, at + 1:at + n:3] = top
        v[i, :, at + n:] = top
    got = ops.tree_attention(q, k, v, ln, par)
    some = sorted({0, b - 1})
    nodes = sorted({0, 1, 2, 3, n // 2, n - 1})
    ref, tol = attention_ref(q[some], k[some], v[some], ln[some], par[some])
    check(got[some][:, nodes], ref[:, nodes], tol[:, nodes])
    assert got[:, 0].abs().max() < 1.0 and torch.isfinite(got).all()


# (batch, nodes, heads, key heads, dim, rows) that lead to: tiles shared by a block's waves, one block a sequence and keys
# dealt to blocks, up to 64 nodes and more; four row tiles a wave, one block and dealt; a row tile a wave, dealt
LAYOUTS = [(12, 72, 8, 8, 64, 300), (12, 48, 16, 2, 128, 300), (16, 32, 20, 20, 64, 300), (12, 72, 8, 8, 64, 2000), (8, 72, 16, 16, 128, 1000),
           (8, 130, 16, 16, 64, 1000), (3, 130, 20, 20, 128, 2000), (8, 64, 32, 8, 128, 2500), (8, 48, 20, 20, 64, 300),
           (3, 48, 16, 2, 64, 8000), (2, 9, 4, 4, 64, 9000)]


def layout_case(ops, types, shape, kind, spread):
    """Sequences of lengths from what fits down to none, at and around tiles' borders; every third has unused slots."""
    b, n, h, hk, d, rows = shape
    lengths = [max(0, rows - n - spread * i - i % 3) for i in range(b)]
    lengths[-1] = 0 if b > 3 else 1
    if b > 4:
        lengths[1], lengths[2] = 32, 31
    (q, k, v), ln, par = attention_case(ops, types, b, n, h, hk, d, lengths, kind, rows=rows, seed=n + rows)
    for i in range(0, b, 3):
        par[i, 2 + i % 2::7] = -2
        par[i, n - 1 - i:] = -2
    return q, k, v, ln, par


def check_some(got, q, k, v, ln, par, what="", max_rows=None):
    """The first two sequences and the last (the reference goes row by row)."""
    some = sorted({0, 1, q.shape[0] - 1})
    ref, tol = attention_ref(q[some], k[some], v[some], ln[some], par[some], max_rows=max_rows)
    check(got[some], ref, tol, what)
    return ref


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("shape", LAYOUTS)
def test_attention_layouts(ops, types, shape):
    say(f"[gpu] tree attention layouts {types} {shape}")
    q, k, v, ln, par = layout_case(ops, types, shape, "tree", 17)
    got = ops.tree_attention(q, k, v, ln, par)
    check_some(got, q, k, v, ln, par)
    assert torch.equal(got, ops.tree_attention(q, k, v, ln, par))
    # lengths that do not fit, before the others and between them; a bound on the rows below the caches'
    ln[0], ln[-1] = -1, shape[5] - 10
    got = ops.tree_attention(q, k, v, ln, par, max_length=shape[5] - 5)
    check_some(got, q, k, v, ln, par, max_rows=shape[5] - 5)
    assert torch.isnan(got[0]).all() and torch.isnan(got[-1]).all()


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("shape", LAYOUTS)
def test_attention_layouts_hidden_and_odd_values(ops, types, shape):
    """Unused slots and rows behind the tree hold NaN and infinities, which no node gets; a node's own row holds one, which
    the nodes below it get."""
    say(f"[gpu] tree attention layouts, hidden and odd values {types} {shape}")
    q, k, v, ln, par = layout_case(ops, types, shape, "forest", 40)
    n, odd = shape[1], (INF, -INF, NAN)
    for i in (0, 1, shape[0] - 1):
        at = int(ln[i])
        for j, path in enumerate(paths(par[i].tolist())):
            if not path:
                k[i, :, at + j], v[i, :, at + j] = odd[j % 3], odd[(i + j) % 3]
        k[i, :, at + n:], v[i, :, at + n:] = NAN, odd[i % 3]
        v[i, 0, at + 1, 5], v[i, -1, at + 5, 9] = odd[i % 3], odd[(i + 1) % 3]
    got = ops.tree_attention(q, k, v, ln, par)
    some = sorted({0, 1, shape[0] - 1})
    ref, tol = attention_ref(q[some], k[some], v[some], ln[some], par[some])
    got, fin = got[some], torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(torch.isinf(got), torch.isinf(ref))
    assert torch.equal(got.double()[torch.isinf(ref)], ref[torch.isinf(ref)])
    assert ((got.double() - ref).abs()[fin] <= tol[fin]).all() and not fin.all()


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("shape", [LAYOUTS[0], LAYOUTS[1], LAYOUTS[6], LAYOUTS[9]])
def test_attention_layouts_strides_and_scales(ops, types, shape):
    say(f"[gpu] tree attention layouts, strides and scales {types} {shape}")
    q, k, v, ln, par = layout_case(ops, types, shape, "chain", 5)
    b, n, h, hk, d, rows = shape
    want = ops.tree_attention(q, k, v, ln, par)
    q2 = torch.empty(b, h, n, d + 16, dtype=q.dtype, device="cuda").transpose(1, 2)[..., :d]
    k2 = torch.empty(rows, b, hk, d, dtype=k.dtype, device="cuda").permute(1, 2, 0, 3)
    v2 = torch.empty(hk, b, rows + 9, 2 * d, dtype=v.dtype, device="cuda").transpose(0, 1)[:, :, 4:rows + 4, d:]
    for to, t in ((q2, q), (k2, k), (v2, v)):
        to.copy_(t)
    out = torch.full((b, h, n, d + 32), 7.0, dtype=q.dtype, device="cuda")
    got = ops.tree_attention(q2, k2, v2, ln, par, out=out.transpose(1, 2)[..., :d])
    assert torch.equal(got, want) and (out[..., d:] == 7.0).all()
    some = [0, b - 1]
    for scale in (1.0, -0.25, 0.0):
        ref, tol = attention_ref(q[some], k[some], v[some], ln[some], par[some], scale=scale)
        check(ops.tree_attention(q, k, v, ln, par, scale=scale)[some], ref, tol, f"scale {scale}")


@pytest.mark.parametrize("types", [(F32, BF16), (BF16, BF16), (F16, F16)])
def test_attention_shared_tiles_in_a_graph(ops, types):
    """Lengths and trees that change under a captured launch whose blocks share tiles and keys."""
    say(f"[gpu] tree attention: shared tiles in a graph {types}")
    q, k, v, ln, par = layout_case(ops, types, (3, 130, 20, 20, 128, 2000), "tree", 500)
    ops.tree_attention(q, k, v, ln, par)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = ops.tree_attention(q, k, v, ln, par)
    for turn, lengths in enumerate(([1870, 0, 3], [0, 0, 0], [-1, 1871, 1870], [700, 900, 1100])):
        ln.copy_(ints(lengths))
        par.copy_(ints([shape_tree(("tree", "star", "chain")[(turn + i) % 3], 130, turn) for i in range(3)]))
        want = ops.tree_attention(q, k, v, ln, par)
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.nan_to_num(7.0), want.nan_to_num(7.0)), lengths
        check(out[1:2], *attention_ref(q[1:2], k[1:2], v[1:2], ln[1:2], par[1:2]))


@pytest.mark.parametrize("value", [INF, -INF])
@pytest.mark.parametrize("n,h,hk,d,length", [(1, 2, 2, 64, 290), (1, 4, 2, 128, 9000), (9, 8, 2, 64, 700), (72, 8, 8, 64, 300), (48, 16, 2, 128, 300),
                                             (72, 8, 8, 64, 2000), (130, 16, 16, 64, 900)])
def test_attention_infinities_of_small_weights(ops, value, n, h, hk, d, length):
    """Float16: keys whose weight is 2^-40 and 2^-100 of the others' sum hold an infinity in one element, which is then the result's; the
    finite ones stay as they are."""
    say(f"[gpu] tree attention infinities of small weights {value} n={n} h={h}/{hk} d={d} length={length}")
    g = gen(22)
    x = torch.ones(1, n, h, d, device="cuda", dtype=F16)
    k, v = (torch.zeros(1, hk, length + n, d, device="cuda", dtype=F16) for _ in range(2))
    v.copy_(randn(g, *v.shape))
    ln, par = ints([length]), ints([[-1] + [0] * (n - 1)])
    scale = 1.0 / d                                          # a score is a key's elements
    k[:, :, :length] = -28.0                                 # 2^-40
    k[:, :, :length:8] = 0.0                                 # (some in every tile: the maximum is theirs for every wave)
    k[:, :, 3:length:64] = -69.0                             # 2^-99.5
    v[:, 0, 67, 5] = v[:, 0, 131, 40] = value                # such a key's, among keys that all nodes see
    v[:, 1, 100, 17] = value                                 # one of the first kind
    got = ops.tree_attention(x, k, v, ln, par, scale=scale)
    rows = sorted({0, 1 % n, n - 1})
    ref, tol = attention_ref(x, k, v, ln, par, scale=scale) if n < 10 else (None, None)
    if ref is not None:
        inf = torch.isinf(ref)
        assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(got.double()[inf], ref[inf])
        assert ((got.double() - ref).abs()[~inf] <= tol[~inf]).all()
    group = h // hk
    odd = torch.zeros(h, d, dtype=torch.bool, device="cuda")
    odd[:group, 5] = odd[:group, 40] = odd[group:2 * group, 17] = True
    assert (got[0, rows][:, odd] == value).all() and torch.isfinite(got[0, rows][:, ~odd]).all()


@pytest.mark.parametrize("types", [(F32, BF16), (F32, F32), (BF16, BF16)])
def test_attention_blocks_of_no_weight(ops, types):
    """A block's keys lie so far below the row's largest score that their weight is 0 as a float: what their values are, finite
    or not, is then neither raised nor lost in the joining."""
    say(f"[gpu] tree attention: a block without weight {types}")
    q, kv = types
    g = gen(21)
    x = torch.ones(1, 2, 2, 64, device="cuda", dtype=q)
    k, v = (0.05 * randn(g, 1, 2, 9000, 64)).to(kv), randn(g, 1, 2, 9000, 64, dtype=kv)
    k[:, :, :4000], k[:, :, 5], k[:, :, 8000] = -25.0, -24.75, 2.5   # scores -200, -198 and 20, the others' about 0
    v[:, :, 5] = 1e38
    ln, par = ints([8990]), ints([[-1, 0]])
    check(ops.tree_attention(x, k, v, ln, par), *attention_ref(x, k, v, ln, par))
    v[:, 0, 5] = INF
    got = ops.tree_attention(x, k, v, ln, par)
    assert (got[:, :, 0] == INF).all() and torch.isfinite(got[:, :, 1]).all()


def test_attention_lengths_that_do_not_fit(ops):
    say("[gpu] tree attention lengths that do not fit")
    lengths = [-1, 57, 56, 2 ** 31 - 1, -2 ** 31, 0]
    (q, k, v), _, par = attention_case(ops, (F32, BF16), 6, 8, 4, 4, 64, [56] * 6, "tree", rows=64)
    ln = ints(lengths)
    got = ops.tree_attention(q, k, v, ln, par)
    check(got, *attention_ref(q, k, v, ln, par))
    assert torch.isnan(got[[0, 1, 3, 4]]).all() and torch.isfinite(got[[2, 5]]).all()
    part = ops.tree_attention(q, k, v, ln, par, max_length=60)
    assert torch.isnan(part[2]).all() and torch.equal(part[5], got[5])
    # 100 rows behind the bound, split over blocks
    (q, k, v), _, par = attention_case(ops, (F32, BF16), 2, 4, 1, 1, 64, [9000, 9000], "tree", rows=9100)
    got = ops.tree_attention(q, k, v, ints([9000, 8999]), par, max_length=9003)
    assert torch.isnan(got[0]).all() and torch.isfinite(got[1]).all()


@pytest.mark.parametrize("types", TYPES)
def test_attention_strides(ops, types):
    """Heads before nodes, rows with gaps, caches laid out row by row, one cache for all sequences."""
    say(f"[gpu] tree attention strides {types}")
    (q, k, v), ln, par = attention_case(ops, types, 3, 6, 4, 2, 64, [40, 90, 0], "tree", rows=100)
    want = ops.tree_attention(q, k, v, ln, par)
    q2 = torch.empty(3, 4, 6, 80, dtype=q.dtype, device="cuda").transpose(1, 2)[..., :64]
    q2.copy_(q)
    k2 = torch.empty(3, 100, 2, 64, dtype=k.dtype, device="cuda").transpose(1, 2)
    k2.copy_(k)
    v2 = torch.empty(2, 3, 120, 128, dtype=v.dtype, device="cuda").transpose(0, 1)[:, :, 10:110, 64:]
    v2.copy_(v)
    out = torch.full((3, 4, 6, 96), 7.0, dtype=q.dtype, device="cuda")
    par2 = torch.zeros(3, 11, dtype=torch.int32, device="cuda")
    par2[:, :6] = par
    got = ops.tree_attention(q2, k2, v2, ln, par2[:, :6], out=out.transpose(1, 2)[..., :64])
    assert torch.equal(got, want) and (out[..., 64:] == 7.0).all()
    shared = ops.tree_attention(q, k[:1].expand(3, -1, -1, -1), v[:1].expand(3, -1, -1, -1), ln, par)
    check(shared, *attention_ref(q, k[:1].expand(3, -1, -1, -1), v[:1].expand(3, -1, -1, -1), ln, par))


@pytest.mark.parametrize("types", TYPES)
def test_attention_large_scores(ops, types):
    """Scores far apart, early and late (the running maximum moves), and negative scales."""
    say(f"[gpu] tree attention large scores {types}")
    (q, k, v), ln, par = attention_case(ops, types, 2, 12, 2, 2, 64, [900, 333], "tree")
    for key, f in ((0, 30.0), (5, 3.0), (400, 20.0), (899, 40.0)):
        k[:, :, key] *= f
    for scale in (0.125, 1.0, -0.5, 0.0):
        ref, tol = attention_ref(q, k, v, ln, par, scale=scale)
        check(ops.tree_attention(q, k, v, ln, par, scale=scale), ref, tol, f"scale {scale}")


def test_attention_past_32_bits(ops):
    """A cache of more than 2^32 bytes (and 2^31 elements): the last sequence's rows lie behind them."""
    say("[gpu] tree attention past 2^31 elements")
    d = 64
    big_k = torch.as_strided(torch.zeros(2_300_000_000, dtype=BF16, device="cuda"), (2, 1, 600, d),
                             (2_200_000_000 // d * d, 600 * d, d, 1))
    g = gen(3)
    big_k.copy_(randn(g, 2, 1, 600, d))
    q, v = randn(g, 2, 3, 1, d, dtype=BF16), big_k.flip(0).contiguous()
    ln, par = ints([500, 590]), ints([[-1, 0, 1]] * 2)
    check(ops.tree_attention(q, big_k, v, ln, par), *attention_ref(q, big_k, v, ln, par))


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("n,h,hk,d,rows,lengths", [
    (1, 2, 1, 64, 24000, [(i * 7919) % 23990 if i % 3 else i % 5 - 1 for i in range(150)]),  # more sequences than lanes
    (3, 2, 2, 64, 9000, [8990] + [0] * 20), (3, 2, 2, 64, 9000, [0, -1, 7, 31, 8997, 8998, 2 ** 31 - 1]),
    (20, 8, 2, 128, 9000, [1, 8000, 333, 4096, 2500]), (64, 8, 2, 128, 6000, [5900, 17, 3001]), (130, 2, 2, 64, 7000, [6850, 64, 1700]),
])
def test_attention_keys_dealt_to_blocks(ops, types, n, h, hk, d, rows, lengths):
    """Sequences of any lengths over one cache (stride 0 between them) that is long enough for its keys to be
    dealt to a launch's blocks in equal parts: parts that end inside tiles and sequences, sequences of one
    part, of many, without rows, and ones that do not fit."""
    say(f"[gpu] tree attention dealt {types} n={n} h={h}/{hk} d={d} {len(lengths)} lengths")
    b, (q, kv) = len(lengths), types
    g = gen(b + n)
    x = (1.5 * randn(g, b, n, h, d)).to(q)
    k, v = (randn(g, 1, hk, rows, d, dtype=kv).expand(b, -1, -1, -1) for _ in range(2))
    par = ints([shape_tree("tree", n, i) for i in range(b)])
    got = ops.tree_attention(x, k, v, ints(lengths), par)
    some = sorted(set(range(0, b, max(1, b // 12))) | {b - 1})  # (the reference goes row by row)
    check(got[some][:, ::9], *(t[:, ::9] for t in attention_ref(x[some], k[some], v[some], [lengths[i] for i in some], par[some])))
    for i, length in enumerate(lengths):
        assert torch.isnan(got[i]).all() == (length < 0 or length + n > rows)


def test_attention_graph_follows_lengths(ops):
    """A captured launch deals its keys by the lengths of each replay."""
    say("[gpu] tree attention: lengths change under a graph")
    g = gen(12)
    q, k, v = randn(g, 3, 5, 4, 64), randn(g, 3, 2, 12000, 64, dtype=BF16), randn(g, 3, 2, 12000, 64, dtype=BF16)
    par, ln = ints([shape_tree("tree", 5, i) for i in range(3)]), ints([11000, 5, 6000])
    ops.tree_attention(q, k, v, ln, par)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = ops.tree_attention(q, k, v, ln, par)
    for lengths in ([0, 0, 0], [11995, 11995, 11995], [1, -1, 900], [11996, 3, 40], [11000, 5, 6000]):
        ln.copy_(ints(lengths))
        want = ops.tree_attention(q, k, v, ln, par)
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.nan_to_num(7.0), want.nan_to_num(7.0)), lengths
        check(out, *attention_ref(q, k, v, lengths, par))


# ---- scores --------------------------------------------------------------------------------
def scores_ref(x, tokens, top):
    x = x.double().cpu()
    m = x.amax(-1, keepdim=True)
    z = torch.where(m == -INF, torch.full_like(x, -INF), x - m)  # nothing but -inf: no probability at all
    # log of the sum, less the maximum's own 1: log(1 + 2e-24) is 0 in float64 where log1p(2e-24) is 2e-24
    others = torch.exp(z).scatter(1, z.argmax(-1, keepdim=True), 0.0).sum(-1, keepdim=True)
    others = torch.where(torch.isnan(m) | torch.isinf(m), m + m * 0.0, others)  # (NaN: no such row has a sum)
    lp = torch.where(m == -INF, z, z - torch.log1p(others))
    p = torch.exp(lp)
    ent = -torch.where(p == 0, 0.0, p * lp).sum(-1)
    order = torch.sort(torch.where(torch.isnan(x), -INF, x), dim=-1, descending=True, stable=True)[1][:, :top]
    t = tokens.long().cpu()
    given = lp.gather(1, t.clamp(0, x.shape[1] - 1))
    given = torch.where(t == -1, 0.0, torch.where((t < 0) | (t >= x.shape[1]), NAN, given))
    return given, ent, order.int(), lp.gather(1, order.long())


def scores_check(r, x, tokens, top):
    given, ent, order, best = scores_ref(x, tokens, top)
    assert torch.equal(r.top_tokens.cpu(), order)
    v = x.shape[1]
    # x - m is exact to half a step of the range; the sum's terms are off by their arguments' rounding (exp of a
    # rounded argument), the sum by 2 sqrt(v) / 2^24 at most; log1p and the last subtraction round once more
    fin = x.double().cpu()
    fin = torch.where(torch.isfinite(fin), fin, 0.0)
    rng = float(fin.max() - fin.min()) + math.log(v) + 1
    for got, ref in ((r.log_probs, given), (r.top_log_probs, best)):
        got, ref = got.double().cpu(), ref
        same = (got == ref) | (torch.isnan(got) & torch.isnan(ref))
        tol = EPS * (4 * ref.abs().nan_to_num(0, 0, 0) + (8 + math.log2(v)) * 2 * (1 - torch.exp(ref)).abs().nan_to_num(0) + 1e-3)
        off = (got - ref).abs()
        assert (same | (off <= tol)).all(), (off / tol)[~same].max()
    same = (r.entropy.double().cpu() == ent) | (torch.isnan(ent) & torch.isnan(r.entropy.cpu()))
    tol = EPS * (16 + 2 * math.log2(v) + 2 * rng) * ent + 1e-37
    off = (r.entropy.double().cpu() - ent).abs()
    assert (same | (off <= tol)).all(), (off / tol)[~same].max()


def logits(g, r, v, dtype, spread=3.0):
    return (spread * randn(g, r, v)).to(dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("r,v,given,top", [
    (1, 1, 1, 1), (3, 2, 2, 2), (1, 8194, 1, 10), (64, 8194, 7, 8), (5, 63, 3, 63), (5, 65, 3, 64), (2, 255, 1, 3), (2, 257, 1, 64),
    (9, 1000, 1, 0), (2, 4097, 16, 20), (300, 513, 1, 5), (3, 60510, 1, 20), (1, 131072, 4, 64), (2, 200003, 2, 33),
])
def test_scores_match_float64(ops, dtype, r, v, given, top):
    say(f"[gpu] scores {dtype} {r} x {v}, {given} given, top {top}")
    g = gen(r * v + top)
    x = logits(g, r, v, dtype)
    tokens = torch.randint(0, v, (r, given), generator=g, device="cuda").int()
    scores_check(ops.token_scores(x, tokens, top), x, tokens, top)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("v", [17001, 33000])
def test_scores_of_many_long_rows(ops, dtype, v):
    """Rows that one block reads in several turns, and whose best tokens come first, last or in between."""
    say(f"[gpu] scores of 600 rows of {v} {dtype}")
    g = gen(v)
    x = logits(g, 600, v, dtype)
    ramp = torch.linspace(0, 12, v, device="cuda")
    x[0], x[1], x[2], x[3] = ramp.to(dtype), (-ramp).to(dtype), -(ramp - 6).abs().to(dtype), (ramp - 6).abs().to(dtype)
    x[4] = -INF
    x[4, -1], x[4, 8200] = 1.0, 2.0
    # the twelfth is one of three alike: the row's last token, which is read in the first turn, and two of later ones
    x[5:8] = -5.0
    x[5:8, 100:111], x[5:8, -1] = 10.0, 3.0
    x[6, 16900], x[7, 16500:16510] = 3.0, 3.0
    # the same value in every place but the first turn's
    x[8], x[9, :16384], x[9, 16384:] = 1.0, 0.0, 1.0
    tokens = torch.randint(0, v, (600, 2), generator=g, device="cuda").int()
    scores_check(ops.token_scores(x, tokens, 12), x, tokens, 12)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("v", [70, 8194, 40000])
def test_scores_ties_masks_and_odd_values(ops, dtype, v):
    say(f"[gpu] scores ties, masks and odd values {dtype} {v}")
    g = gen(v)
    x = logits(g, 12, v, dtype, 2.0)
    x[0] = 1.5                                  # all alike
    x[1] = -INF                                 # nothing allowed
    x[2] = -INF
    x[2, v - 1] = 2.0                           # one token
    x[3, torch.randperm(v, generator=g, device="cuda")[: v // 2]] = -INF
    x[4] = (x[4] * 2).round() / 2               # many ties
    x[5] = torch.arange(v, device="cuda").to(dtype) / v        # rising: the best last
    x[6] = -torch.arange(v, device="cuda").to(dtype) / v
    x[7, v // 3] = NAN
    x[8, 5] = INF
    x[9, 3], x[9, 9] = -0.0, 0.0
    x[9] = torch.where(x[9] > 0, -x[9], x[9])   # the zeros of both signs come first, in their order
    x[10, v // 2] = 60.0                        # nearly all the probability: entropy near 0
    x[11] = torch.finfo(dtype).min              # a mask of the type's lowest value, in every place but one
    x[11, 7] = 0.0
    tokens = torch.randint(0, v, (12, 5), generator=g, device="cuda").int()
    tokens[:, 1] = -1
    tokens[:, 2] = v - 1
    tokens[::2, 3], tokens[1::2, 3] = v, -2
    tokens[10, 4] = v // 2
    for top in (1, 64):
        scores_check(ops.token_scores(x, tokens, top), x, tokens, top)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("v", [1030, 1300, 1543, 2047, 20000])
def test_scores_few_waves_and_masked_ranges(ops, dtype, v):
    """Vocabularies that leave a block's last waves without tokens, and masks that allow one range of them."""
    say(f"[gpu] scores {v} {dtype}: waves without tokens")
    g = gen(v + 1)
    x = logits(g, 9, v, dtype)
    for i, (lo, hi) in enumerate(((0, 70), (500, 1029), (100, 101), (v - 40, v), (0, v - 1), (256, 512))):
        x[i, :lo], x[i, hi:] = -INF, -INF
    tokens = torch.randint(0, v, (9, 2), generator=g, device="cuda").int()
    for top in (1, 5, 20, 64):
        scores_check(ops.token_scores(x, tokens, top), x, tokens, top)


def test_scores_forms(ops):
    """One token a row, none, rows with gaps and rows that do not start at 16 bytes."""
    say("[gpu] scores forms")
    g = gen(1)
    for dtype in (F32, BF16, F16):
        whole = logits(g, 6, 3011, dtype)
        x = whole[:, 3:3000]
        t = torch.randint(0, x.shape[1], (6, 4), generator=g, device="cuda").int()
        scores_check(ops.token_scores(x, t[:, ::2][:, :1].contiguous(), 4), x, t[:, :1], 4)
        r = ops.token_scores(x, t[:, 0].contiguous(), 4)
        assert r.log_probs.shape == (6,)
        assert torch.equal(r.log_probs, ops.token_scores(x, t, 0).log_probs[:, 0])
        a, b = ops.token_scores(x, None, 4), ops.token_scores(x.contiguous(), t[:, 1:3], 4)
        assert a.log_probs is None and torch.equal(a.top_tokens, b.top_tokens) and torch.equal(a.entropy, b.entropy)
        scores_check(b, x, t[:, 1:3], 4)
        assert ops.token_scores(x[:0], t[:0], 4).top_tokens.shape == (0, 4)


# ---- kept rows -----------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("layers,b,h,d,rows", [(1, 1, 1, 64, 40), (3, 4, 5, 64, 300), (2, 3, 2, 128, 290), (1, 2, 3, 24, 60)])
def test_keep_matches_copies(ops, dtype, layers, b, h, d, rows):
    say(f"[gpu] keep {dtype} {layers} x {b} x {h} x {rows} x {d}")
    g = gen(rows)
    for n_path in (1, 2, 7, 33):
        k, v = randn(g, layers, b, h, rows, d, dtype=dtype), randn(g, layers, b, h, rows, d, dtype=dtype)
        lengths = torch.randint(0, max(1, rows - 40), (b,), generator=g, device="cuda").int()
        path = torch.full((b, n_path), -1)
        for i in range(b):
            m = n_path - i % (n_path + 1)
            path[i, :m] = torch.randperm(min(40, rows - int(lengths[i])))[:m].sort()[0]
            if i == 1 and n_path > 2:
                path[i] = torch.arange(n_path)  # nothing moves
        wk, wv, want = k.clone(), v.clone(), lengths.clone()
        for i in range(b):
            for j, p in enumerate(path[i].tolist()):
                if p < 0:
                    break
                wk[:, i, :, int(lengths[i]) + j] = k[:, i, :, int(lengths[i]) + p]
                wv[:, i, :, int(lengths[i]) + j] = v[:, i, :, int(lengths[i]) + p]
                want[i] += 1
        new = ops.cache_keep(k, v, lengths, path.int().cuda())
        assert torch.equal(new, want) and torch.equal(k, wk) and torch.equal(v, wv)


def test_keep_refuses_paths_on_the_device(ops):
    """Paths that do not rise or leave the cache, negative lengths: nothing moves, -1 comes back, and
    the other sequences are served."""
    say("[gpu] keep: paths out of order and out of range")
    g = gen(5)
    k, v = randn(g, 2, 7, 2, 50, 64), randn(g, 2, 7, 2, 50, 64)
    k0, v0 = k.clone(), v.clone()
    lengths = ints([10, 10, 10, -1, 50, 48, 2 ** 31 - 1])
    path = ints([[0, 2, 2], [3, 1, -1], [0, 40, -1], [0, 1, 2], [0, -1, -1], [1, -1, 5], [0, 1, -1]])
    new = ops.cache_keep(k, v, lengths, path)
    assert new.tolist() == [-1, -1, -1, -1, -1, 49, -1]
    k0[:, 5, :, 48], v0[:, 5, :, 48] = k0[:, 5, :, 49], v0[:, 5, :, 49]
    assert torch.equal(k, k0) and torch.equal(v, v0)


def test_keep_strides_and_four_dimensions(ops):
    say("[gpu] keep strides")
    g = gen(6)
    base = randn(g, 3, 40, 2, 5, 64, dtype=BF16)
    k = base.permute(0, 3, 2, 1, 4)           # [3][5][2][40][64], rows interleaved
    v = randn(g, 3, 5, 2, 60, 80, dtype=BF16)[:, :, :, 4:44, 16:]
    wk, wv = k.clone(), v.clone()
    lengths, path = ints([3, 0, 30, 7, 12]), ints([[0, 4, 9]] * 5)
    for i, n in enumerate(lengths.tolist()):
        for j, p in enumerate((0, 4, 9)):
            wk[:, i, :, n + j], wv[:, i, :, n + j] = k[:, i, :, n + p], v[:, i, :, n + p]
    four_k, four_v = k[1].clone(), v[1].contiguous()
    assert torch.equal(ops.cache_keep(k, v, lengths, path), lengths + 3)
    assert torch.equal(k, wk) and torch.equal(v, wv)
    assert torch.equal(ops.cache_keep(four_k, four_v, lengths, path), lengths + 3)
    assert torch.equal(four_k, wk[1]) and torch.equal(four_v, wv[1])


def test_keep_of_one_memory_for_keys_and_values(ops):
    """k and v the same tensor: its rows move once (twice, rows would follow that have moved already)."""
    say("[gpu] keep: v is k")
    g = gen(8)
    k = randn(g, 3, 2, 4, 40, 64)
    lengths, path = ints([5, 20]), ints([[1, 2, 4, 7], [0, 3, 9, -1]])
    want = k.clone()
    for i, (n, p) in enumerate(((5, (1, 2, 4, 7)), (20, (0, 3, 9)))):
        for j, node in enumerate(p):
            want[:, i, :, n + j] = k[:, i, :, n + node]
    assert ops.cache_keep(k, k, lengths, path).tolist() == [9, 23]
    assert torch.equal(k, want)


@pytest.mark.parametrize("shape", [(2, 3, 0, 40, 64), (0, 3, 2, 40, 64), (0, 3, 0, 40, 64), (3, 0, 40, 64)])
def test_keep_of_caches_without_layers_or_heads(ops, shape):
    """No rows to move: the lengths alone, and -1 for paths that are refused."""
    say(f"[gpu] keep without rows {shape}")
    k, v = torch.zeros(shape, dtype=BF16, device="cuda"), torch.zeros(shape, dtype=BF16, device="cuda")
    new = ops.cache_keep(k, v, ints([5, 0, 38]), ints([[1, 2, -1], [2, 1, -1], [0, 1, 2]]))
    assert new.tolist() == [7, -1, -1]


# ---- streams, graphs, refusals -----------------------------------------------------------------
def drafted(ops, s):
    """The three as they are used: a draft's attention, its scores, the accepted rows kept."""
    o = ops.tree_attention(s["q"], s["k"], s["v"], s["lengths"], s["parents"])
    r = ops.token_scores(o.flatten(2)[:, :, :500].reshape(-1, 500), s["tokens"], 5)
    k, v = s["k"].clone(), s["v"].clone()
    new = ops.cache_keep(k, v, s["lengths"], s["path"])
    again = ops.tree_attention(s["q"], k, v, new, s["parents"])
    return [o, r.log_probs, r.entropy, r.top_tokens, r.top_log_probs, k, v, new, again]


def drafted_state(seed, rows=2600):
    g = gen(seed)
    ln = [rows - 20 - 100 * i for i in range(3)]
    par = ints([shape_tree("tree", 9, seed + i) for i in range(3)])
    return dict(q=randn(g, 3, 9, 8, 64), k=randn(g, 3, 8, rows, 64, dtype=BF16), v=randn(g, 3, 8, rows, 64, dtype=BF16),
                lengths=ints(ln), parents=par, tokens=torch.randint(0, 500, (27, 2), generator=g, device="cuda").int(),
                path=ints([[0, 3, 5], [0, -1, -1], [1, 2, 8]]))


def test_run_of_all_three(ops):
    say("[gpu] a draft's attention, scores and kept rows together")
    s = drafted_state(11)
    o, lp, ent, top, toplp, k, v, new, again = drafted(ops, s)
    check(o, *attention_ref(s["q"], s["k"], s["v"], s["lengths"], s["parents"]))
    x = o.flatten(2)[:, :, :500].reshape(-1, 500)
    scores_check(ops.token_scores(x, s["tokens"], 5), x, s["tokens"], 5)
    assert new.tolist() == [n + c for n, c in zip(s["lengths"].tolist(), (3, 1, 3))]
    check(again, *attention_ref(s["q"], k, v, new, s["parents"]))


def test_streams(ops):
    """Two streams at once, and tensors made on another stream than the one that uses them."""
    say("[gpu] operators on two streams")
    states = [drafted_state(s) for s in (1, 2)]
    want = [drafted(ops, s) for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    for _ in range(3):
        got = []
        for st, s in zip(streams, states):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got.append(drafted(ops, s))
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_graphs(ops):
    """Captured and replayed on new inputs, two graphs in one pool, eager work in between."""
    say("[gpu] operators in graphs")
    states = [drafted_state(s) for s in (3, 4)]
    for s in states:
        drafted(ops, s)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in states:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(drafted(ops, s))
        graphs.append(gr)
    for turn in range(3):
        new = [drafted_state(10 + 2 * turn + i) for i in range(2)]
        want = [drafted(ops, s) for s in new]
        for s, n in zip(states, new):
            for key in s:
                s[key].copy_(n[key])
        torch.cuda.synchronize()
        for gr in graphs:
            gr.replay()
        drafted(ops, new[0])
        torch.cuda.synchronize()
        for a, b in zip(want, outs):
            assert all(torch.equal(x, y) for x, y in zip(a, b)), turn


def test_gpu_refusals(ops):
    say("[gpu] operator refusals")
    (q, k, v), ln, par = attention_case(ops, (F32, BF16), 2, 4, 4, 2, 64, [10, 20], "tree")

    def refuses(match, f, *a, **kw):
        with pytest.raises(H.ValidationError, match=match):
            f(*a, **kw)

    t = ops.tree_attention
    refuses("lengths", t, q, k, v, ln.long(), par)
    refuses("lengths", t, q, k, v, ln.cpu(), par)
    refuses("parents", t, q, k, v, ln, par[:, :3])
    refuses("k:", t, q, k[:1], v[:1], ln, par)
    refuses("v:", t, q, k, v.float(), ln, par)
    refuses("kv_dtype", t, q.half(), k, v, ln, par)
    refuses("q:", t, q[..., ::2], k, v, ln, par)
    wide = torch.zeros(2, 2, 24, 72, dtype=BF16, device="cuda")
    refuses("k: rows", t, q, wide[..., 4:68], wide[..., :64], ln, par)
    refuses("head_dim", t, q[..., :32], k[..., :32], v[..., :32], ln, par)
    refuses("max_length", t, q, k, v, ln, par, max_length=1000)
    refuses("max_seq", t, q, k, v, ln, par, max_length=0)
    refuses("out", t, q, k, v, ln, par, out=q.half())
    refuses("out: rows", t, q, k, v, ln, par, out=torch.empty(1, 4, 4, 64, device="cuda").expand(2, 4, 4, 64))
    refuses("scale", t, q, k, v, ln, par, scale=NAN)
    refuses("q: requires", t, q.clone().requires_grad_(), k, v, ln, par)
    refuses("tokens", ops.token_scores, torch.zeros(2, 9, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda"))
    refuses("tokens", ops.token_scores, torch.zeros(2, 9, device="cuda"), torch.zeros(2, device="cuda"))
    refuses("top_n", ops.token_scores, torch.zeros(2, 9, device="cuda"), top_n=10)
    refuses("vocab", ops.token_scores, torch.zeros(2, 0, device="cuda"))
    refuses("path", ops.cache_keep, k, v, ln, torch.zeros(1, 2, dtype=torch.int32, device="cuda"))
    # host memory at a C entry, where the kernel would fault
    import ctypes as C

    host = torch.zeros(2, 9)
    a = H.itts_token_scores_args(host.data_ptr(), None, None, None, None, None, 2, 9, 0, 0, H.ITTS_F32, 9, 0)
    refuses("logits: not device memory", lambda: H._check(H.lib.itts_token_scores(C.byref(a), None, 0, None)))
    assert ops.token_scores(torch.zeros(2, 9, device="cuda")).entropy.shape == (2,)  # and the next call works


def test_tensors_that_are_not_what_their_memory_holds(ops):
    """Lazily negated tensors and ones with a forward-mode tangent: refused, by name; resolved and primal ones served."""
    from torch.autograd import forward_ad
    say("[gpu] lazy negations and forward-mode tangents")
    g = gen(31)
    q, k, v = randn(g, 1, 2, 2, 64), randn(g, 1, 2, 12, 64), randn(g, 1, 2, 12, 64)
    ln, par, path = ints([5]), ints([[-1, 0]]), ints([[1]])
    x = randn(g, 3, 20)
    want, best = ops.tree_attention(q, k, v, ln, par), ops.token_scores(x, None, 2)

    def negated(t):
        return torch.complex(torch.zeros_like(t), -t).conj().imag  # reads as t, holds -t

    def calls(change):
        return [("q", lambda: ops.tree_attention(change(q), k, v, ln, par)), ("k", lambda: ops.tree_attention(q, change(k), v, ln, par)),
                ("v", lambda: ops.tree_attention(q, k, change(v), ln, par)),
                ("out", lambda: ops.tree_attention(q, k, v, ln, par, out=change(torch.zeros_like(q)))),
                ("logits", lambda: ops.token_scores(change(x), None, 2)), ("k", lambda: ops.cache_keep(change(k), v.clone(), ln, path)),
                ("v", lambda: ops.cache_keep(k.clone(), change(v), ln, path))]

    n = negated(torch.ones(2, device="cuda"))
    assert n.is_neg() and n.tolist() == [1.0, 1.0]
    for name, call in calls(negated):
        with pytest.raises(H.ValidationError, match=f"{name}: .*resolve_neg"):
            call()
    assert torch.equal(ops.tree_attention(negated(q.transpose(1, 2)).transpose(1, 2).resolve_neg().contiguous(), k, v, ln, par), want)
    with forward_ad.dual_level():
        for name, call in calls(lambda t: forward_ad.make_dual(t, torch.ones_like(t))):
            with pytest.raises(H.ValidationError, match=f"{name}: .*tangent"):
                call()
        assert torch.equal(ops.tree_attention(q, k, v, ln, par), want)
        assert torch.equal(ops.token_scores(x, None, 2).top_tokens, best.top_tokens)


def test_arguments_by_name(ops):
    """Every argument by its name, in any order."""
    say("[gpu] arguments by name")
    g = gen(77)
    q, k, v = randn(g, 2, 3, 4, 64), randn(g, 2, 2, 20, 64), randn(g, 2, 2, 20, 64)
    lengths, parents = ints([4, 9]), ints([[-1, 0, 1]] * 2)
    assert torch.equal(ops.tree_attention(parents=parents, lengths=lengths, v=v, k=k, q=q), ops.tree_attention(q, k, v, lengths, parents))
    x = randn(g, 5, 70)
    one, other = ops.token_scores(top_n=3, logits=x), ops.token_scores(x, None, 3)
    assert torch.equal(one.entropy, other.entropy) and torch.equal(one.top_tokens, other.top_tokens)
    path = ints([[1, 2], [0, -1]])
    k2, v2 = k.unsqueeze(0).clone(), v.unsqueeze(0).clone()
    assert ops.cache_keep(path=path, lengths=lengths, v=v2, k=k2).tolist() == [6, 10]


def test_values_that_do_not_fit_are_refused(ops):
    """What has no place in the library's 32-bit fields is refused, not cut."""
    from itts_hip import ValidationError
    say("[gpu] values past the library's types")
    q, ln, par = torch.zeros(1, 1, 2, 64, device="cuda"), ints([1]), ints([[-1]])
    k = torch.zeros(1, 2, 4, 64, device="cuda")
    for scale in (1e300, -1e300):
        with pytest.raises(ValidationError):
            ops.tree_attention(q, k, k, ln, par, scale=scale)
    with pytest.raises(ValidationError):
        ops.tree_attention(q, k, k, ln, par, max_length=-(1 << 40))
    with pytest.raises(ValidationError, match="rows"):
        ops.token_scores(torch.zeros(1, 2, device="cuda").expand((1 << 23) + 1, 2))
    with pytest.raises(ValidationError):
        ops.cache_keep(k, k, ln, torch.zeros(1, 1, dtype=torch.int32, device="cuda").expand(1, 1 << 33))
