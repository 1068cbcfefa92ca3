"""The operators over paged caches and on logits (itts_hip.ops) against their definitions in float64.

Tolerances.  Attention: a score is a sum of dim products in float32, off by at most about 2 sqrt(dim) roundings of its products'
magnitudes (A = sum |q k| scale), and one or two roundings on its way through the exponential; a probability is then off by
twice that, relative, and a row of n keys sums to within 2 sqrt(n) roundings.  Under 16-bit queries a probability enters the second
product as two planes, off by 2^-16 of it (bf16; 2^-21 fp16), in the product and in the sum of what is divided by; outputs of 16
bits add half a step of the result.  Over 4 bits a score is formed as sum q (1 + c / 16) - sum q, times 16 scale, plus base sum q:
sums of magnitudes up to A4 = sum_groups (48 |scale| + |base|) sum |q|; values in the same way, from 16 + c of one key and c - 31 of the next,
with V4 = sum p (48 |scale| + |base|) in place of P = sum p |v| (48 is less than the second kind's 62: on the strict side).
Appended and gathered rows: worked out in 64 bits (append) or with one operation (gather), so one rounding; codes are exact.
Logits: at most six operations in float32 and one rounding to the type."""
import itertools
import math
import sys

import pytest
import torch

import itts_hip as H

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24  # half a step of float32
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF = {F32: EPS, BF16: 2.0 ** -8, F16: 2.0 ** -11}
PLANES = {F32: 0.0, BF16: 2.0 ** -15, F16: 2.0 ** -20}
TYPES = [(F32, BF16), (F32, F32), (BF16, BF16), (F16, F16), (BF16, 4), (F16, 4), (F32, 4)]
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


# ---- sequences in pages ------------------------------------------------------------------
def values(codes, pairs):
    """Rows of 4 bits [..., dim / 2] with pairs [..., dim / 64, 2] in float64."""
    c = torch.stack([codes % 16, codes // 16], -1).flatten(-2).double().unflatten(-1, (-1, 64))
    return (c * pairs[..., :1].double() + pairs[..., 1:].double()).flatten(-2)


class Seqs:
    """Sequences of `lens` rows whose last `news` are the tokens, in pages of a shuffled cache.  Every row that no token sees
    holds NaN, and table entries without a visible row name no page."""

    def __init__(self, ops, types, lens, news, h, hk, d, page=16, window=0, sinks=0, seed=0, spare=2, layout=None):
        g = gen(seed)
        self.q_type, kv = types
        self.lens, self.news, self.h, self.hk, self.d, self.page, self.window, self.sinks = lens, news, h, hk, d, page, window, sinks
        wide = max([1] + [-(-n // page) for n in lens])
        seen = [sorted({t for pos in range(n - m, n) for t in self.sees(pos)}) if m else [] for n, m in zip(lens, news)]
        used = [sorted({t // page for t in rows}) for rows in seen]
        count = sum(map(len, used)) + spare
        order = iter(torch.randperm(count, generator=torch.Generator().manual_seed(seed)).tolist())
        self.map = [{p: next(order) for p in u} for u in used]
        junk = itertools.cycle([-1, count, 2 ** 31 - 1, -2 ** 31])
        self.table = ints([[m[p] if p in m else next(junk) for p in range(wide)] for m in self.map])
        self.rows = []  # (keys, values, |...| of 4 bits) in float64 [hk][len][d]
        bits4 = kv == 4
        if layout is not None:
            self.cache = layout(count, hk, page, d)
        else:
            self.cache = ops.paged_cache(count, hk, page, d, BF16 if bits4 else kv, bits=4 if bits4 else 32 if kv == F32 else 16)
        for t in self.cache:
            if t is not None:
                t.fill_(NAN if t.dtype.is_floating_point else 255)
        for b, rows in enumerate(seen):
            n, at = lens[b], torch.tensor(rows, dtype=torch.long, device="cuda")
            pg = torch.tensor([self.map[b][t // page] for t in rows], dtype=torch.long, device="cuda")
            one = []
            for which in range(2):
                full = torch.full((hk, max(n, 0), d), NAN, dtype=torch.float64, device="cuda")
                if bits4:
                    codes = torch.randint(0, 256, (len(rows), hk, d // 2), generator=g, device="cuda", dtype=torch.uint8)
                    pairs = torch.stack([0.1 + 0.2 * torch.rand((len(rows), hk, d // 64), generator=g, device="cuda"),
                                         randn(g, len(rows), hk, d // 64) - 1.5], -1).half()
                    self.cache[which][pg, :, at % page], self.cache[2 + which][pg, :, at % page] = codes, pairs
                    full[:, at] = values(codes, pairs).transpose(0, 1)
                    mag = torch.zeros((hk, max(n, 0), d // 64), dtype=torch.float64, device="cuda")
                    mag[:, at] = (48 * pairs[..., 0].double().abs() + pairs[..., 1].double().abs()).transpose(0, 1)
                    one += [full, mag.repeat_interleave(64, -1)]
                else:
                    x = randn(g, len(rows), hk, d, dtype=kv)
                    self.cache[which][pg, :, at % page] = x
                    full[:, at] = x.double().transpose(0, 1)
                    one += [full, None]
            self.rows.append(one)
        self.starts_list = [0] + list(itertools.accumulate(news))
        self.starts, self.lengths = ints(self.starts_list), ints(lens)
        self.q = (1.5 * randn(g, self.starts_list[-1], h, d)).to(self.q_type)

    def sees(self, pos):
        return [t for t in range(pos + 1) if not self.window or t > pos - self.window or t < self.sinks]

    def ref(self, scale=None):
        """(result, tolerance) in float64, token by token over the rows that it sees."""
        d, group = self.d, self.h // self.hk
        scale = d ** -0.5 if scale is None else scale
        ref = torch.zeros(self.q.shape, dtype=torch.float64, device="cuda")
        tol = torch.zeros_like(ref)
        for b, (n, m) in enumerate(zip(self.lens, self.news)):
            k, km, v, vm = (None if x is None else x.repeat_interleave(group, 0) for x in self.rows[b])
            for i in range(m):
                pos, token = n - m + i, self.starts_list[b] + i
                if pos < 0:
                    continue
                at = torch.tensor(self.sees(pos), device="cuda")
                qq, kk, vv = self.q[token].double().unsqueeze(1), k[:, at], v[:, at]
                p = torch.softmax((qq * kk).sum(-1) * scale, -1).unsqueeze(-1)
                amag = (qq * kk).abs() if km is None else qq.abs() * km[:, at]
                mag = amag.sum(-1).amax(-1, keepdim=True) * abs(scale)
                pv = (p * (vv.abs() if vm is None else vm[:, at])).sum(1)
                ref[token] = (p * vv).sum(1)
                tol[token] = pv * EPS * (2 * 2 * (math.sqrt(d) + 2) * mag + 2 * math.sqrt(len(at)) + 8)
                if self.q_type != F32:
                    planes = PLANES[BF16 if vm is not None else self.q_type]
                    tol[token] += HALF[self.q_type] * ref[token].abs() + planes * pv
        return ref, tol + 1e-30

    def run(self, ops, **over):
        f = dict(window=self.window, sinks=self.sinks)
        f.update(over)
        return ops.paged_attention(self.q, self.cache, self.starts, self.lengths, self.table, **f)


# blocks of a token's rows, of several tokens' rows, of many rows over shared tiles; and keys shared by blocks
ENDS = [([60, 33, 70, 16, 100, 45, 8], [1] * 7, 4, 2, 64), ([50] * 5 + [200], [4, 4, 4, 4, 20, 3], 4, 2, 64),
        ([220, 180, 40, 200, 300, 90], [60, 50, 10, 40, 50, 9], 8, 2, 64), ([3000] * 6, [2, 1, 3, 1, 2, 1], 4, 2, 128),
        ([2600] * 6, [40, 30, 50, 20, 40, 39], 8, 2, 64)]


def check(got, ref, tol, what=""):
    bad_nan = torch.isnan(ref) != torch.isnan(got.double())
    assert not bad_nan.any(), f"{what}: NaN in other places ({int(bad_nan.sum())})"
    off = (got.double() - ref).abs().nan_to_num(0.0)
    assert (off <= tol).all(), f"{what}: off by {(off / tol).max().item():.2f} of the tolerance"


# ---- attention ---------------------------------------------------------------------------
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("lens,news,h,hk,d,page", [
    ([1, 15, 16, 17, 31, 32, 33, 700], [1] * 8, 4, 4, 64, 16),
    ([5, 1, 1000, 64], [1] * 4, 8, 2, 128, 48),
    ([300], [1], 28, 4, 128, 32),
    ([40, 2, 90], [3, 2, 0], 5, 5, 64, 16),
    ([7, 0, 65, 200], [7, 0, 20, 33], 12, 4, 64, 64),
    ([130, 131], [130, 17], 2, 1, 128, 16),
    ([9, 9, 9], [0, 9, 0], 6, 1, 128, 16),
    ([250, 77, 4], [99, 77, 1], 20, 20, 64, 80),
    ([400, 35], [140, 35], 8, 1, 64, 16),
])
def test_attention_matches_float64(ops, types, lens, news, h, hk, d, page):
    say(f"[gpu] paged attention {types} lens={lens} news={news} h={h}/{hk} d={d} page={page}")
    s = Seqs(ops, types, lens, news, h, hk, d, page)
    check(s.run(ops), *s.ref())


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("lens,news,window,sinks,page", [
    ([1, 30, 200, 333], [1, 1, 1, 1], 32, 0, 16),
    ([500, 70, 20], [1, 3, 20], 50, 4, 16),
    ([300, 260], [40, 9], 1, 0, 32),
    ([300, 260], [40, 9], 1, 1, 16),
    ([400, 64], [150, 64], 33, 40, 16),
    ([600], [5], 64, 100, 16),
    ([220, 100], [220, 100], 96, 7, 48),
    ([100], [9], 2 ** 31 - 1, 2 ** 31 - 1, 16),
])
def test_attention_windows_and_sinks(ops, types, lens, news, window, sinks, page):
    say(f"[gpu] paged attention window {types} lens={lens} news={news} window={window} sinks={sinks} page={page}")
    s = Seqs(ops, types, lens, news, 6, 2, 64 if window % 2 else 128, page, window, sinks, seed=3)
    check(s.run(ops), *s.ref())


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("lens,news,h,hk,d,window,sinks", [
    ([20011, 5, 0], [1, 1, 0], 2, 1, 64, 0, 0), ([6007], [3], 4, 2, 128, 0, 0), ([9001, 40, 300], [40, 1, 2], 2, 1, 64, 0, 0),
    ([15000, 9000], [2, 1], 2, 2, 64, 5000, 70)])
def test_attention_split_over_keys(ops, types, lens, news, h, hk, d, window, sinks):
    """Long sequences shared by blocks: the same bits each time, with another bound on the rows the same within rounding."""
    say(f"[gpu] paged attention split {types} lens={lens} news={news} h={h}/{hk} d={d} window={window}")
    s = Seqs(ops, types, lens, news, h, hk, d, 64, window, sinks)
    ref, tol = s.ref()
    got = s.run(ops)
    check(got, ref, tol)
    assert torch.equal(got, s.run(ops))
    check(s.run(ops, max_length=max(lens)), ref, tol)


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("d,window,sinks", [(64, 0, 0), (128, 0, 0), (64, 1500, 70), (128, 1500, 0)])
def test_attention_of_many_rows_split_over_keys(ops, types, d, window, sinks):
    """Pieces of prompts whose keys blocks share, beside one that sees few rows, one without tokens and a bad length."""
    say(f"[gpu] paged attention split of many rows {types} d={d} window={window}")
    s = Seqs(ops, types, [2600, 150, 40, 2000, 300], [140, 150, 0, 130, 20], 8, 2, d, 16, window, sinks, seed=21)
    ref, tol = s.ref()
    check(s.run(ops), ref, tol)
    lens = s.lengths.clone()
    lens[3] = -1
    got = ops.paged_attention(s.q, s.cache, s.starts, lens, s.table, window=window, sinks=sinks)
    assert torch.isnan(got[290:420]).all()
    check(got[:290], ref[:290], tol[:290])
    check(got[420:], ref[420:], tol[420:])


@pytest.mark.parametrize("types", [(F32, BF16), (BF16, BF16), (F16, 4)])
@pytest.mark.parametrize("batch", [65, 300])
def test_attention_many_sequences(ops, types, batch):
    """More sequences than a wave has lanes, many without tokens."""
    say(f"[gpu] paged attention many {types} batch={batch}")
    news = [(i * 7) % 4 if i % 3 else 0 for i in range(batch)]
    lens = [n + (i * 13) % 90 for i, n in enumerate(news)]
    s = Seqs(ops, types, lens, news, 4, 2, 64, 16)
    check(s.run(ops), *s.ref())
    assert torch.equal(s.run(ops, max_length=16 * s.table.shape[1]), s.run(ops))


@pytest.mark.parametrize("types", [(F32, BF16), (BF16, BF16), (F16, F16), (F32, F32)])
@pytest.mark.parametrize("news", [1, 37, 300])
@pytest.mark.parametrize("h,hk", [(2, 2), (20, 1)])
def test_attention_of_thousands_of_sequences(ops, types, news, h, hk):
    """Every third one without tokens; each token sees its own row alone, so that results are the values."""
    say(f"[gpu] paged attention thousands {types} {news} {h}/{hk}")
    d, page, batch = 64, 16, 70_000 // (news + 6)
    count = torch.tensor([0 if i % 3 == 1 else 1 + i * 7 % news for i in range(batch)], dtype=torch.int32)
    wide = -(-news // page)
    cache = ops.paged_cache(batch * wide, hk, page, d, types[1], bits=32 if types[1] == F32 else 16)
    cache.k.zero_(), cache.v.copy_(randn(gen(8), *cache.v.shape))
    table = torch.randperm(batch * wide, generator=torch.Generator().manual_seed(9)).int().view(batch, wide).cuda()
    starts = torch.cat([torch.zeros(1, dtype=torch.int32), count.cumsum(0).int()])
    own = torch.repeat_interleave(torch.arange(batch), count)
    row = torch.arange(len(own)) - starts[own]
    q = randn(gen(9), len(own), h, d, dtype=types[0])
    got = ops.paged_attention(q, cache, starts.cuda(), count.cuda(), table, window=1)
    want = cache.v[table[own.cuda(), row.cuda() // page].long(), :, row.cuda() % page].repeat_interleave(h // hk, 1).to(types[0])
    # (a probability over itself: two roundings of 2^-24, under fp32 queries seen)
    tol = 4 * EPS * want.double().abs() if types[0] == F32 else torch.zeros_like(want, dtype=torch.float64)
    assert ((got.double() - want.double()).abs() <= tol).all()


@pytest.mark.parametrize("types", [(F32, BF16), (F32, F32), (BF16, BF16), (F16, F16)])
@pytest.mark.parametrize("value", [NAN, INF, -INF])
@pytest.mark.parametrize("window", [0, 12])
def test_attention_odd_values_stay_where_they_are_seen(ops, types, value, window):
    """A value that is an infinity or NaN reaches the tokens that see its row alone, one after the other and past a window."""
    say(f"[gpu] paged attention odd values {types} {value} window={window}")
    s = Seqs(ops, types, [60, 90], [40, 3], 4, 2, 64, 16, window, 3)
    for row in (30, 59):
        s.cache.v[s.map[0][row // 16], 1, row % 16, 7] = value
        s.rows[0][2][1, row, 7] = value
    s.cache.k[s.map[0][35 // 16], 0, 35 % 16, 3] = value  # a score of either infinity or NaN
    s.rows[0][0][0, 35, 3] = value
    ref, tol = s.ref()
    got = s.run(ops)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(torch.isinf(got), torch.isinf(ref))
    fin = torch.isfinite(ref)
    assert torch.equal(got[~fin & ~torch.isnan(ref)].double(), ref[~fin & ~torch.isnan(ref)])
    assert ((got.double() - ref).abs()[fin] <= tol[fin]).all()
    assert fin[:10].all() and not fin[10, 2:, 7].any() and fin[40:].all()
    assert fin[25, 2:].all() == (window > 0)


@pytest.mark.parametrize("types", [(F32, BF16), (F32, F32), (BF16, BF16), (F16, F16)])
@pytest.mark.parametrize("value", [NAN, INF, -INF])
@pytest.mark.parametrize("d,window", [(64, 0), (128, 0), (64, 70), (128, 70)])
def test_attention_odd_values_in_long_prompts(ops, types, value, d, window):
    """The same where blocks of many query rows share tiles, in every quarter of a tile, seen by all rows of a block or by some."""
    say(f"[gpu] paged attention odd values of prompts {types} {value} d={d} window={window}")
    s = Seqs(ops, types, [210, 150], [170, 150], 4, 2, d, 16, window, 5, seed=7)
    rows = (2, 41, 57, 70, 84, 99, 111, 130, 200)  # (values of a head each, one element each)
    for i, row in enumerate(rows):
        s.cache.v[s.map[0][row // 16], i % 2, row % 16, 3 * i] = value
        s.rows[0][2][i % 2, row, 3 * i] = value
    s.cache.k[s.map[1][90 // 16], 1, 90 % 16, 3] = value
    s.rows[1][0][1, 90, 3] = value
    ref, tol = s.ref()
    got = s.run(ops)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(torch.isinf(got), torch.isinf(ref))
    fin = torch.isfinite(ref)
    assert torch.equal(got[~fin & ~torch.isnan(ref)].double(), ref[~fin & ~torch.isnan(ref)])
    assert ((got.double() - ref).abs()[fin] <= tol[fin]).all()
    assert not fin[100, :2, 0].all() and fin[:170, :, 60:].all()


@pytest.mark.parametrize("value", [INF, -INF])
@pytest.mark.parametrize("lens,news,h,hk,d", [([290], [1], 2, 2, 64), ([9000], [1], 4, 2, 128), ([700, 300], [20, 9], 8, 2, 64), ([700, 400], [150, 70], 8, 2, 64),
                                              ([400], [200], 4, 2, 128), ([5000, 600], [140, 130], 8, 4, 128)])
def test_attention_infinities_of_small_weights(ops, value, lens, news, h, hk, d):
    """Float16: keys whose weight is 2^-40 and 2^-100 of the others' sum hold an infinity in one element, which is then the result's; the
    finite ones stay as they are."""
    say(f"[gpu] paged attention infinities of small weights {value} {lens} {news} h={h}/{hk} d={d}")
    s, scale = Seqs(ops, (F16, F16), lens, news, h, hk, d, 16, seed=23), 1.0 / d
    s.q.fill_(1.0)                                                # a score is a key's elements
    for b, n in enumerate(lens):
        row, page = torch.arange(n, device="cuda"), torch.tensor([s.map[b][t // 16] for t in range(n)], device="cuda")
        key = torch.full((n,), -28.0, device="cuda")              # 2^-40
        key[::8], key[3::64] = 0.0, -69.0                         # (some in every tile: the maximum is theirs for every wave); 2^-99.5
        s.cache.k[page, :, row % 16] = key.half().view(n, 1, 1)
        s.rows[b][0].copy_(key.view(1, n, 1).expand_as(s.rows[b][0]))
        for head, t, e in ((0, 67, 5), (0, 131, 40), (1, 100, 17)):
            s.cache.v[s.map[b][t // 16], head, t % 16, e] = value
            s.rows[b][2][head, t, e] = value
    ref, tol = s.ref(scale)
    got, inf = s.run(ops, scale=scale), torch.isinf(ref)
    group = h // hk
    assert inf[:, :group, 5].all() and inf[:, group:2 * group, 17].all() and inf.sum() == len(ref) * 3 * group
    assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(got.double()[inf], ref[inf])
    assert ((got.double() - ref).abs()[~inf] <= tol[~inf]).all()


@pytest.mark.parametrize("types", TYPES)
def test_attention_odd_calls(ops, types):
    """Lengths out of range, more tokens than rows, pages that do not exist, tokens of no sequence."""
    say(f"[gpu] paged attention odd calls {types}")
    s = Seqs(ops, types, [50, 50, 50, 50, 50, 200], [4, 4, 4, 4, 20, 3], 4, 2, 64, 16)
    s.table[4, 2] = 10 ** 6    # rows 32 .. 47 of sequence 4, seen from its third token on
    lens = s.lengths.clone()
    lens[0], lens[1], lens[2] = -1, 16 * s.table.shape[1] + 1, 2
    ref, tol = s.ref()
    s2 = Seqs(ops, types, [2], [2], 4, 2, 64, 16)
    for got in (ops.paged_attention(s.q, s.cache, s.starts, lens, s.table),
                ops.paged_attention(s.q, s.cache, s.starts, lens, s.table, max_length=200)):
        assert torch.isnan(got[:8]).all()
        assert (got[8:10] == 0).all() and torch.isfinite(got[10:12]).all()  # rows 0 and 1 of sequence 2 are its tokens 2 and 3
        check(got[12:18], ref[12:18], tol[12:18])
        assert torch.isnan(got[18:36]).all()
        check(got[36:], ref[36:], tol[36:])
    # starts that leave tokens out: in front, behind; that fall or pass the end: that sequence alone has none
    out = torch.full_like(s.q, 7.0)
    starts = s.starts.clone()
    starts[0], starts[-1] = 2, 37
    got = ops.paged_attention(s.q, s.cache, starts, s.lengths, s.table, out=out)
    assert got.data_ptr() == out.data_ptr() and (got[:2] == 0).all() and (got[37:] == 0).all() and torch.isfinite(got[2:16]).all()
    starts = s.starts.clone()
    starts[3] = 10 ** 6
    got = ops.paged_attention(s.q, s.cache, starts, s.lengths, s.table)
    check(got[:8], ref[:8], tol[:8])
    check(got[36:], ref[36:], tol[36:])
    assert ops.paged_attention(s.q[:0], s.cache, s.starts * 0, s.lengths, s.table).shape == (0, 4, 64)
    # a table without pages: only empty sequences fit
    got = ops.paged_attention(s.q, s.cache, s.starts, s.lengths * 0, s.table[:, :0])
    assert (got == 0).all()
    del s2


@pytest.mark.parametrize("types", TYPES)
def test_attention_strides(ops, types):
    """Queries in one product's result, heads between tokens in the output, pages with all heads of a row together, keys beside
    values, a table inside a larger one."""
    say(f"[gpu] paged attention strides {types}")

    def layout(n, hk, size, d):
        if types[1] == 4:
            x = torch.empty((n, size, 2, hk, d // 2), dtype=torch.uint8, device="cuda")
            p = torch.empty((n, size, 2, hk, d // 64, 2), dtype=F16, device="cuda")
            y, z = x.permute(2, 0, 3, 1, 4), p.permute(2, 0, 3, 1, 4, 5)
            return ops.PagedCache(y[0], y[1], z[0], z[1])
        x = torch.empty((n, size, 2, hk, d), dtype=types[1], device="cuda").permute(2, 0, 3, 1, 4)
        return ops.PagedCache(x[0], x[1])

    for d, news in ((64, [5, 1, 18]), (128, [5, 1, 18]), (64, [70, 33, 60]), (128, [70, 33, 60])):
        s = Seqs(ops, types, [100, 33, 260], news, 6, 2, d, 16, seed=5, layout=layout)
        wide = torch.zeros((s.q.shape[0], 10, d), dtype=s.q_type, device="cuda")
        wide[:, 1:7] = s.q
        s.q = wide[:, 1:7]
        big = torch.full((3, 40), -1, dtype=torch.int32, device="cuda")
        big[:, 3:3 + s.table.shape[1]] = s.table
        s.table = big[:, 3:3 + s.table.shape[1]]
        out = torch.empty((6, s.q.shape[0], d), dtype=s.q_type, device="cuda").transpose(0, 1)
        ref, tol = s.ref()
        check(s.run(ops, out=out), ref, tol)
        check(s.run(ops, scale=-0.3), *s.ref(-0.3))


@pytest.mark.parametrize("types", [(BF16, BF16), (F16, 4)])
def test_attention_past_32_bits(ops, types):
    """Pages more than 2^32 bytes into the cache."""
    say(f"[gpu] paged attention far pages {types}")
    s = Seqs(ops, types, [100, 40], [3, 1], 8, 4, 64, 32)
    count = 2 ** 32 // (4 * 32 * (32 if types[1] == 4 else 128)) + 40
    far = []
    for t in s.cache:
        if t is None:
            far.append(None)
            continue
        big = torch.empty((count, *t.shape[1:]), dtype=t.dtype, device="cuda")
        big[count - t.shape[0]:] = t
        far.append(big)
    table = torch.where((s.table >= 0) & (s.table < s.cache.k.shape[0]), s.table + count - s.cache.k.shape[0], -1)
    got = ops.paged_attention(s.q, ops.PagedCache(*far), s.starts, s.lengths, table)
    assert torch.equal(got, s.run(ops))


@pytest.mark.parametrize("types", [(F32, BF16), (BF16, BF16), (F32, F32), (F16, 4)])
@pytest.mark.parametrize("lens,news", [([3000, 200, 1], [1, 1, 1]), ([700, 90, 300], [200, 90, 3])])
def test_attention_graphs_and_streams(ops, types, lens, news):
    """Captured and replayed with other lengths, on its own stream, eager calls between the replays."""
    say(f"[gpu] paged attention graph {types} {lens} {news}")
    s = Seqs(ops, types, lens, news, 4, 2, 64, 16)
    first = s.run(ops)
    lens2 = ints([lens[0] - 900 if news[0] == 1 else lens[0], lens[1], lens[2]])
    other = ops.paged_attention(s.q, s.cache, s.starts, lens2, s.table)
    out, held = torch.zeros_like(first), s.lengths.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            ops.paged_attention(s.q, s.cache, s.starts, held, s.table, out=out)
        for use, want in ((s.lengths, first), (lens2, other), (s.lengths, first)):
            held.copy_(use)
            graph.replay()
            assert torch.equal(ops.paged_attention(s.q, s.cache, s.starts, use, s.table), want)
            stream.synchronize()
            assert torch.equal(out, want)


@pytest.mark.parametrize("types", [(BF16, BF16), (F16, F16), (F32, BF16), (F32, F32), (BF16, 4), (F16, 4), (F32, 4)])
def test_attention_of_long_prompts(ops, types):
    """Pieces of prompts of many tiles beside single tokens, against a whole product in float64."""
    say(f"[gpu] paged attention prompts {types}")
    for d, h, hk, window, sinks in ((128, 8, 2, 0, 0), (64, 4, 4, 0, 0), (64, 6, 2, 300, 40)):
        lens, news = [1500, 640, 900, 1, 77], [700, 640, 1, 1, 0]
        g = gen(9)
        page, q_type, kv = 64, *types
        wide = 24
        cache = ops.paged_cache(5 * wide, hk, page, d, BF16 if kv == 4 else kv, bits=4 if kv == 4 else 32 if kv == F32 else 16)
        table = torch.randperm(5 * wide, generator=torch.Generator().manual_seed(1)).int().view(5, wide).cuda()
        rows = []
        for which in range(2):
            if kv == 4:
                cache[which].random_(0, 256, generator=g)
                cache[2 + which][..., 0] = 0.1 + 0.2 * torch.rand(cache[2].shape[:-1], generator=g, device="cuda")
                cache[2 + which][..., 1] = randn(g, *cache[2].shape[:-1]) - 1.5
                rows.append(values(cache[which], cache[2 + which]))
                mags = 48 * cache[2 + which][..., 0].double().abs() + cache[2 + which][..., 1].double().abs()
                rows.append(mags.repeat_interleave(64, -1))
            else:
                cache[which].copy_(randn(g, *cache[which].shape))
                rows += [cache[which].double(), cache[which].double().abs()]
        starts = [0] + list(itertools.accumulate(news))
        q = (1.5 * randn(g, starts[-1], h, d)).to(q_type)
        got = ops.paged_attention(q, cache, ints(starts), ints(lens), table, window=window, sinks=sinks)
        assert torch.equal(got, ops.paged_attention(q, cache, ints(starts), ints(lens), table, window=window, sinks=sinks))
        for b, (n, m) in enumerate(zip(lens, news)):
            at = torch.arange(n, device="cuda")
            k, km, v, vm = (x[table[b].long()].transpose(0, 1).flatten(1, 2)[:, :n] for x in rows)
            pos = torch.arange(n - m, n, device="cuda").unsqueeze(1)
            hidden = at > pos
            if window:
                hidden |= (at <= pos - window) & (at >= sinks)
            for head in range(h):
                x = q[starts[b]:starts[b + 1], head].double()
                sc = (x @ k[head // (h // hk)].T * d ** -0.5).masked_fill(hidden, -INF)
                mag = (x.abs() @ km[head // (h // hk)].T * d ** -0.5).masked_fill(hidden, 0.0).amax(-1, keepdim=True)
                p = torch.softmax(sc, -1)
                ref, pv = p @ v[head // (h // hk)], p @ vm[head // (h // hk)]
                tol = pv * EPS * (4 * (math.sqrt(d) + 2) * mag + 2 * math.sqrt(n) + 8)
                if q_type != F32:
                    tol = tol + HALF[q_type] * ref.abs() + PLANES[BF16 if kv == 4 else q_type] * pv
                check(got[starts[b]:starts[b + 1], head], ref, tol + 1e-30, f"d={d} sequence {b} head {head}")


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_attention_of_many_rows_at_the_ends(ops, types, d):
    """More tokens than rows, empty and bad sequences, missing pages and tokens of no sequence among blocks of many rows; more than
    64 sequences."""
    say(f"[gpu] paged attention many rows at the ends {types} d={d}")
    s = Seqs(ops, types, [150, 0, 3, 170, 90, 200], [150, 0, 170, 100, 90, 130], 8, 2, d, 16, seed=11)
    s.table[3, 6] = 10 ** 6    # rows 96 .. 111 of sequence 3, seen from its 27th token on
    lens = s.lengths.clone()
    lens[4] = -7
    ref, tol = s.ref()
    at = s.starts_list
    got = ops.paged_attention(s.q, s.cache, s.starts, lens, s.table)
    for b in (0, 2, 5):
        check(got[at[b]:at[b + 1]], ref[at[b]:at[b + 1]], tol[at[b]:at[b + 1]], f"sequence {b}")
    assert (got[at[2]:at[2] + 167] == 0).all()
    check(got[at[3]:at[3] + 26], ref[at[3]:at[3] + 26], tol[at[3]:at[3] + 26])
    assert torch.isnan(got[at[3] + 26:at[4]]).all() and torch.isnan(got[at[4]:at[5]]).all()
    starts = s.starts.clone()
    starts[0], starts[6] = 4, at[6] - 9
    out = torch.full_like(s.q, 5.0)
    ops.paged_attention(s.q, s.cache, starts, lens, s.table, out=out)
    assert (out[:4] == 0).all() and (out[at[6] - 9:] == 0).all()
    lens, news = [60 + 7 * (i % 9) for i in range(70)], [30 + i % 20 for i in range(70)]
    s = Seqs(ops, types, lens, news, 8, 2, d, 16, seed=12)
    check(s.run(ops), *s.ref())


@pytest.mark.parametrize("types", [(BF16, BF16), (F32, F32), (F16, 4)])
@pytest.mark.parametrize("tokens", [3, 90])
def test_attention_of_starts_that_fall(ops, types, tokens):
    """Starts that name the same tokens again and again give more rows than there are tokens: nothing leaves its memory, and a call
    with good ones after it is what it was (long sequences, so that blocks share them)."""
    say(f"[gpu] paged attention falling starts {types} {tokens}")
    s = Seqs(ops, types, [3000] * 40, [tokens] + [0] * 39, 4, 2, 64, 16, seed=13)
    first = s.run(ops)
    starts = ints([0, tokens] * 20 + [0])
    for over in ({}, dict(max_length=100)):
        assert ops.paged_attention(s.q, s.cache, starts, s.lengths, s.table, **over).shape == s.q.shape
    assert torch.equal(first, s.run(ops))
    check(first, *s.ref())


@pytest.mark.parametrize("q_type", [F32, F16, BF16])
@pytest.mark.parametrize("batch", [1, 64])
def test_attention_of_even_weights_over_long_contexts(ops, q_type, batch):
    """4 bits, 60,000 rows of the same weight: the mean of their values, much smaller than each, as exact as their number lets it be.

    A sum's running value is a walk of n steps of at most 31 scales, within 3 * 24 sqrt(n) scales; it is rounded n / 16 times at random,
    by 2^-24 of that at most, four waves' sums being less.  Four deviations: 4 * 2^-24 * 72 sqrt(n) * sqrt(n / 16) scales, over n."""
    say(f"[gpu] paged attention even weights {q_type} batch={batch}")
    n, hk, d, page = 60_000, 8, 128, 64
    count, g = -(-n // page), gen(4)
    cache = ops.paged_cache(count, hk, page, d, bits=4)
    cache.k.zero_(), cache.k_params.zero_()
    cache.v.random_(0, 256, generator=g)
    scale = 0.125 + 0.125 * torch.rand(cache.v_params.shape[:-1], generator=g, device="cuda")
    cache.v_params.copy_(torch.stack([scale, -7.5 * scale * (0.9 + 0.2 * torch.rand(scale.shape, generator=g, device="cuda"))], -1))
    ref = torch.stack([values(cache.v[:, h], cache.v_params[:, h]).flatten(0, 1)[:n].mean(0) for h in range(hk)])
    table = torch.arange(count, dtype=torch.int32, device="cuda").expand(batch, -1).contiguous()
    q = torch.zeros((batch, 2 * hk, d), dtype=q_type, device="cuda")
    got = ops.paged_attention(q, cache, ints(range(batch + 1)), ints([n] * batch), table)
    ref = ref.repeat_interleave(2, 0).expand(batch, -1, -1)
    tol = 4 * 2.0 ** -24 * 72 / 4 * 0.25 + (0 if q_type == F32 else HALF[q_type] * ref.abs())
    check(got, ref, tol)


@pytest.mark.parametrize("kv", [BF16, 4])
def test_attention_of_more_rows_than_a_quotient_holds(ops, kv):
    """320,000 tokens of 127 heads, each of which sees its own row alone: results are the values.  (2^32 / 127, rounded up, gives a
    token too many from row 2^32 / 111 on.)"""
    say(f"[gpu] paged attention 320,000 tokens of 127 heads {kv}")
    n, group, d = 320_000, 127, 64
    cache = ops.paged_cache(n // 64, 1, 64, d, BF16, bits=4 if kv == 4 else 16)
    for t in cache[:2]:
        t.zero_() if t.is_floating_point() else t.random_(0, 256)
    if kv == 4:
        cache.k_params.zero_()
        cache.v_params[..., 0], cache.v_params[..., 1] = 0.125, -1.0  # (values in eighths, exact in 16 bits)
        # 4 bits: a value is the difference of scale (16 + code) p / l, at most 4, and (16 scale - base) p / l = 3, where p and l are fp32
        # numbers with a rounding each and the sums and products round four times more: 8 steps of 2^-24 of 7 in all
        tol = 8 * 2.0 ** -24 * 7
        want = values(cache.v, cache.v_params)[:, 0].flatten(0, 1).to(BF16)
    else:
        cache.v.copy_(randn(gen(3), *cache.v.shape))
        want = cache.v[:, 0].flatten(0, 1)
    table = torch.arange(n // 64, dtype=torch.int32, device="cuda").unsqueeze(0)
    q = torch.zeros((n, group, d), dtype=BF16, device="cuda")
    got = ops.paged_attention(q, cache, ints([0, n]), ints([n]), table, window=1)
    del q
    for at in range(0, n, 20_000):
        off = (got[at:at + 20_000].float() - want[at:at + 20_000].unsqueeze(1).float()).abs()
        assert off.max() <= (tol + HALF[BF16] * want.abs().max() if kv == 4 else 0.0)


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("lens,news,h,hk,d", ENDS)
def test_attention_in_place(ops, types, lens, news, h, hk, d):
    """The result where the queries are: every kernel and layout gives what it gives elsewhere, tokens of no sequence among them."""
    say(f"[gpu] paged attention in place {types} {lens} {news}")
    s = Seqs(ops, types, lens, news, h, hk, d, 16, seed=44)
    for starts in (s.starts_list, s.starts_list[:2] + [10 ** 6] + s.starts_list[3:]):
        want, q = ops.paged_attention(s.q, s.cache, ints(starts), s.lengths, s.table), s.q.clone()
        assert ops.paged_attention(q, s.cache, ints(starts), s.lengths, s.table, out=q).data_ptr() == q.data_ptr()
        assert torch.equal(q, want)
    for x, out in ((q[:-1], q[1:]), (q[1:], q[:-1])):
        with pytest.raises(H.ValidationError, match="out: "):
            ops.paged_attention(x, s.cache, s.starts, s.lengths, s.table, out=out)


def test_attention_refuses(ops):
    s = Seqs(ops, (F32, BF16), [20], [1], 4, 2, 64)
    for over, match in ((dict(window=-1), "window"), (dict(max_length=33), "max_length"), (dict(scale=NAN), "scale"),
                        (dict(out=s.q.half()), "out"), (dict(window=2 ** 40), "does not fit")):
        with pytest.raises(H.ValidationError, match=match):
            s.run(ops, **over)
    with pytest.raises(H.ValidationError, match="q_dtype"):
        ops.paged_attention(s.q.half(), s.cache, s.starts, s.lengths, s.table)
    with pytest.raises(H.ValidationError, match="lengths"):
        ops.paged_attention(s.q, s.cache, s.starts, s.lengths.long(), s.table)
    with pytest.raises(H.ValidationError, match="starts"):
        ops.paged_attention(s.q, s.cache, s.starts[:1], s.lengths, s.table)
    with pytest.raises(H.ValidationError, match="cache.k_params"):
        ops.paged_attention(s.q, ops.PagedCache(s.cache.k, s.cache.v, s.q, s.q), s.starts, s.lengths, s.table)
    with pytest.raises(H.ValidationError, match="gradient"):
        ops.paged_attention(s.q.clone().requires_grad_(), s.cache, s.starts, s.lengths, s.table)


# ---- append ------------------------------------------------------------------------------
def rotation_table(rows, n):
    angle = torch.arange(rows, dtype=torch.float64).unsqueeze(1) * 10000.0 ** (-torch.arange(n // 2, dtype=torch.float64) / (n // 2))
    return torch.cat([angle.cos(), angle.sin()], 1).float().cuda()


def turn(x, table, pos, interleaved):
    x, n = x.double().clone(), table.shape[1] // 2
    for i in range(n):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
        c, s = table[pos, i].double().unsqueeze(-1), table[pos, n + i].double().unsqueeze(-1)
        xa, xb = x[..., a].clone(), x[..., b].clone()
        x[..., a], x[..., b] = xa * c - xb * s, xb * c + xa * s
    return x


def quantise(x):
    x = x.unflatten(-1, (-1, 64))
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale, base = ((hi - lo) / 15).float().half(), lo.float().half()
    code = torch.where(scale == 0, 0.0, ((x - base.double()) / scale.double()).round().clamp(0, 15))
    code = code.to(torch.uint8).flatten(-2)
    return code[..., ::2] | code[..., 1::2] << 4, torch.cat([scale, base], -1)


def one_rounding(got, want):
    """Off by half a step of the type at most (and a little: 64 bits go to 16 by way of 32)."""
    t = got.dtype
    step = HALF[t] * want.abs() + (2.0 ** -25 if t == F16 else 1e-40)
    assert ((got.double() - want).abs() <= step * (1 + 2.0 ** -12)).all()


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("news,lens,h,hk,d,page,rot,interleaved", [
    ([1, 1, 1], [0, 15, 100], 4, 4, 64, 16, 64, False), ([1], [33], 20, 20, 64, 64, 0, False), ([5, 0, 40, 1], [10, 3, 0, 31], 8, 2, 128, 16, 128, False),
    ([17, 3], [0, 47], 6, 2, 64, 48, 32, True), ([9], [7], 28, 4, 128, 32, 48, False), ([33, 2], [1, 0], 0, 1, 128, 16, 128, True),
    ([2] * 70, list(range(70)), 3, 1, 64, 16, 16, False)])
def test_append_matches_float64(ops, types, news, lens, h, hk, d, page, rot, interleaved):
    say(f"[gpu] paged append {types} news={news[:5]} lens={lens[:5]} h={h}/{hk} d={d} page={page} rot={rot} {interleaved}")
    q_type, kv = types
    g, tokens = gen(1), sum(news)
    wide = max(-(-(n + m) // page) for n, m in zip(lens, news)) + 1
    cache = ops.paged_cache(len(news) * wide + 1, hk, page, d, BF16 if kv == 4 else kv, bits=4 if kv == 4 else 32 if kv == F32 else 16)
    for t in cache:
        if t is not None:
            t.copy_(torch.randint(0, 200, t.shape, generator=g, device="cuda"))
    before = [None if t is None else t.clone() for t in cache]
    order = torch.randperm(len(news) * wide, generator=torch.Generator().manual_seed(3)).int().view(len(news), wide)
    x = randn(g, tokens, h + 2 * hk, d, dtype=q_type)
    q, k, v = x[:, :h], x[:, h:h + hk], x[:, h + hk:]
    table = rotation_table(max(lens) + max(news) + 3, rot) if rot else None
    starts = [0] + list(itertools.accumulate(news))
    row = torch.tensor([n + i for n, m in zip(lens, news) for i in range(m)], device="cuda")
    for pos in (None, (row * 7 + 2) % (table.shape[0] if rot else 5)):
        got = ops.paged_append(cache, k, v, ints(starts), ints(lens), order.cuda(), q=q if h else None, rotation=table,
                               positions=None if pos is None else pos.int(), interleaved=interleaved)
        assert got.lengths.tolist() == [n + m for n, m in zip(lens, news)]
        at = row if pos is None else pos
        kk, qq = (turn(k, table, at, interleaved), turn(q, table, at, interleaved)) if rot else (k.double(), q.double())
        if h:
            one_rounding(got.q, qq)
        else:
            assert got.q is None
        page_at = torch.tensor([int(order[b, (n + i) // page]) for b, (n, m) in enumerate(zip(lens, news)) for i in range(m)], device="cuda")
        for which, want in ((0, kk), (1, v.double())):
            rest = before[which].clone()
            if kv == 4:
                codes, pairs = quantise(want)
                assert torch.equal(cache[which][page_at, :, row % page], codes)
                assert torch.equal(cache[2 + which][page_at, :, row % page], pairs)
                rest[page_at, :, row % page] = codes
                assert torch.equal(cache[which], rest)
            else:
                one_rounding(cache[which][page_at, :, row % page], want)
                rest[page_at, :, row % page] = cache[which][page_at, :, row % page]
                assert torch.equal(cache[which], rest)  # nothing else was written


def test_append_codes_at_borders(ops):
    """Values halfway between two codes go to the even one; constant rows, rows with one value apart, tiny and large ranges."""
    say("[gpu] paged append borders")
    x = torch.zeros(8, 1, 64, device="cuda")
    x[0, 0] = torch.arange(64, device="cuda") % 31 * 0.5          # codes 0, 0.5, 1 ...
    x[1, 0] = 3.25
    x[2, 0, 5] = 1e-9                                             # a range below float16's smallest step
    x[3, 0] = torch.linspace(-6e4, 6e4, 64, device="cuda")
    x[4, 0] = torch.linspace(-1e5, 1e5, 64, device="cuda")        # beyond float16
    x[5, 0], x[5, 0, 9] = 1.0, NAN
    x[6, 0], x[6, 0, 63] = 1.0, -INF
    x[7, 0] = 1000.0 + torch.arange(64, device="cuda") * 0.01     # a small range on a large base
    cache = ops.paged_cache(1, 1, 16, 64, bits=4)
    for t in cache:
        t.zero_()
    ops.paged_append(cache, x, x, ints([0, 8]), ints([0]), ints([[0]]))
    codes, pairs = quantise(x.double())
    for i in (0, 1, 2, 3, 7):
        assert torch.equal(cache.k[0, 0, i], codes[i, 0]) and torch.equal(cache.v_params[0, 0, i], pairs[i, 0]), i
    k, _ = ops.paged_gather(cache, ints([8]), ints([[0]]), 8)
    assert torch.isnan(k[0, 0, 4:7]).all() and torch.isfinite(k[0, 0, [0, 1, 2, 3, 7]]).all()
    assert torch.equal(k[0, 0, 0].double(), (x[0, 0].double()).round()) and (k[0, 0, 1] == 3.25).all()


@pytest.mark.parametrize("bits", [16, 4])
def test_append_into_rows_of_all_heads(ops, bits):
    """Pages whose rows hold all heads, keys beside values, as one tensor; several sequences, a table inside a larger one."""
    say(f"[gpu] paged append strides {bits}")
    g, d, hk = gen(14), 128, 3
    k, v = (randn(g, 40, hk, d, dtype=BF16) for _ in range(2))
    wide = torch.full((3, 9), -1, dtype=torch.int32, device="cuda")
    wide[:, 2:4] = ints([[4, 0], [2, 5], [1, 3]])
    starts, lens = ints([0, 17, 17, 40]), ints([3, 5, 0])
    plain = ops.paged_cache(6, hk, 16, d, BF16, bits=bits)
    if bits == 4:
        x, p = torch.zeros((6, 16, 2, hk, d // 2), dtype=torch.uint8, device="cuda"), torch.zeros((6, 16, 2, hk, d // 64, 2), dtype=F16, device="cuda")
        y, z = x.permute(2, 0, 3, 1, 4), p.permute(2, 0, 3, 1, 4, 5)
        other = ops.PagedCache(y[0], y[1], z[0], z[1])
    else:
        y = torch.zeros((6, 16, 2, hk, d), dtype=BF16, device="cuda").permute(2, 0, 3, 1, 4)
        other = ops.PagedCache(y[0], y[1])
    for c in (plain, other):
        for t in c:
            if t is not None:
                t.zero_()
        assert ops.paged_append(c, k, v, starts, lens, wide[:, 2:4]).lengths.tolist() == [20, 5, 23]
    for a, b in zip(plain, other):
        assert a is None and b is None or torch.equal(a, b)


@pytest.mark.parametrize("q_type", [F32, BF16, F16])
@pytest.mark.parametrize("value", [NAN, INF, -INF])
@pytest.mark.parametrize("rot,interleaved", [(128, False), (96, False), (80, False), (64, False), (128, True), (0, False)])
def test_append_odd_values_stay_in_their_group(ops, q_type, value, rot, interleaved):
    """4 bits of 128: one of a row's two groups of 64 holds a value that is no finite number, at either end of a run of 8 and in
    every run; the other group's codes and pair are as without it.  Keys turn, so that a pair's other element is odd as well."""
    say(f"[gpu] paged append odd groups {q_type} {value} rot={rot} interleaved={interleaved}")
    g, d, hk, at = gen(31), 128, 2, [*range(0, 128, 8), *range(7, 128, 8), 5, 70]
    n = len(at) + 2
    k, v = (randn(g, n, hk, d, dtype=q_type) for _ in range(2))
    for i, e in enumerate(at):
        k[i, i % 2, e] = v[i, 1 - i % 2, e] = value
    k[n - 2, 0, 3] = k[n - 2, 0, 90] = v[n - 2, 0, 3] = v[n - 2, 0, 90] = value     # both groups; the last row has none
    cache, table = ops.paged_cache(3, hk, 16, d, bits=4), rotation_table(n + 5, rot) if rot else None
    for t in cache:
        t.zero_()
    pos = torch.arange(5, n + 5, device="cuda")
    got = ops.paged_append(cache, k, v, ints([0, n]), ints([0]), ints([[2, 0, 1]]), rotation=table, positions=pos.int(), interleaved=interleaved)
    assert got.lengths.tolist() == [n]
    page, row = ints([2, 0, 1])[torch.arange(n, device="cuda") // 16].long(), torch.arange(n, device="cuda") % 16
    back = ops.paged_gather(cache, ints([n]), ints([[2, 0, 1]]), n)
    for which, want in ((0, turn(k, table, pos, interleaved) if rot else k.double()), (1, v.double())):
        fine = torch.isfinite(want).unflatten(-1, (2, 64)).all(-1)
        assert fine.any(-1).sum() > n and (~fine).sum() > len(at)
        codes, pairs = quantise(want)
        mine, own = cache[which][page, :, row].unflatten(-1, (2, 32)), cache[2 + which][page, :, row]
        assert torch.equal(mine[fine], codes.unflatten(-1, (2, 32))[fine]) and torch.equal(own[fine], pairs[fine])
        read = back[which][0].transpose(0, 1).unflatten(-1, (2, 64))
        assert torch.isfinite(read[fine]).all() and torch.isnan(read[~fine]).all()


def test_append_pairs_round_twice(ops):
    """Scale and base go to float16 by way of float32, for every one of many turned rows."""
    say("[gpu] paged append pairs")
    g = gen(13)
    k = randn(g, 6000, 8, 128, dtype=BF16)
    cache, rot = ops.paged_cache(375, 8, 16, 128, bits=4), rotation_table(6000, 128)
    ops.paged_append(cache, k, k, ints([0, 6000]), ints([0]), torch.arange(375, dtype=torch.int32, device="cuda").view(1, -1), rotation=rot)
    codes, pairs = quantise(turn(k, rot, torch.arange(6000, device="cuda"), False))
    assert torch.equal(cache.k_params.transpose(1, 2).flatten(0, 1), pairs)
    assert torch.equal(cache.k.transpose(1, 2).flatten(0, 1), codes)


@pytest.mark.parametrize("types", [(F32, BF16), (BF16, 4)])
def test_append_odd_calls(ops, types):
    say(f"[gpu] paged append odd calls {types}")
    q_type, kv = types
    g = gen(2)
    cache = ops.paged_cache(6, 2, 16, 64, BF16, bits=kv if kv == 4 else 16)
    for t in cache:
        if t is not None:
            t.zero_()
    x = randn(g, 14, 2, 64, dtype=q_type)
    q = randn(g, 14, 2, 64, dtype=q_type)
    rot = rotation_table(20, 64)
    table = ints([[0, 1], [2, 99], [3, 4], [5, -1], [5, -1]])
    # too long; past the end of its table's pages; its second row in no page; fine; positions past the table
    starts, lens = ints([1, 3, 5, 8, 10, 12]), ints([-1, 31, 15, 0, 8])
    pos = ints([0] * 10 + [19, 20] + [0] * 2)
    got = ops.paged_append(cache, x, x, starts, lens, table, q=q, rotation=rot, positions=pos)
    assert got.lengths.tolist() == [-1, -1, 18, 2, 10]
    assert (got.q[:1] == 0).all() and (got.q[12:] == 0).all() and torch.isnan(got.q[1:5]).all() and torch.isfinite(got.q[5:11]).all()
    assert torch.isnan(got.q[11]).all()
    k, v = ops.paged_gather(cache, ints([32]), ints([[5, 0]]), 32, dtype=BF16)
    assert torch.isfinite(k[0, :, :9]).all() and torch.isnan(k[0, :, 9]).all() and torch.isfinite(v[0]).all() and (k[0, :, 16:] == 0).all()
    assert (k[0, :, 8] != 0).any() and (k[0, :, 2:8] == 0).all()
    got = ops.paged_append(cache, x, x, ints([0, 2]), ints([15]), ints([[1, 77]]))   # the row that has a page is written
    assert got.lengths.tolist() == [-1] and got.q is None
    assert (ops.paged_gather(cache, ints([16]), ints([[1]]), 16, dtype=BF16)[1][0, :, 15] != 0).any()
    # starts that fall: that sequence has none, the tokens nothing claims stay out
    got = ops.paged_append(cache, x, x, ints([0, 5, 2, 99]), ints([0, 0, 0]), ints([[0], [1], [2]]), q=q)
    assert got.lengths.tolist() == [5, -1, -1]
    got = ops.paged_append(cache, x[:0], x[:0], ints([0, 0]), ints([7]), ints([[1]]), q=q[:0])
    assert got.lengths.tolist() == [7] and got.q.shape == (0, 2, 64)


def test_append_in_place_and_captured(ops):
    """Queries turned in place; captured with lengths that move on with every replay."""
    say("[gpu] paged append captured")
    g = gen(4)
    cache, table = ops.paged_cache(8, 2, 16, 64, bits=4), ints([[3, 1, 7], [0, 5, 2]])
    for t in cache:
        t.zero_()
    x, q = randn(g, 2, 2, 64), randn(g, 2, 4, 64)
    rot, starts, lens = rotation_table(48, 64), ints([0, 1, 2]), ints([0, 20])
    q2 = q.clone()
    got = ops.paged_append(cache, x, x, starts, lens, table, q=q2, q_out=q2, rotation=rot)
    assert got.q.data_ptr() == q2.data_ptr()
    one_rounding(q2, turn(q, rot, torch.tensor([0, 20], device="cuda"), False))
    held, qo = lens.clone(), torch.empty_like(q)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            held.copy_(ops.paged_append(cache, x, x, starts, held, table, q=q, q_out=qo, rotation=rot).lengths)
        for step in range(5):
            graph.replay()
            stream.synchronize()
            assert held.tolist() == [step + 1, 21 + step]
            one_rounding(qo, turn(q, rot, torch.tensor([step, 20 + step], device="cuda"), False))
    codes, pairs = quantise(turn(x[1:], rot, torch.tensor([24], device="cuda"), False))
    assert torch.equal(cache.k[5, :, 8], codes[0]) and torch.equal(cache.k_params[5, :, 8], pairs[0])


# ---- starts that do not rise --------------------------------------------------------------
def spans_of(starts, tokens):
    """(first token, tokens) of each sequence, or None: starts that fall or leave the tensors, or come back to in front of where an
    earlier sequence ends."""
    reach, out = 0, []
    for i, j in zip(starts, starts[1:]):
        fits = 0 <= i <= j <= tokens
        out.append((i, j - i) if fits and (i == j or i >= reach) else None)
        reach = max(reach, j) if fits and j > i else reach
    return out


def bad_starts(s):
    """Starts of at least six sequences, each with something wrong about it."""
    yield "past the end", s[:2] + [10 ** 6] + s[3:]
    yield "below 0", s[:2] + [-5] + s[3:]
    yield "falls", s[:3] + [s[1]] + s[4:]
    yield "first too large", [s[4]] + s[1:]
    yield "last too small", s[:-1] + [s[2]]
    yield "around others", s[:1] + [s[5]] + s[2:]
    yield "first and last", [s[3]] + s[1:-1] + [s[1]]
    yield "nothing fits", [0, s[-1] + 50] + [s[-1]] * (len(s) - 2)


@pytest.mark.parametrize("types", [(F32, BF16), (BF16, BF16), (F32, F32), (F16, 4)])
@pytest.mark.parametrize("lens,news,h,hk,d", ENDS)
def test_attention_of_tokens_without_a_sequence(ops, types, lens, news, h, hk, d):
    """Starts that do not rise: tokens of no sequence get zeros, those of the others their results, every time."""
    say(f"[gpu] paged attention bad starts {types} {lens} {news}")
    s = Seqs(ops, types, lens, news, h, hk, d, 16, seed=41)
    good = s.starts_list
    for what, starts in bad_starts(good):
        say("  ", what, starts)
        spans = spans_of(starts, good[-1])
        s.starts_list, s.news = [x[0] if x else 0 for x in spans], [x[1] if x else 0 for x in spans]
        ref, tol = s.ref()
        none = torch.ones(good[-1], dtype=torch.bool, device="cuda")
        for i, n in zip(s.starts_list, s.news):
            none[i:i + n] = False
        assert (ref[none] == 0).all()
        for _ in range(3):
            out = torch.full_like(s.q, 7.0)
            ops.paged_attention(s.q, s.cache, ints(starts), s.lengths, s.table, out=out)
            assert (out[none] == 0).all(), what
            check(out, ref, tol, what)


@pytest.mark.parametrize("types", [(F32, BF16), (BF16, 4)])
def test_append_of_tokens_without_a_sequence(ops, types):
    """The same of appended rows: a sequence's are all there, or none and its new length is -1."""
    say(f"[gpu] paged append bad starts {types}")
    q_type, kv = types
    g, hk, d, lens, news = gen(42), 2, 64, [3, 14, 0, 31, 7, 9, 20], [4, 1, 5, 40, 2, 3, 0]
    good = [0] + list(itertools.accumulate(news))
    n = good[-1]
    k, v, q = randn(g, n, hk, d, dtype=q_type), randn(g, n, hk, d, dtype=q_type), randn(g, n, 4, d, dtype=q_type)
    table = torch.arange(7 * 6, dtype=torch.int32).view(7, 6).cuda()
    for what, starts in [*bad_starts(good), ("falls", [0, 5, 2, n + 9]), ("falls", [0, 7, 3, 7, 20])]:
        b = len(starts) - 1
        say("  ", what, starts)
        cache = ops.paged_cache(42, hk, 16, d, BF16, bits=kv if kv == 4 else 16)
        for t in cache:
            if t is not None:
                t.fill_(0)
        got = ops.paged_append(cache, k, v, ints(starts), ints(lens[:b]), table[:b], q=q)
        spans = spans_of(starts, n)
        assert got.lengths.tolist() == [m + x[1] if x else -1 for m, x in zip(lens, spans)], what
        want_q, rows = torch.zeros_like(q), [torch.zeros_like(t) if t is not None else None for t in cache]
        for i, x in enumerate(spans):
            if not x:
                continue
            own = slice(x[0], x[0] + x[1])
            want_q[own] = q[own]
            at = torch.arange(lens[i], lens[i] + x[1], device="cuda")
            for which, src in ((0, k), (1, v)):
                if kv == 4:
                    rows[which][table[i][at // 16].long(), :, at % 16], rows[2 + which][table[i][at // 16].long(), :, at % 16] = quantise(src[own].double())
                else:
                    rows[which][table[i][at // 16].long(), :, at % 16] = src[own].to(BF16)
        assert torch.equal(got.q, want_q), what
        assert all(torch.equal(x, y) for x, y in zip(cache, rows) if x is not None), what


@pytest.mark.parametrize("types", [(F32, BF16), (F16, 4)])
@pytest.mark.parametrize("batch,news,long", [(70, 1, 0), (70, 3, 2500), (200, 40, 0), (100, 300, 0), (500, 2, 0), (5000, 2, 0), (5000, 9, 0)])
@pytest.mark.parametrize("hk", [1, 8])
def test_bad_starts_of_many_sequences(ops, types, batch, news, long, hk):
    """More sequences than a wave has lanes: what is wrong about some starts may leave neighbours without tokens, but each sequence has all
    its rows and results, or a new length of -1 and zeros."""
    say(f"[gpu] paged bad starts of many sequences {types} {batch} {news} {long} {hk}")
    q_type, kv = types
    gt = torch.Generator().manual_seed(batch + news)
    count = torch.randint(0, news + 1, (batch,), generator=gt)
    good = [0] + count.cumsum(0).tolist()
    n, d, wide = good[-1], 64, -(-news // 16) + -(-long // 16)
    cache = ops.paged_cache(batch * wide, hk, 16, d, BF16, bits=kv if kv == 4 else 16)
    table, lens = torch.arange(batch * wide, dtype=torch.int32).view(batch, wide).cuda(), ints([long] * batch)
    num = torch.arange(n) % 13 + 1.0                                 # a token's value in all its elements: exact in every type
    v = num.to(q_type).cuda().view(n, 1, 1).expand(n, hk, d).contiguous()
    k, q = torch.zeros_like(v), torch.ones_like(v)
    for trial in range(12):
        starts = list(good)
        for _ in range(trial % 4):
            at, what = (int(x) for x in torch.randint(0, 10 ** 6, (2,), generator=gt))
            starts[at % (batch + 1)] = [10 ** 6, -1, 0, n, what % (n + 1)][what % 5]
        say("  ", trial, [(i, x) for i, (x, y) in enumerate(zip(starts, good)) if x != y])
        for t in cache:
            if t is not None:
                t.zero_()
        r = ops.paged_append(cache, k, v, ints(starts), lens, table, q=q)
        owned, want, long_ones = torch.zeros(n, dtype=torch.bool), torch.zeros(batch, wide * 16), torch.zeros(n, dtype=torch.bool)
        for b, (i, j, m) in enumerate(zip(starts, starts[1:], r.lengths.tolist())):
            assert m == -1 or (0 <= i <= j <= n and m == long + j - i)
            if 0 <= i <= j <= n and long + j - i > wide * 16:  # (no room: none is written, queries are NaN)
                long_ones[i:j] = True
            if m > long:
                assert not owned[i:j].any()
                owned[i:j], want[b, long:m] = True, num[i:j]
        assert owned.all() or trial % 4
        rows = ops.paged_gather(cache, ints([wide * 16] * batch), table, wide * 16, dtype=None if kv != 4 else q_type)[1]
        assert (rows == want.cuda().view(batch, 1, -1, 1)).all()
        owned, odd = owned.cuda(), torch.isnan(r.q)
        assert ((r.q == owned.view(n, 1, 1)) | odd & long_ones.cuda().view(n, 1, 1)).all() and not odd[owned].any()
        # each token over its own row alone, so that results are the values; and over all rows
        held = r.lengths.clamp(min=0)
        for window in (1, 0):
            first = None
            for _ in range(2):
                out = torch.full_like(q, 7.0)
                ops.paged_attention(q, cache, ints(starts), held, table, window=window, out=out)
                zero = (out == 0).flatten(1).all(1)
                fits = ((out.float() - v.float()).abs() < 1e-2 if window else (out > 0) & (out < 13.5)).flatten(1).all(1)
                assert (zero | fits).all() and zero[~owned].all() and (fits.all() or trial % 4)
                assert first is None or torch.equal(out, first)
                first = out


# ---- gather ------------------------------------------------------------------------------
@pytest.mark.parametrize("kv", [F32, BF16, F16, 4])
@pytest.mark.parametrize("lens,hk,d,page,rows", [([0, 1, 16, 17, 50], 3, 64, 16, 50), ([100, 33], 1, 128, 48, 120), ([70], 2, 64, 64, 31)])
def test_gather(ops, kv, lens, hk, d, page, rows):
    say(f"[gpu] paged gather {kv} {lens} hk={hk} d={d} page={page} rows={rows}")
    g = gen(6)
    wide = max(-(-n // page) for n in lens)
    cache = ops.paged_cache(len(lens) * wide, hk, page, d, BF16 if kv == 4 else kv, bits=4 if kv == 4 else 32 if kv == F32 else 16)
    for t in cache:
        if t is not None:
            t.copy_(torch.randint(0, 256, t.shape, generator=g, device="cuda") if t.dtype == torch.uint8 else randn(g, *t.shape))
    order = torch.randperm(len(lens) * wide, generator=torch.Generator().manual_seed(3)).int().view(len(lens), wide)
    for dtype in ([F32, BF16, F16] if kv == 4 else [kv]):
        k = torch.full((len(lens), hk, rows + 4, d), 5.0, dtype=dtype, device="cuda")
        got = ops.paged_gather(cache, ints(lens), order.cuda(), rows, k_out=k[:, :, :rows], dtype=dtype)
        assert got[1].shape == (len(lens), hk, rows, d) and got[1].dtype == dtype and (k[:, :, rows:] == 5).all()
        for which in range(2):
            x = values(cache[which], cache[2 + which]) if kv == 4 else cache[which].double()
            for b, n in enumerate(lens):
                m = min(n, rows)
                want = x[order[b].long().cuda()].transpose(0, 1).flatten(1, 2)[:, :m]
                if kv == 4:
                    one_rounding(got[which][b, :, :m], want)
                else:
                    assert torch.equal(got[which][b, :, :m].double(), want)
                assert (got[which][b, :, m:] == 0).all()


def test_gather_odd_calls(ops):
    say("[gpu] paged gather odd calls")
    cache = ops.paged_cache(3, 2, 16, 64, F32, bits=32)
    cache.k.fill_(1.0), cache.v.fill_(2.0)
    k, v = ops.paged_gather(cache, ints([-1, 33, 32, 20]), ints([[0, 1], [0, 1], [1, 3], [-5, 2]]), 24)
    assert torch.isnan(k[:2]).all() and (k[2, :, :16] == 1).all() and torch.isnan(k[2, :, 16:]).all()
    assert torch.isnan(v[3, :, :16]).all() and (v[3, :, 16:20] == 2).all() and (v[3, :, 20:] == 0).all()
    assert ops.paged_gather(cache, ints([0]), ints([[0]]), 0)[0].shape == (1, 2, 0, 64)
    for f, match in ((lambda: ops.paged_gather(cache, ints([0]), ints([[0]]), -1), "rows"),
                     (lambda: ops.paged_gather(cache, ints([0]), ints([[0]]), 4, dtype=F16), "dtype"),
                     (lambda: ops.paged_gather(cache, ints([0]), ints([[0]]), 4, k_out=k, v_out=k), "k_out")):
        with pytest.raises(H.ValidationError, match=match):
            f()


# ---- logits ------------------------------------------------------------------------------
def adjust_ref(x, history=None, rep=None, freq=None, pres=None, tokens=None, bias=None, allowed=None):
    """(result, tolerance) in float64."""
    r, v = x.shape
    y, mag = x.double(), x.double().abs()
    if history is not None:
        count = torch.zeros((r, v), dtype=torch.float64, device=x.device)
        for i, row in enumerate(history.tolist()):
            for t in row:
                if 0 <= t < v:
                    count[i, t] += 1
        rep, freq, pres = (t.double().unsqueeze(1) if isinstance(t, torch.Tensor) else t for t in (rep, freq, pres))
        new = torch.where(y < 0, y * rep, y / rep)
        pen = freq * count + pres * (count > 0)
        mag = torch.where(count > 0, new.abs() + (freq * count).abs() + abs(pres), mag)
        y = torch.where(count > 0, new - pen, y)
    if tokens is not None:
        add = torch.zeros((r, v), dtype=torch.float64, device=x.device)
        for i, (row, b) in enumerate(zip(tokens.tolist(), bias.double().tolist())):
            for t, one in zip(row, b):
                if 0 <= t < v:
                    add[i, t] = one
        y, mag = y + add, mag + add.abs()
    if allowed is not None:
        t = torch.arange(v, device=x.device)
        y = y.masked_fill((allowed.long() & 0xffffffff)[:, t // 32] >> (t % 32) & 1 == 0, -INF)
    step = HALF[x.dtype] if x.dtype != F32 else 0.0
    return y, mag * EPS * 6 + step * (y.abs() + mag * EPS * 6) + (2.0 ** -24 if x.dtype == F16 else 1e-40)


def same(got, ref, tol):
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    inf = torch.isinf(ref)
    assert torch.equal(got[inf].double(), ref[inf])
    ok = ~inf & ~torch.isnan(ref)
    assert ((got.double() - ref).abs()[ok] <= tol[ok]).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,vocab,n,m,masked", [(1, 8194, 900, 0, False), (3, 70, 40, 5, True), (2, 2048, 0, 3, False), (4, 2049, 300, 0, True),
                                                   (1, 1, 2, 1, True), (2, 131, 0, 0, True), (2, 40001, 5000, 200, True), (3, 33, 0, 0, False)])
def test_adjust_matches_float64(ops, dtype, rows, vocab, n, m, masked):
    say(f"[gpu] adjust logits {dtype} {rows}x{vocab} history={n} biases={m} masked={masked}")
    g = gen(8)
    x = (3 * randn(g, rows, vocab)).to(dtype)
    history = torch.randint(-2, min(vocab, 500) + 2, (rows, n), generator=g, device="cuda").int()
    kw = dict(history=history, repetition=1 + torch.rand(rows, generator=g, device="cuda"), frequency=torch.rand(rows, generator=g, device="cuda"),
              presence=0.7)
    ref = [history, kw["repetition"], kw["frequency"], 0.7, None, None, None]
    if m:
        kw["bias_tokens"] = torch.randint(-1, vocab + 1, (rows, m), generator=g, device="cuda").int()  # some twice: the last counts
        kw["bias"] = randn(g, rows, m)
        ref[4], ref[5] = kw["bias_tokens"], kw["bias"]
    if masked:
        kw["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (rows, (vocab + 31) // 32), generator=g, device="cuda").int()
        ref[6] = kw["allowed"]
    want, tol = adjust_ref(x, *ref)
    got = ops.adjust_logits(x, **kw)
    same(got, want, tol)
    for _ in range(3):
        assert torch.equal(got, ops.adjust_logits(x, **kw))
    y = x.clone()
    assert ops.adjust_logits(y, out=y, **kw).data_ptr() == y.data_ptr() and torch.equal(y, got)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_adjust_odd_values(ops, dtype):
    """Infinities and NaN, a row whose mask leaves nothing, the same token all over a history, rows at odd addresses, lists
    shared by all rows."""
    say(f"[gpu] adjust logits odd values {dtype}")
    wide = (2 * randn(gen(1), 4, 2100)).to(dtype)
    x = wide[:, 3:2096]
    x[0, 5], x[0, 6], x[0, 7], x[1, 2092] = INF, -INF, NAN, -INF
    history = ints([[5, 6, 7, 7, 9, 2092] + [11] * 60000]).expand(4, -1)
    allowed = torch.full((4, 66), -1, dtype=torch.int32, device="cuda")
    allowed[2] = 0
    out = torch.full((4, 2100), 9.0, dtype=dtype, device="cuda")
    got = ops.adjust_logits(x, history=history, repetition=1.3, frequency=0.01, presence=-0.2, allowed=allowed, out=out[:, 1:2094])
    want, tol = adjust_ref(x, history, 1.3, 0.01, -0.2, allowed=allowed)
    same(got, want, tol)
    assert (got[2] == -INF).all() and (out[:, 0] == 9).all() and (out[:, 2094:] == 9).all()
    plain = ops.adjust_logits(x)
    assert torch.equal(plain.view(torch.int16 if dtype != F32 else torch.int32), x.contiguous().view(torch.int16 if dtype != F32 else torch.int32))
    assert ops.adjust_logits(x[:0]).shape == (0, 2093)
    for kw, match in ((dict(repetition=0.0), "repetition"), (dict(presence=INF), "presence"), (dict(bias=x.float()), "bias_tokens"),
                      (dict(allowed=allowed[:, :65]), "allowed"), (dict(history=history.long()), "history"),
                      (dict(frequency=torch.ones(3, device="cuda")), "frequency"), (dict(out=wide[:, :2093]), None)):
        if match is None:
            continue
        with pytest.raises(H.ValidationError, match=match):
            ops.adjust_logits(x, **kw)


def test_adjust_refuses_shifted_memory(ops):
    """Out beside logits in their memory is fine, over them in other places is not."""
    say("[gpu] adjust logits in shifted memory")
    wide = randn(gen(3), 4, 2100)
    x = wide[:, 3:2096]
    for out in (wide[:, :2093], wide[:, 7:2100], wide.flatten()[2100 + 3:2100 + 3 + 3 * 2093].view(3, 2093)):
        with pytest.raises(H.ValidationError, match="out: "):
            ops.adjust_logits(x[:len(out)], out=out)
    both = torch.cat([x, x], 1)
    want = ops.adjust_logits(x, repetition=2.0, history=ints([[5, 9]]).expand(4, -1))
    ops.adjust_logits(both[:, :2093], repetition=2.0, history=ints([[5, 9]]).expand(4, -1), out=both[:, 2093:])
    assert torch.equal(both[:, 2093:], want) and torch.equal(both[:, :2093], x)


# ---- together ----------------------------------------------------------------------------
@pytest.mark.parametrize("types", [(F32, BF16), (BF16, 4)])
def test_decoding_over_pages(ops, types):
    """Prompts, then steps of two sequences, as a program runs them: appended with rotation, attended, the step's logits
    adjusted and scored, in one captured step; every result against the rows kept apart in float64, and in the end against
    the tree attention over the gathered caches."""
    say(f"[gpu] decoding over pages {types}")
    q_type, kv = types
    h, hk, d, page, steps = 4, 2, 64, 16, 6
    g = gen(12)
    cache = ops.paged_cache(12, hk, page, d, BF16, bits=4 if kv == 4 else 16)
    for t in cache:
        if t is not None:
            t.fill_(255 if t.dtype == torch.uint8 else NAN)
    table, rot = ints([[4, 9, 1, 7], [2, 0, 11, 5]]), rotation_table(64, d)
    kept = [[], []]
    prompt = [29, 14]

    def remember(k, starts, lens):
        kk = k.double()
        for b in range(2):
            for i in range(starts[b + 1] - starts[b]):
                kept[b].append(turn(kk[starts[b] + i:starts[b] + i + 1], rot, torch.tensor([lens[b] + i], device="cuda"), False)[0])

    def expected(q, starts, lens):
        k, v = ops.paged_gather(cache, ints(lens), table, max(lens))
        for b in range(2):
            for i in range(starts[b + 1] - starts[b]):
                pos = lens[b] - (starts[b + 1] - starts[b]) + i
                kk, vv = (t[b, :, :pos + 1].double().repeat_interleave(h // hk, 0) for t in (k, v))
                p = torch.softmax((q[starts[b] + i].double().unsqueeze(1) * kk).sum(-1) * d ** -0.5, -1)
                yield starts[b] + i, (p.unsqueeze(-1) * vv).sum(1)

    x = randn(g, sum(prompt), h + 2 * hk, d, dtype=q_type)
    starts = [0, prompt[0], sum(prompt)]
    r = ops.paged_append(cache, x[:, h:h + hk], x[:, h + hk:], ints(starts), ints([0, 0]), table, q=x[:, :h], rotation=rot)
    out = ops.paged_attention(r.q, cache, ints(starts), r.lengths, table)
    remember(x[:, h:h + hk], starts, [0, 0])
    loose = 0.02 if q_type == BF16 else 2e-5  # of values around 1: half a step of the result, and what the tests above bound
    for token, want in expected(r.q, starts, prompt):
        assert ((out[token].double() - want).abs() <= loose).all()

    head = randn(g, h * d, 300) * 0.1
    held, one = r.lengths.clone(), ints([0, 1, 2])
    step_x = torch.empty((2, h + 2 * hk, d), dtype=q_type, device="cuda")
    history = torch.full((2, steps), -1, dtype=torch.int32, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())

    def step():
        a = ops.paged_append(cache, step_x[:, h:h + hk], step_x[:, h + hk:], one, held, table, q=step_x[:, :h], rotation=rot)
        o = ops.paged_attention(a.q, cache, one, a.lengths, table)
        logits = ops.adjust_logits(o.float().flatten(1) @ head, history=history, repetition=1.2, frequency=0.1)
        held.copy_(a.lengths)
        return a.q, o, logits, ops.token_scores(logits, top_n=1)

    with torch.cuda.stream(stream):
        step_x.zero_()
        step()  # the library of the product with `head` sets itself up with its first call, which must not be captured
        held.copy_(r.lengths)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            q, o, logits, scores = step()
        lens = list(prompt)
        for i in range(steps):
            step_x.copy_(randn(g, 2, h + 2 * hk, d, dtype=q_type))
            graph.replay()
            stream.synchronize()
            remember(step_x[:, h:h + hk], [0, 1, 2], lens)
            lens = [n + 1 for n in lens]
            assert held.tolist() == lens
            for token, want in expected(q, [0, 1, 2], lens):
                assert ((o[token].double() - want).abs() <= loose).all()
            want, tol = adjust_ref((o.float().flatten(1) @ head), history, 1.2, 0.1, 0.0)
            same(logits, want, tol + 1e-4)
            assert torch.equal(scores.top_tokens[:, 0].long(), logits.argmax(-1))
            history[:, i] = scores.top_tokens[:, 0]
    # the cache holds what was appended, and as one piece gives the tree attention the same rows
    k, v = ops.paged_gather(cache, held, table, 64)
    for b in range(2):
        want = torch.stack(kept[b], 1)
        got = k[b, :, :lens[b]].double()
        tol = HALF[BF16] * want.abs() + 1e-30 if kv != 4 else (want.amax(-1, keepdim=True) - want.amin(-1, keepdim=True)) / 15 * 0.51 + 1e-2
        assert ((got - want).abs() <= tol).all()
    k, v = k.to(BF16), v.to(BF16)
    tree = ops.tree_attention(q.unsqueeze(1), k, v, ints([n - 1 for n in lens]), ints([[-1], [-1]]))
    assert ((tree[:, 0].double() - o.double()).abs() <= (loose if kv != 4 else 0.05)).all()
