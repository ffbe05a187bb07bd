"""Operators of a decoder that reads an encoder's states (attention to them, heads with positions of several axes, page bookkeeping on the device), each
against its definition in 64 bits at the sizes, lengths and masks where it can go wrong, and all of them together as they are used.

Tolerances.  float32 attention: a score is a sum of d products (rounded 2^-24 of its terms each), an exponent moves by that times log2(e), the result is a mean of
values: 2^-24 * (sqrt(d) for the sums + a few) of values of size one stays below 4e-6.  bfloat16 attention: the results and the weights are rounded
to 2^-9 of themselves each (half a step is eps / 2 = 2^-8 of the value at worst); a weighted mean of values of size v with weights that are off by 2^-8 at
most is off by 2^-8 of the mean of |v| (at most 4.5 here: normal draws), and rounding it adds 2^-8 of itself: 2 * 2^-8 * max|v| bounds any element, and the 2-norm's share is below
2^-8.  Heads: one rounding of the result (2^-8 or, with the norm's four roundings in 32 bits and the angle's, 2^-21 of |x| for float32).
"""
import math
import random
from types import SimpleNamespace

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
DTYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(scope="module")
def ops():
    from marin_b200.kernels import ops as o
    return o


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


# ---- attention to an encoder's states ----------------------------------------------------------------------------------------

class Case:
    """Queries of requests with `new` tokens over sources of `src` positions, in scattered pages; what no request sees is NaN."""

    def __init__(self, dtype, H, K, d, page, new, src, spans=None, seed=0, wide=0, pad_rows=0, size=1.0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.H, self.K, self.d, self.page, self.new, self.src = H, K, d, page, new, src
        counts = [-(-s // page) for s in src]
        order = torch.randperm(sum(counts) + 2, generator=g, device=DEV).tolist()
        self.k, self.v = (torch.full((len(order), K, page, d), float("nan"), device=DEV, dtype=dtype) for _ in range(2))
        table = [[0] * (max(counts + [1]) + 1) for _ in src]
        self.keys, self.values = [], []
        for r, (s, n) in enumerate(zip(src, counts)):
            key, value = (torch.randn(s, K, d, generator=g, device=DEV).to(dtype) for _ in range(2))
            for j in range(n):
                p = table[r][j] = order.pop()
                rows = slice(j * page, min(s, (j + 1) * page))
                self.k[p, :, :rows.stop - rows.start] = key[rows].transpose(0, 1)
                self.v[p, :, :rows.stop - rows.start] = value[rows].transpose(0, 1)
            self.keys.append(key.double())
            self.values.append(value.double())
        T = sum(new)
        whole = (size * torch.randn(T + pad_rows, H * d + wide, generator=g, device=DEV)).to(dtype)
        self.q = whole[:, :H * d]
        self.out = torch.full((T + pad_rows, H * d), 7.0, device=DEV, dtype=dtype)
        self.table, self.lens, self.scale = ints(table), ints(src), 1.0 / math.sqrt(d)
        cu = [sum(new[:r]) for r in range(len(new) + 1)]
        nd = next((i for i, n in enumerate(new) if n != 1), len(new))
        self.ctx = SimpleNamespace(num_tokens=T, num_requests=len(new), num_decode=nd, max_query_len=max(new), cu_tokens=ints(cu))
        self.limits = spans if spans is not None else [(0, s) for s, n in zip(src, new) for _ in range(n)]
        self.spans = None if spans is None else ints(spans + [(0, 1 << 30)] * pad_rows)

    def run(self, ops):
        ops.attention_cross(self.q, self.k, self.v, self.out, self.ctx, ops.Source(self.table, self.lens, max(self.src)), self.H, self.K, self.d, self.scale, self.spans)
        return self.out

    def want(self):
        H, d, G, T = self.H, self.d, self.H // self.K, sum(self.new)
        out = torch.full(self.out.shape, 7.0, device=DEV, dtype=torch.float64)
        first = 0
        for r, n in enumerate(self.new):
            s = self.src[r]
            for h in range(H):
                limit = torch.tensor(self.limits[first:first + n], device=DEV, dtype=torch.int64).view(-1, 2)
                at = torch.arange(s, device=DEV)
                seen = (at >= limit[:, :1]) & (at < limit[:, 1:])
                scores = self.q[first:first + n, h * d:(h + 1) * d].double() @ self.keys[r][:, h // G].t() * self.scale
                p = torch.softmax(scores.masked_fill(~seen, -math.inf), -1).nan_to_num(0.0)
                out[first:first + n, h * d:(h + 1) * d] = p @ self.values[r][:, h // G]
            first += n
        return out

    def check(self, ops):
        got, want = self.run(ops).double(), self.want()
        T = sum(self.new)
        assert torch.equal(got[T:], want[T:])                        # rows behind the last request stay as they were
        if T == 0:
            return
        empty = torch.tensor([hi <= lo or lo >= s or hi <= 0 for (lo, hi), s in zip(self.limits, [s for s, n in zip(self.src, self.new) for _ in range(n)])], device=DEV)
        assert (got[:T][empty] == 0).all()
        if self.q.dtype == torch.float32:
            torch.testing.assert_close(got, want, rtol=0, atol=4e-6)
        else:
            most = max([float(v.abs().max()) for v in self.values if v.numel()] or [1.0])
            torch.testing.assert_close(got, want, rtol=0, atol=2 * most * 2.0 ** -8)
            off = (got[:T] - want[:T]).norm() / want[:T].norm().clamp(min=1e-30)
            assert float(off) <= 2.0 ** -8 or float(want[:T].norm()) == 0.0


LAYOUTS = [(32, 8, 128, 16), (40, 8, 128, 32), (16, 8, 64, 64), (8, 8, 80, 16), (14, 2, 96, 16), (6, 6, 48, 16), (4, 1, 16, 8), (5, 1, 20, 4), (3, 3, 7, 1), (2, 1, 256, 16), (34, 2, 64, 16)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,K,d,page", LAYOUTS)
def test_cross_layouts(ops, dtype, H, K, d, page):
    """Every head layout and page size: single tokens and portions in one step, sources of one position to several chunks, one request without any."""
    Case(dtype, H, K, d, page, [1, 1, 1, 7, 33, 2, 70], [1, 0, 300, 129, 64, 0, 515], seed=H).check(ops)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("src", [1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 257, 1000, 2049])
def test_cross_source_lengths(ops, dtype, src):
    Case(dtype, 8, 2, 64, 16, [1, 40], [src, src], seed=src).check(ops)
    Case(dtype, 8, 2, 128, 16, [1, 1, 5], [src, 3, src], seed=src).check(ops)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [1, 2, 3, 16, 31, 32, 33, 63, 64, 65, 128, 200])
def test_cross_portion_lengths(ops, dtype, new):
    Case(dtype, 16, 4, 128, 16, [new], [200], seed=new).check(ops)
    Case(dtype, 10, 2, 64, 32, [1] * 3 + [new + 1, new + 5], [77, 0, 500, 130, 33], seed=new).check(ops)


def spread_spans(new, src, seed):
    """Runs of every kind: all of the source, none, one position, past the end, from the middle, reversed and negative bounds."""
    rng = random.Random(seed)
    out = []
    for n, s in zip(new, src):
        for _ in range(n):
            kind = rng.randrange(7)
            a, b = sorted((rng.randint(0, s), rng.randint(0, s)))
            out.append([(0, s), (0, 0), (a, a + 1), (a, s + 50), (a, b), (b + 1, a), (-5, b)][kind])
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,K,d,page", [(32, 8, 128, 16), (8, 8, 64, 32), (14, 2, 80, 16), (5, 1, 24, 4)])
def test_cross_spans(ops, dtype, H, K, d, page):
    new, src = [1, 1, 1, 1, 9, 50, 150], [300, 0, 1, 700, 200, 900, 64]
    for seed in range(3):
        Case(dtype, H, K, d, page, new, src, spread_spans(new, src, seed), seed=seed, pad_rows=3).check(ops)
    empty = [(5, 5)] * sum(new)
    Case(dtype, H, K, d, page, new, src, empty).check(ops)


@pytest.mark.parametrize("dtype", DTYPES)
def test_cross_what_is_not_seen_may_be_anything(ops, dtype):
    """NaN and infinities in positions of the source that a token's span leaves out do not reach it, also where other tokens of the portion do see them."""
    new, src = [1, 12, 40], [200, 300, 150]
    spans = [(10, 100)] + [(0, 120) if t % 2 else (130, 300) for t in range(12)] + [(0, 100) if t % 3 else (60, 150) for t in range(40)]
    case = Case(dtype, 8, 2, 64, 16, new, src, spans, seed=4)
    for r, places in ((0, [3, 150]), (1, [125, 200]), (2, [120])):
        for j in places:
            page, at = int(case.table[r, j // 16]), j % 16
            case.v[page, :, at], case.k[page, :, at] = float("nan"), float("inf")
    got, want = case.run(ops).double(), case.want()                  # (want has the finite source)
    tokens = [True] + [t % 2 == 1 for t in range(12)] + [t % 3 != 0 for t in range(40)]
    clean = torch.tensor(tokens, device=DEV)
    atol = 4e-6 if dtype == torch.float32 else 2 * 4.5 * 2.0 ** -8
    torch.testing.assert_close(got[clean], want[clean], rtol=0, atol=atol)
    assert torch.isnan(got[~clean]).all()                            # those that see it


@pytest.mark.parametrize("dtype", DTYPES)
def test_cross_large_scores(ops, dtype):
    """Scores of a few hundred: one position takes all the weight, the running maximum moves far and often."""
    case = Case(dtype, 8, 2, 64, 16, [1, 1, 60], [900, 40, 700], size=200.0, seed=5)
    got, want = case.run(ops).double(), case.want()
    # scores up to 1,000 are off by 2^-24 of the largest of their terms' sums: weights by up to 1e-3 of themselves in float32
    torch.testing.assert_close(got, want, rtol=0, atol=2e-3 if dtype == torch.float32 else 2 * 4.5 * 2.0 ** -8)


@pytest.mark.parametrize("dtype", DTYPES)
def test_cross_columns_of_wider_rows_and_rows_behind(ops, dtype):
    for wide in (8, 24, 3):
        Case(dtype, 8, 2, 64, 16, [1, 1, 20], [100, 30, 260], wide=wide, pad_rows=5, seed=wide).check(ops)


def test_cross_float32_bits_do_not_depend_on_the_batch(ops):
    """A row's float32 result is the same bits alone, in a portion, cut into portions and in a batch with longer sources."""
    whole = Case(torch.float32, 8, 2, 64, 16, [1, 90], [500, 700], seed=9)
    got = whole.run(ops).clone()
    rows = [got[1:]]
    for parts in ([30, 60], [1, 89], [2, 3, 85]):
        at, outs = 1, []
        for n in parts:
            ctx = SimpleNamespace(num_tokens=n, num_requests=1, num_decode=int(n == 1), max_query_len=n, cu_tokens=ints([0, n]))
            out = torch.empty(n, 512, device=DEV)
            ops.attention_cross(whole.q[at:at + n], whole.k, whole.v, out, ctx, ops.Source(whole.table[1:], whole.lens[1:], 5000), 8, 2, 64, whole.scale)
            outs.append(out)
            at += n
        rows.append(torch.cat(outs))
    for other in rows[1:]:
        assert torch.equal(other, rows[0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_cross_twice_and_from_a_graph(ops, dtype):
    """The same bits in every run; a captured call reads the buffers of its replay, two captured calls share nothing, another stream than the tensors' own."""
    a, b = (Case(dtype, 32, 8, 128, 16, [1, 1, 30], [900, 0, 1500], seed=s) for s in (1, 2))
    first, second = a.run(ops).clone(), b.run(ops).clone()
    assert torch.equal(a.run(ops), first)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(stream):
        for c in (a, b):
            c.run(ops)
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                c.run(ops)
            graphs.append(graph)
    stream.synchronize()
    a.out.zero_(), b.out.zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        graphs[0].replay()
    graphs[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(a.out, first) and torch.equal(b.out, second)
    a.lens[0] = 37                                                   # another length of the same buffers
    a.src[0], a.keys[0], a.values[0], a.limits[0] = 37, a.keys[0][:37], a.values[0][:37], (0, 37)
    graphs[0].replay()
    torch.testing.assert_close(a.out.double(), a.want(), rtol=0, atol=4e-6 if dtype == torch.float32 else 2 * 4.6 * 2.0 ** -8)


@pytest.mark.parametrize("dtype", DTYPES)
def test_cross_infinite_scores(ops, dtype):
    """What softmax makes of infinities: keys that score minus infinity have no weight; where all of them do, or one scores plus infinity, the result is NaN."""
    case = Case(dtype, 8, 2, 64, 16, [1, 20], [200, 200], seed=8)
    case.q[:, :] = 1.0
    for r in range(2):
        for j in range(0, 200, 3):
            case.k[int(case.table[r, j // 16]), :, j % 16] = float("-inf")
        case.keys[r][::3] = float("-inf")
    torch.testing.assert_close(case.run(ops).double(), case.want(), rtol=0, atol=4e-6 if dtype == torch.float32 else 2 * 4.5 * 2.0 ** -8)
    for r in range(2):
        for page in case.table[r, :13].tolist():
            case.k[page] = float("-inf")
    assert torch.isnan(case.run(ops)).all()
    for r in range(2):
        case.k[int(case.table[r, 3]), :, 5] = float("inf")
    assert torch.isnan(case.run(ops)).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,K,d", [(8, 2, 64), (32, 2, 128)])
def test_cross_infinite_values(ops, dtype, H, K, d):
    """A value that is infinite and seen makes its column infinite, and no other."""
    case = Case(dtype, H, K, d, 16, [1, 1, 20], [300, 16, 300], seed=9)
    for r in range(3):
        case.v[int(case.table[r, 0]), :, 5, 3] = float("inf")
        case.v[int(case.table[r, 0]), :, 7, 9] = float("-inf")
        case.values[r][5, :, 3], case.values[r][7, :, 9] = float("inf"), float("-inf")
    got, want = case.run(ops).double(), case.want()
    assert torch.equal(got.isposinf(), want.isposinf()) and torch.equal(got.isneginf(), want.isneginf()) and want.isinf().sum() == 2 * 22 * H
    whole = want.isfinite()
    torch.testing.assert_close(got[whole], want[whole], rtol=0, atol=4e-6 if dtype == torch.float32 else 2 * 5.0 * 2.0 ** -8)


@pytest.mark.parametrize("dtype", DTYPES)
def test_cross_padded_batch(ops, dtype):
    """Requests without a token among those of single tokens and behind them (what a captured step of a fixed size holds): the rows that others have, and those behind, are theirs."""
    case = Case(dtype, 8, 2, 64, 16, [1, 1, 1], [100, 37, 64], seed=10, pad_rows=3)
    want = case.want()
    case.ctx.num_requests = case.ctx.num_decode = 6
    case.ctx.cu_tokens = ints([0, 1, 2, 3, 3, 3, 3])
    case.table, case.lens = torch.cat([case.table, case.table]), ints([100, 37, 64, 100, 37, 0])
    got = case.run(ops).double()
    assert torch.equal(got[3:], want[3:])
    torch.testing.assert_close(got, want, rtol=0, atol=4e-6 if dtype == torch.float32 else 2 * 4.5 * 2.0 ** -8)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [[1, 1], [1], [9, 30]])
def test_cross_one_row_for_all(ops, dtype, new):
    """Queries that are one row in memory (a stride of nothing), and a single row with a stride that says nothing."""
    case = Case(dtype, 8, 2, 64, 16, new, [100, 37][:len(new)], seed=16)
    case.q = case.q[:1].expand(sum(new), -1) if len(new) > 1 else torch.as_strided(case.q, (1, 512), (3, 1))
    case.check(ops)


def test_cross_many_requests_and_long_batches(ops):
    """More requests and tiles than places for blocks, single tokens ahead of portions of unlike lengths."""
    rng = random.Random(3)
    new = [1] * 150 + [rng.choice([2, 17, 33, 64, 65, 129]) for _ in range(40)]
    src = [rng.choice([0, 1, 16, 63, 64, 65, 100, 333]) for _ in new]
    Case(torch.bfloat16, 16, 4, 64, 16, new, src, seed=12).check(ops)
    Case(torch.bfloat16, 5, 1, 128, 32, new, src, spread_spans(new, src, 4), seed=13).check(ops)
    Case(torch.float32, 4, 2, 32, 16, new, src, spread_spans(new, src, 5), seed=14).check(ops)


@pytest.mark.parametrize("dtype", DTYPES)
def test_cross_one_long_portion_among_many(ops, dtype):
    """Tiles found by the rows there are: more requests than a search step looks at, some without a token, the long portion first, in the middle and last."""
    for at, n, seed in ((0, 40, 1), (517, 1100, 2), (32, 33, 3), (0, 1, 4)):
        new = [(2, 0, 5, 33)[i % 4] for i in range(n)]
        new[at] = 700
        src = [(17, 64, 0, 65, 30)[i % 5] for i in range(n)]
        src[at] = 130
        Case(dtype, 4, 2, 16, 16, new, src, seed=seed, pad_rows=2).check(ops)


@pytest.mark.parametrize("K", [4, 64])
@pytest.mark.parametrize("R", [127, 128, 129])
def test_cross_many_single_tokens(ops, R, K):
    """More single tokens than places for their blocks: every request once, sources of all lengths and of one, some of nothing; padded ones among them."""
    rng = random.Random(R)
    for src in ([rng.choice([0, 1, 17, 300, 301]) for _ in range(R)], [33] * R):
        case = Case(torch.bfloat16, K, K, 16, 16, [1] * R, src, seed=R)
        case.check(ops)
    case.ctx.cu_tokens[R:] = R - 1                                    # the last has no token
    case.out.fill_(7.0)
    got, want = case.run(ops).double(), case.want()
    assert (got[R - 1] == 7.0).all()
    torch.testing.assert_close(got[:R - 1], want[:R - 1], rtol=0, atol=2 * 5.0 * 2.0 ** -8)


def test_cross_far_pages(ops):
    """Pages whose first element lies past 2^31 in the cache."""
    H, K, d, page = 4, 2, 128, 64
    pages = (1 << 31) // (K * page * d) + 70                         # a little over 2^31 elements, 4.3 GB each
    k, v = (torch.empty(pages, K, page, d, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    case = Case(torch.bfloat16, H, K, d, page, [1, 30], [500, 260], seed=11)
    far = pages - case.k.shape[0]
    k[far:], v[far:] = case.k, case.v
    case.k, case.v, case.table = k, v, (case.table + far).contiguous()
    case.check(ops)


# ---- heads with positions of several axes ----------------------------------------------------------------------------------------

def axes_want(rows, qw, kw, eps, positions, axis_of, inv_freq, rotary, interleaved, H, K, d):
    T, half = rows.shape[0], rotary // 2
    x = rows[:, :(H + 2 * K) * d].double().view(T, H + 2 * K, d)
    done = x.clone()
    for part, w in ((slice(0, H), qw), (slice(H, H + K), kw)):
        y = x[:, part]
        if w is not None:
            y = y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + eps) * w.double()
        y = y.clone()
        if inv_freq is not None:
            angle = (positions[axis_of.long()].double().t() * inv_freq.double())[:, None]
            a, b = (slice(0, rotary, 2), slice(1, rotary, 2)) if interleaved else (slice(0, half), slice(half, rotary))
            p, q = y[..., a].clone(), y[..., b].clone()
            y[..., a], y[..., b] = p * angle.cos() - q * angle.sin(), q * angle.cos() + p * angle.sin()
        done[:, part] = y
    return done[:, :H], done[:, H:H + K], done[:, H + K:]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,K,d,rotary,page", [(32, 8, 128, 128, 16), (40, 8, 128, 64, 32), (16, 16, 80, 80, 16), (14, 2, 96, 96, 64), (5, 1, 64, 64, 16), (3, 2, 256, 256, 16),
                                               (4, 2, 40, 20, 4), (2, 1, 7, 6, 1), (6, 3, 512, 512, 16), (0, 4, 128, 128, 16), (1, 1, 24, 16, 16), (9, 3, 72, 48, 8), (64, 64, 32, 32, 16), (1, 1, 256, 256, 16), (96, 8, 128, 128, 16)])
def test_axes(ops, dtype, H, K, d, rotary, page):
    g = torch.Generator(device=DEV).manual_seed(d + H)
    for T, axes, interleaved, norm, wide, padded in ((1, 1, False, True, 0, 0), (9, 3, True, False, 8, 2), (70, 2, False, True, 16, 3), (33, 4, True, True, 5, 0), (12, 3, False, False, 0, 1)):
        half = rotary // 2
        rows = torch.randn(T, (H + 2 * K) * d + wide, generator=g, device=DEV).to(dtype)[:, :(H + 2 * K) * d]
        qw, kw = ((1 + 0.3 * torch.randn(d, generator=g, device=DEV)) if norm else None for _ in range(2))
        axis_of = torch.randint(0, axes, (half,), generator=g, device=DEV).int()
        inv_freq = torch.pow(10000.0, -2.0 * torch.arange(half, device=DEV) / rotary).float()
        positions = torch.randint(0, 2_000_000_000 if T == 9 else 5000, (axes, T), generator=g, device=DEV).int()
        pages = -(-T // page) + 2
        slots = torch.randperm(pages * page, generator=g, device=DEV)[:T].int()
        if padded:
            slots[-padded:] = -1
        if T == 70:
            slots[0] = pages * page + 3                              # no place of the cache: nothing is stored
        k, v = (torch.full((pages, K, page, d), 9.0, device=DEV, dtype=dtype) for _ in range(2))
        q_out = torch.empty(T, H * d, device=DEV, dtype=dtype) if H else None
        ops.qk_norm_axes_write(rows, q_out, qw, kw, 1e-6, positions, axis_of, inv_freq, rotary, interleaved, slots, k, v, H, K, d)
        q_want, k_want, v_want = axes_want(rows, qw, kw, 1e-6, positions, axis_of, inv_freq, rotary, interleaved, H, K, d)
        k_ref, v_ref = (torch.full((pages, K, page, d), 9.0, device=DEV, dtype=torch.float64) for _ in range(2))
        for t, s in enumerate(slots.tolist()):
            if 0 <= s < pages * page:
                k_ref[s // page, :, s % page], v_ref[s // page, :, s % page] = k_want[t], v_want[t]
        tol = dict(rtol=2.0 ** -21, atol=2.0 ** -19) if dtype == torch.float32 else dict(rtol=2.0 ** -8, atol=2.0 ** -17)
        if H:
            torch.testing.assert_close(q_out.double(), q_want.reshape(T, H * d), **tol)
        torch.testing.assert_close(k.double(), k_ref, **tol)
        assert torch.equal(v.double(), v_ref)                        # values are copied


def test_axes_queries_alone_and_without_rotation(ops):
    g = torch.Generator(device=DEV).manual_seed(1)
    rows = torch.randn(11, 8 * 64, generator=g, device=DEV).bfloat16()
    w = 1 + 0.2 * torch.randn(64, generator=g, device=DEV)
    q = torch.empty_like(rows)
    ops.qk_norm_axes_write(rows, q, w, None, 1e-6, None, None, None, 0, False, None, None, None, 8, 0, 64, write_kv=False)
    want, _, _ = axes_want(rows, w, None, 1e-6, None, None, None, 0, False, 8, 0, 64)
    torch.testing.assert_close(q.double(), want.reshape(11, -1), rtol=2.0 ** -8, atol=2.0 ** -17)


def test_axes_one_axis_is_the_rotation_that_was_there(ops):
    """With one axis and near positions the result is qk_norm_rope_write's up to one rounding."""
    g = torch.Generator(device=DEV).manual_seed(2)
    H, K, d, T, page = 8, 2, 128, 20, 16
    rows = torch.randn(T, (H + 2 * K) * d, generator=g, device=DEV).bfloat16()
    qw, kw = (1 + 0.2 * torch.randn(d, generator=g, device=DEV) for _ in range(2))
    inv_freq = torch.pow(10000.0, -2.0 * torch.arange(64, device=DEV) / 128).float()
    positions, slots = torch.arange(T, device=DEV).int(), torch.arange(T, device=DEV).int()
    got, was = ([torch.zeros(T, H * d, device=DEV, dtype=torch.bfloat16)] + [torch.zeros(2, K, page, d, device=DEV, dtype=torch.bfloat16) for _ in range(2)] for _ in range(2))
    ops.qk_norm_axes_write(rows, got[0], qw, kw, 1e-6, positions[None].contiguous(), torch.zeros(64, device=DEV).int(), inv_freq, 128, False, slots, got[1], got[2], H, K, d)
    ops.qk_norm_rope_write(rows, was[0], qw, kw, 1e-6, positions, inv_freq, 128, False, slots, was[1], was[2], H, K, d)
    for a, b in zip(got, was):
        torch.testing.assert_close(a.float(), b.float(), rtol=2.0 ** -7, atol=2.0 ** -15)


# ---- page bookkeeping on the device ------------------------------------------------------------------------------------------------

def page_step_want(before, after, table, free, count, page, room):
    """One request after another, as a host would."""
    R, columns = len(before), len(table[0])
    need = [-(-max(a, b) // page) for a, b in zip(after, before)]
    taken = sum(max(0, -(-a // page) - -(-b // page)) for a, b in zip(after, before))
    back = sum(max(0, -(-b // page) - -(-a // page)) for a, b in zip(after, before))
    tokens = sum(max(0, a - b) for a, b in zip(after, before))
    status = 0
    if min(before + after) < 0 or max(need) > columns:
        status = 3
    elif tokens > room:
        status = 2
    elif not 0 <= count <= len(free):
        status = 4
    elif taken > count + back:
        status = 1
    elif count + back - taken > len(free):
        status = 4
    if status:
        return table, free, [count, status], [0] * (R + 1), [0] * room, [0] * room, [-1] * room
    table, free, stack = [list(row) for row in table], list(free), list(free[:count])
    for r in range(R):
        stack += table[r][-(-after[r] // page):-(-before[r] // page)]
    cu, req, pos, slots = [0], [], [], []
    for r in range(R):
        for c in range(-(-before[r] // page), -(-after[r] // page)):
            table[r][c] = stack.pop()
        for p in range(before[r], after[r]):
            req.append(r), pos.append(p), slots.append(table[r][p // page] * page + p % page)
        cu.append(len(req))
    free[count:len(stack)] = stack[count:]
    pad = room - len(req)
    return table, free, [len(stack), 0], cu, req + [0] * pad, pos + [0] * pad, slots + [-1] * pad


def page_case(R, page, kind, seed):
    rng = random.Random(seed)
    before = [rng.choice([0, 1, page - 1, page, page + 1, rng.randint(0, 9 * page)]) for _ in range(R)]
    grow = {"decode": lambda b: b + 1, "mixed": lambda b: rng.choice([b, b + 1, b + rng.randint(0, 5 * page), 0, b // 2, max(0, b - 1)]), "ended": lambda b: 0,
            "prompts": lambda b: b + rng.randint(1, 300), "same": lambda b: b}[kind]
    after = [grow(b) for b in before]
    held = [-(-b // page) for b in before]
    columns = max(-(-max(a, b) // page) for a, b in zip(after, before)) + rng.randint(0, 2) or 1
    taken = sum(max(0, -(-a // page) - h) for a, h in zip(after, held))
    back = sum(max(0, h - -(-a // page)) for a, h in zip(after, held))
    count = max(0, taken - back) + rng.choice([0, 0, 3, 50])
    ids = list(range(sum(held) + count))
    rng.shuffle(ids)
    table = [[ids.pop() for _ in range(h)] + [-1] * (columns - h) for h in held]
    free = ids + [-7] * (sum(held) + rng.choice([0, 4]))
    room = sum(max(0, a - b) for a, b in zip(after, before)) + rng.choice([0, 0, 1, 40])
    return before, after, table, free, count, page, room


def run_pages(ops, before, after, table, free, count, page, room):
    t = [ints(before), ints(after), ints(table), ints(free).reshape(-1), ints([count])]
    out = [torch.full((n,), 99, dtype=torch.int32, device=DEV) for n in (2, len(before) + 1, room, room, room)]
    ops.page_step(*t, page, *out)
    assert t[0].tolist() == list(before) and t[1].tolist() == list(after) and t[4].tolist() == [count]
    return [t[2].tolist(), t[3].tolist()] + [x.tolist() for x in out]


@pytest.mark.parametrize("kind", ["decode", "mixed", "ended", "prompts", "same"])
@pytest.mark.parametrize("R,page", [(1, 16), (2, 1), (7, 16), (31, 64), (256, 16), (257, 32), (1023, 16), (2500, 8)])
def test_page_step(ops, kind, R, page):
    for seed in range(3):
        case = page_case(R, page, kind, seed)
        assert run_pages(ops, *case) == [list(x) for x in page_step_want(*case)]


def test_page_step_all_or_nothing(ops):
    """Where a step cannot be done no page moves and the status says why."""
    before, after, table, free, count, page, room = page_case(40, 16, "mixed", 3)
    cases = []
    need = page_step_want(before, after, table, free, count, page, room)[2][0]
    cases.append((before, [a + 16 * (need + 1) * (i == 0) if i == 0 else a for i, a in enumerate(after)], [row + [-1] * (need + 40) for row in table], free, count, page, room + 16 * need + 2000))
    cases.append((before, after, table, free, count, page, room - 45))
    cases.append((before, after[:-1] + [len(table[0]) * 16 + 1], table, free, count, page, room + 4000))
    cases.append((before, after[:-1] + [-3], table, free, count, page, room))
    cases.append(([b if i else -1 for i, b in enumerate(before)], after, table, free, count, page, room))
    cases.append((before, after, table, free, len(free) + 1, page, room))
    cases.append((before, after, table, free, -1, page, room))
    cases.append((before, [0] * 40, table, free[:count + 1], count, page, room))
    cases.append(([0] * 40, [2 ** 31 - 1] * 40, table, free, count, page, room))
    seen = set()
    for case in cases:
        if case[-1] < 0:
            continue
        want = [list(x) for x in page_step_want(*case)]
        assert run_pages(ops, *case) == want
        seen.add(want[2][1])
    assert {1, 3, 4} <= seen


def test_page_step_most_requests_and_steps_in_a_row(ops):
    R, page, columns = ops.PAGE_STEP_REQUESTS, 16, 4
    case = ([0] * R, [i % 60 for i in range(R)], [[-1] * columns for _ in range(R)], list(range(4 * R)), 4 * R, page, 59 * R)
    assert run_pages(ops, *case) == [list(x) for x in page_step_want(*case)]
    # thirty steps, each taking over what the one before left: no page is lost or held twice
    rng = random.Random(8)
    R, total = 33, 400
    lens, table, free, left = ints([0] * R), torch.full((R, 12), -1, dtype=torch.int32, device=DEV), ints(list(range(total))), ints([total, 0])
    room = 33 * 60
    host = [0] * R
    for _ in range(30):
        nxt = [rng.choice([0, n, min(190, n + 1), min(190, n + rng.randint(0, 60)), n // 2]) for n in host]
        after, out, now = ints(nxt), [torch.empty(n, dtype=torch.int32, device=DEV) for n in (R + 1, room, room, room)], torch.empty(2, dtype=torch.int32, device=DEV)
        ops.page_step(lens, after, table, free, left[:1].contiguous(), 16, now, *out)
        lens, left = after, now
        host = nxt if int(now[1]) == 0 else host
        if int(now[1]) != 0:
            lens = ints(host)
        rows, n = table.tolist(), int(left[0])
        held = [p for r in range(R) for p in rows[r][:-(-host[r] // 16)]] + free.tolist()[:n]
        assert sorted(held) == list(range(total))


# ---- together -------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
def test_source_operators_together(ops, dtype):
    """An encoder's states come in and are paged, their keys and values written, then two steps of the decoder attend to them: as a layer would run it."""
    g = torch.Generator(device=DEV).manual_seed(3)
    H, K, d, page, src = 8, 2, 64, 16, [90, 0, 33]
    R, room, columns = 3, 140, 8
    table, free = torch.full((R, columns), -1, dtype=torch.int32, device=DEV), torch.randperm(20, generator=g, device=DEV).int()
    left, cu, req, pos, slots = (torch.empty(n, dtype=torch.int32, device=DEV) for n in (2, R + 1, room, room, room))
    ops.page_step(ints([0] * R), ints(src), table, free, ints([20]), page, left, cu, req, pos, slots)
    states = torch.randn(room, 2 * K * d, generator=g, device=DEV).to(dtype)
    k, v = (torch.full((20, K, page, d), float("nan"), device=DEV, dtype=dtype) for _ in range(2))
    kw = 1 + 0.2 * torch.randn(d, generator=g, device=DEV)
    half = d // 2
    inv_freq = torch.pow(10000.0, -2.0 * torch.arange(half, device=DEV) / d).float()
    axis_of = ints(ops.axis_sections([8, 12, 12]))
    at = torch.arange(room, device=DEV)
    positions = torch.stack([at * 0, at // 9, at % 9]).int()
    ops.qk_norm_axes_write(states, None, None, kw, 1e-6, positions, axis_of, inv_freq, d, False, slots, k, v, 0, K, d)
    _, k_want, v_want = axes_want(states, None, kw, 1e-6, positions, axis_of, inv_freq, d, False, 0, K, d)
    for new in ([5, 3, 8], [1, 1, 1]):
        T = sum(new)
        q = torch.randn(T, H * d, generator=g, device=DEV).to(dtype)
        out = torch.empty_like(q)
        ctx = SimpleNamespace(num_tokens=T, num_requests=R, num_decode=R if max(new) == 1 else 0, max_query_len=max(new), cu_tokens=ints([sum(new[:i]) for i in range(R + 1)]))
        ops.attention_cross(q, k, v, out, ctx, ops.Source(table, ints(src), 90), H, K, d, 0.125)
        first = row = 0
        for n, s in zip(new, src):
            for h in range(H):
                keys, values = (x[first:first + s, h // 4].to(dtype).double() for x in (k_want, v_want))
                want = torch.softmax(q[row:row + n, h * d:(h + 1) * d].double() @ keys.t() * 0.125, -1) @ values if s else torch.zeros(n, d, device=DEV, dtype=torch.float64)
                # (a key that rounds to the other side of a bfloat16 step moves a score by 2^-8 of one product: counted with the weights' rounding)
                torch.testing.assert_close(out[row:row + n, h * d:(h + 1) * d].double(), want, rtol=0, atol=1e-5 if dtype == torch.float32 else 3 * 4.5 * 2.0 ** -8)
            first, row = first + s, row + n


# ---- refusals -----------------------------------------------------------------------------------------------------------------------------

def test_refusals_on_the_device(ops):
    case = Case(torch.bfloat16, 8, 2, 64, 16, [1, 4], [20, 30])
    src = ops.Source(case.table, case.lens, 30)
    run = lambda **kw: ops.attention_cross(**{**dict(q=case.q, k_cache=case.k, v_cache=case.v, out=case.out, ctx=case.ctx, source=src, H=8, K=2, d=64, scale=0.1), **kw})  # noqa: E731
    for bad in (dict(q=case.q.float()), dict(k_cache=case.k.float()), dict(K=3), dict(d=32), dict(out=case.out[:, :8]), dict(spans=ints([[0, 1]])), dict(H=0), dict(q=case.q.cpu()),
                dict(source=ops.Source(case.table.long(), case.lens, 30)), dict(source=ops.Source(case.table[:1], case.lens, 30)), dict(k_cache=case.k[:, :, :12], v_cache=case.v[:, :, :12]),
                dict(q=case.q.half(), out=case.out.half(), k_cache=case.k.half(), v_cache=case.v.half()), dict(out=case.q), dict(scale=0.0), dict(scale=1e39), dict(scale=1e-50), dict(scale=float("nan"))):
        with pytest.raises(ops.KernelError):
            run(**bad)
    one = ints([0])
    two = ints([0, 0])
    t = lambda: ints([[1, 2]])  # noqa: E731
    good = dict(before=one, after=ints([5]), table=t(), free=ints([3, 4]), count=ints([2]), page_size=16, left=two, cu_tokens=ints([0, 0]), req_index=ints([0] * 9), positions=ints([0] * 9), slots=ints([0] * 9))
    ops.page_step(**good)
    for bad in (dict(page_size=12), dict(after=ints([1, 2])), dict(before=one.long()), dict(slots=ints([0] * 8)), dict(table=ints([1])), dict(left=one), dict(after=good["before"], left=good["free"]),
                dict(count=good["left"][:1]), dict(cu_tokens=good["before"]), dict(before=one.cpu())):
        with pytest.raises(ops.KernelError):
            ops.page_step(**{**good, **bad})
    rows = torch.zeros(3, 6 * 64, device=DEV, dtype=torch.bfloat16)
    k, v = (torch.zeros(2, 1, 16, 64, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    good = dict(rows=rows, q_out=torch.zeros(3, 256, device=DEV, dtype=torch.bfloat16), q_weight=None, k_weight=None, eps=1e-6, positions=ints([[0, 1, 2]]), axis_of=ints([0] * 32),
                inv_freq=torch.ones(32, device=DEV), rotary_dim=64, interleaved=False, slot_mapping=ints([0, 1, 2]), k_cache=k, v_cache=v, H=4, K=1, d=64)
    ops.qk_norm_axes_write(**good)
    for bad in (dict(rows=rows[:, :300]), dict(H=5), dict(rotary_dim=63), dict(rotary_dim=66), dict(positions=ints([0, 1, 2])), dict(axis_of=ints([0] * 31)), dict(inv_freq=torch.ones(32, device=DEV).double()),
                dict(k_cache=k.float()), dict(slot_mapping=ints([0, 1])), dict(q_out=None), dict(q_weight=torch.ones(63, device=DEV)), dict(v_cache=v[:1]), dict(rows=rows.cpu()), dict(rows=rows.half()),
                dict(slot_mapping=None), dict(k_cache=None), dict(rows=torch.zeros(5, 384, device=DEV, dtype=torch.bfloat16)[:3], q_out=None, H=0, positions=ints([[0, 1]]))):
        with pytest.raises(ops.KernelError):
            ops.qk_norm_axes_write(**{**good, **bad})
    whole = torch.zeros(4 * 384, device=DEV, dtype=torch.bfloat16)
    with pytest.raises(ops.KernelError):
        ops.qk_norm_axes_write(**{**good, "rows": whole[:3 * 384].view(3, 384), "q_out": whole[384:384 + 3 * 256].view(3, 256)})
    assert ops.Source(case.table, case.lens, 1 << 40).longest == 1 << 40
    run(source=ops.Source(case.table, case.lens, 1 << 40))            # (longer than the table's rows: no source is)
    torch.testing.assert_close(case.out.double(), Case.want(_scaled(case, 0.1)), rtol=0, atol=2 * 4.5 * 2.0 ** -8)


def _scaled(case, scale):
    case.scale = scale
    return case


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 20])
def test_axes_where_they_lie(ops, dtype, d):
    """Queries finished in place, as elsewhere."""
    g = torch.Generator(device=DEV).manual_seed(2)
    rows = torch.randn(700, 4 * d, generator=g, device=DEV).to(dtype)
    out, positions = torch.empty_like(rows), torch.arange(1400, device=DEV, dtype=torch.int32).view(2, 700)
    run = lambda to: ops.qk_norm_axes_write(rows, to, torch.ones(d, device=DEV), None, 1e-6, positions, ints([0, 1] * (d // 4)), torch.ones(d // 2, device=DEV), d, False, None, None, None,  # noqa: E731
                                            4, 0, d, write_kv=False)
    run(out)
    run(rows)
    assert torch.equal(rows, out)
