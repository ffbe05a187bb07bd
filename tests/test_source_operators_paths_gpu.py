"""The operators of a decoder that reads an encoder's states, on the paths that only longer or larger calls take; against the same definitions in 64 bits and
with the same tolerances as in ``test_source_operators_gpu.py``.
"""
import random

import pytest
import torch

from test_source_operators_gpu import DEV, DTYPES, Case, axes_want, ints, spread_spans

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from marin_b200.kernels import ops as o
    return o


def most_of(values):
    return max([float(v.abs().max()) for v in values if v.numel()] or [1.0])


def axes_tolerance(dtype):
    return dict(rtol=2.0 ** -21, atol=2.0 ** -19) if dtype == torch.float32 else dict(rtol=2.0 ** -8, atol=2.0 ** -17)


def climbing(dtype, new, src, step):
    """Scores that move by `step` (a power of two) from every 64 positions to the next: the maximum moves with every block of keys, or never does."""
    case = Case(dtype, 8, 2, 64, 16, new, src, seed=len(src))
    case.q[:, :] = 1.0
    for r, s in enumerate(src):
        at = torch.arange(s, device=DEV)
        case.keys[r] = (0.125 * torch.randn(s, 2, 64, device=DEV, generator=torch.Generator(device=DEV).manual_seed(r)) + step / 8 * (at // 64)[:, None, None]).to(dtype).double()
        for j in range(-(-s // 16)):
            rows = case.keys[r][16 * j:16 * j + 16]
            case.k[int(case.table[r, j]), :, :rows.shape[0]] = rows.to(dtype).transpose(0, 1)
    return case


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("step", [8.0, -8.0, 0.0])
def test_cross_scores_that_move_with_every_block(ops, dtype, step):
    """Portions of one to fourteen blocks of keys, cut over a cluster (one request) and not (many): every product of weights and values is waited for, whether or not what
    is added up has to be scaled in between.  A score is a sum of 64 terms and ends at 8 * 13 at most: its additions (33 one after the other, in pairs) are off by 2^-24 of what
    they have by then, half of that on average, 33 * 52 * 2^-24 = 1.1e-4 in all, and a product and the exponent's own rounding add 2e-5.  Weights that are off by 1.3e-4 of
    themselves move a mean of values by twice that times the largest value.  bfloat16 adds the rounding of weights and results, 2^-8 each."""
    for src in ([64], [129], [190], [257], [320], [835]):
        for many in (1, 40):
            case = climbing(dtype, [33] * many, src * many, step)
            first = case.run(ops).clone()
            atol = most_of(case.values) * (2 * 1.3e-4 + (0 if dtype == torch.float32 else 2 * 2.0 ** -8))
            torch.testing.assert_close(first.double(), case.want(), rtol=0, atol=atol)
            case.out.zero_()
            assert torch.equal(case.run(ops), first)
    ops.check_device_errors()


def put(case, r, j, value, columns=slice(None)):
    """Position j of request r has this value (in the columns named), for every head."""
    case.v[int(case.table[r, j // case.page]), :, j % case.page, columns] = value
    case.values[r][j, :, columns] = value


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,K,d,page", [(8, 2, 64, 16), (32, 8, 128, 16), (4, 2, 20, 4), (3, 3, 7, 1), (4, 1, 200, 16), (2, 1, 256, 16), (40, 5, 48, 32)])
@pytest.mark.parametrize("many", [1, 24])
def test_cross_values_that_are_not_finite_concern_who_sees_them(ops, dtype, H, K, d, page, many):
    """Infinities and NaN in values that some rows of a tile see, or all of them, or none: the rows that see them have them (in their columns), the others are as if they were
    not there.  Spans begin and end at the value's place and beside it; cut over a cluster and not."""
    src, at = 300, [70, 71, 200]
    edges = [(0, 300), (0, 70), (0, 71), (70, 71), (71, 72), (71, 200), (72, 200), (72, 201), (200, 201), (201, 300), (5, 5), (64, 128), (128, 192), (0, 1)]
    new = [1, len(edges)] + [9] * many
    spans = [(72, 200)] + edges + [edges[i % len(edges)] for i in range(9 * many)]
    case = Case(dtype, H, K, d, page, new, [src] * len(new), spans, seed=d)
    clean = [v.clone() for v in case.values]
    for r in range(len(new)):
        put(case, r, at[0], float("nan"), slice(0, d // 2))
        put(case, r, at[1], float("inf"), slice(d // 2, d // 2 + 1))
        put(case, r, at[2], float("-inf"), slice(d - 2, d))
    got, want = case.run(ops).double().view(-1, H, d), torch.empty(sum(new), H, d, device=DEV, dtype=torch.float64)
    row, odd = 0, case.values
    case.values = clean
    want[:] = case.want().view(-1, H, d)
    for r, n in enumerate(new):
        for lo, hi in spans[row:row + n]:
            for j in at:                                             # (a weight is positive: what is seen is there)
                if lo <= j < hi:
                    seen = odd[r][j].repeat_interleave(H // K, 0)
                    want[row] = torch.where(seen.isfinite(), want[row], want[row] + seen)
            row += 1
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isposinf(), want.isposinf()) and torch.equal(got.isneginf(), want.isneginf())
    finite = want.isfinite()
    torch.testing.assert_close(got[finite], want[finite], rtol=0, atol=4e-6 if dtype == torch.float32 else 2 * most_of(clean) * 2.0 ** -8)
    ops.check_device_errors()


@pytest.mark.parametrize("dtype,new", [(torch.bfloat16, 512), (torch.float32, 64)])
def test_cross_price_of_a_value_that_is_not_finite(ops, dtype, new):
    """A value (or a key) that is not finite does not hold up the step: where every row sees it nothing is worked out again; where some rows do not, theirs are, in one pass.
    Bounds: reading a tile's values once more is less work than the call itself (a factor of 30 for the small launches here); the rows' own pass over 1,000 positions
    is 100 instructions or so a row and position in a warp, at 4 warps an SM and one instruction in four cycles 512 * 32 * 1000 * 100 * 4 / (148 * 4) cycles, below 10 ms."""
    spans = [(0, 2000) if t % 2 else (0, 1000) for t in range(new)]
    case = Case(dtype, 32, 8, 128, 16, [new], [2000], spans, seed=3)

    def milliseconds():
        case.run(ops)
        best = float("inf")
        for _ in range(5):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            begin.record()
            case.run(ops)
            end.record()
            end.synchronize()
            best = min(best, begin.elapsed_time(end))
        return best

    usual = milliseconds()
    page, at = int(case.table[0, 500 // 16]), 500 % 16
    case.v[page, :, at] = float("nan")                               # (all see it)
    seen_by_all = milliseconds()
    assert case.out.isnan().all()
    case.v[page, :, at] = 0.5
    case.k[page, :, at] = float("nan")
    key = milliseconds()
    assert case.out.isnan().all()
    case.k[page, :, at] = 0.5
    case.v[int(case.table[0, 1500 // 16]), :, 1500 % 16] = float("inf")
    seen_by_half = milliseconds()
    assert case.out[1::2].isposinf().all() and case.out[::2].isfinite().all()
    print(f"{new} tokens: {usual:.3f} ms, a value that all see {seen_by_all:.3f}, a key {key:.3f}, a value that half of the rows see {seen_by_half:.3f}")
    assert key <= 2 * usual + 0.2 and seen_by_all <= 30 * usual + 0.2 and seen_by_half <= 10.0


def places(case):
    """How the blocks of the portions' launch find their tiles: "longest" (requests), "sources" (the longest first), or "rows" (a search), by the rule beside the kernels."""
    nd, G, f32 = case.ctx.num_decode, case.H // case.K, case.q.dtype == torch.float32
    requests, T = case.ctx.num_requests - nd, case.q.shape[0]
    rows = case.ctx.max_query_len * G
    a_token, size = (G, 4 if rows <= 4 else 8 if rows <= 8 else 16 if rows <= 16 else 32) if f32 else (1, 128 // G)
    padded, filled = -(-case.ctx.max_query_len * a_token // size) * requests, requests + T * a_token // size
    if 1 < requests <= 32 and min(padded, filled) * case.K > 296:
        return "sources"
    return "longest" if padded <= filled + filled // 4 else "rows"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("portions", [2, 7, 31, 32, 33])
@pytest.mark.parametrize("ahead", [0, 3])
def test_cross_longest_sources_first(ops, dtype, portions, ahead):
    """Two to 32 portions with more tiles than places for blocks: every tile of every request once, whatever the order of their sources; single tokens ahead, requests without a
    token in between, tokens behind the last request.  (33 portions: the other side of the rule.)"""
    rng = random.Random(portions)
    new = [rng.choice([150, 257, 300]) if portions > 7 else 700 + 61 * i for i in range(portions)]
    sources = {"unlike": [rng.choice([0, 1, 17, 64, 100, 333]) for _ in new], "alike": [90] * portions, "falling": [10 * (portions - i) for i in range(portions)],
               "two lengths": [(40, 200)[i % 2] for i in range(portions)]}
    for name, src in sources.items():
        there = list(new)
        if name in ("unlike", "two lengths") and portions > 2:
            there[1] = there[portions // 2] = 0
        counts, lens = [1] * ahead + there, [50, 0, 130][:ahead] + src
        for spans in (None, spread_spans(counts, lens, portions)):
            case = Case(dtype, 32, 32, 16, 16, counts, lens, spans, seed=portions, pad_rows=5)
            assert (places(case) == "sources") == (portions <= 32)
            case.check(ops)
    case = Case(dtype, 16, 4, 64, 16, [1] * ahead + [x + 640 for x in new], [50, 0, 130][:ahead] + sources["unlike"], seed=portions, pad_rows=3)
    assert (places(case) == "sources") == (portions <= 32)
    case.check(ops)
    ops.check_device_errors()


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("R,K,chunks,sources", [(64, 8, 1, (2047, 2048, 2049, 4100, 6200)), (130, 4, 1, (2047, 2048, 2049, 4100)), (50, 6, 2, (4000, 4097, 4300, 5000)),
                                                (37, 5, 4, (8193, 8300, 40)), (2, 2, 8, (17001, 18432))])
def test_cross_single_tokens_over_long_sources(ops, page, R, K, chunks, sources):
    """Runs of more than 32 stages of 16 positions a warp: where a warp's pages are looked up again.  One to eight blocks a request and kv head; spans that begin inside a stage."""
    src = [sources[i % len(sources)] for i in range(R)]
    assert ops.cross_decode_chunks(R * K, max(src)) == chunks and max(src) > 32 * 64 * chunks
    Case(torch.bfloat16, 2 * K, K, 16, page, [1] * R, src, seed=R).check(ops)
    spans = [[(5, s), (s // 3 + 7, s - 9), (0, s), (s - 2050, s + 10), (100, 2148 + i)][i % 5] for i, s in enumerate(src)]
    Case(torch.bfloat16, 2 * K, K, 16, page, [1] * R, src, spans, seed=R + 1, pad_rows=1).check(ops)


# ---- heads with positions of several axes ----------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("stride", [3, 4 * 64 + 24])
def test_axes_single_row_in_place(ops, dtype, stride):
    """A single token's queries finished where they lie: the row's stride says nothing, whether it is cut out of a wider row or made up."""
    g = torch.Generator(device=DEV).manual_seed(5)
    rows = torch.as_strided(torch.randn(4 * 64 + 24, generator=g, device=DEV).to(dtype), (1, 4 * 64), (stride, 1))
    weight, positions, axis_of, inv_freq = 1 + 0.2 * torch.randn(64, generator=g, device=DEV), ints([[70], [5]]), ints([0, 1] * 16), torch.rand(32, generator=g, device=DEV)
    want, _, _ = axes_want(rows, weight, None, 1e-6, positions, axis_of, inv_freq, 64, False, 4, 0, 64)
    ops.qk_norm_axes_write(rows, rows, weight, None, 1e-6, positions, axis_of, inv_freq, 64, False, None, None, None, 4, 0, 64, write_kv=False)
    torch.testing.assert_close(rows.double(), want.reshape(1, -1), **axes_tolerance(dtype))


LONG_AXES = [(32, 8, 128, 128, 16, 8007), (32, 8, 128, 128, 16, 2501), (16, 16, 80, 80, 16, 2501), (40, 8, 128, 64, 32, 1000), (96, 8, 128, 128, 16, 1501), (0, 1, 512, 512, 16, 1000),
             (0, 1, 256, 256, 16, 1000), (14, 2, 96, 96, 64, 2501), (4, 2, 40, 20, 4, 1000), (1, 1, 24, 16, 16, 2501)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("H,K,d,rotary,page,T", LONG_AXES)
def test_axes_many_tokens(ops, dtype, interleaved, H, K, d, rotary, page, T):
    """Prompts of which every block takes several tokens, one after the other: rows that are on their way ahead, angles and places of groups of tokens in two buffers, a last group and a
    last block that are not full; one part of the heads and several, fewer threads than a head has angles."""
    for axes, norm, wide in ((3, True, 0), (1, False, 8)):
        g = torch.Generator(device=DEV).manual_seed(T + axes)
        half = rotary // 2
        rows = torch.randn(T, (H + 2 * K) * d + wide, generator=g, device=DEV).to(dtype)[:, :(H + 2 * K) * d]
        qw, kw = ((1 + 0.3 * torch.randn(d, generator=g, device=DEV)) if norm else None for _ in range(2))
        axis_of = torch.randint(0, axes, (half,), generator=g, device=DEV).int()
        inv_freq = torch.pow(10000.0, -2.0 * torch.arange(half, device=DEV) / rotary).float()
        positions = torch.randint(0, 50000, (axes, T), generator=g, device=DEV).int()
        pages = -(-T // page) + 2
        slots = torch.randperm(pages * page, generator=g, device=DEV)[:T].int()
        slots[torch.randperm(T, generator=g, device=DEV)[:T // 7]] = -1                     # padded tokens inside the runs
        slots[T // 2] = pages * page                                                          # no place of the cache
        k, v = (torch.full((pages, K, page, d), 9.0, device=DEV, dtype=dtype) for _ in range(2))
        q_out = torch.empty(T, H * d, device=DEV, dtype=dtype) if H else None
        ops.qk_norm_axes_write(rows, q_out, qw, kw, 1e-6, positions, axis_of, inv_freq, rotary, interleaved, slots, k, v, H, K, d)
        q_want, k_want, v_want = axes_want(rows, qw, kw, 1e-6, positions, axis_of, inv_freq, rotary, interleaved, H, K, d)
        k_ref, v_ref = (torch.full((pages, K, page, d), 9.0, device=DEV, dtype=torch.float64) for _ in range(2))
        stored = (slots >= 0) & (slots < pages * page)
        at = slots[stored].long()
        k_ref[at // page, :, at % page], v_ref[at // page, :, at % page] = k_want[stored], v_want[stored]
        if H:
            torch.testing.assert_close(q_out.double(), q_want.reshape(T, H * d), **axes_tolerance(dtype))
        torch.testing.assert_close(k.double(), k_ref, **axes_tolerance(dtype))
        assert torch.equal(v.double(), v_ref)
        if H:                                                        # queries alone, where they lie
            lie = rows[:, :H * d].contiguous()
            ops.qk_norm_axes_write(lie, lie, qw, None, 1e-6, positions, axis_of, inv_freq, rotary, interleaved, None, None, None, H, 0, d, write_kv=False)
            assert torch.equal(lie, q_out)
