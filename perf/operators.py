"""Operators of a decoder that reads an encoder's states beside its own cache, as cases that can be timed: what the framework's
kernels compute, in elementary torch operations (``own`` False) and through the framework's entry points (``own`` True).

Kinds of case (``op``):

``cross``   attention of a step's tokens to an encoder's states (``ops.attention_cross``): keys and values of another length than the
            queries, in pages, every token sees all of its request's states or, with ``spans``, a run of them (text that stands behind one
            of several images sees that image; text before the first sees none and gets zeros).  Single tokens (decode) and portions.
``axes``    norms, rotation by positions of several axes (time, height, width) and the write into the paged cache
            (``ops.qk_norm_axes_write``): every pair of a head turns by the position of the axis that it belongs to.
``pages``   a step's bookkeeping on the device (``ops.page_step``): from the requests' lengths before and after it, pages taken from
            and given back to a free list, block tables, and every new token's request, position and place in the cache.

Sizes: the heads of the Qwen3-4B/8B/14B layouts (32, 32 and 40 over 8 of 128) and smaller ones of the tests, pages of 16 to 64.
"""
import math
import random
from types import SimpleNamespace

import torch

own = False

EPS = 1e-6
THETA = 1000000.0
#: columns of a page_step's table that a request's longest sequence needs besides what the case says
SPARE_PAGES = 5


def listed():
    return [
        # one user's next token over the states of one image: the smallest call, bound by latency
        {"name": "cross decode one", "op": "cross", "dtype": "bf16", "H": 32, "K": 8, "d": 128, "page": 16, "requests": 1, "new_lo": 1, "new_hi": 1,
         "src_lo": 577, "src_hi": 577, "spans": False, "lens": 1},
        # a server's decode step: 64 users, sources of all lengths; bound by the cache's bytes
        {"name": "cross decode 64", "op": "cross", "dtype": "bf16", "H": 32, "K": 8, "d": 128, "page": 16, "requests": 64, "new_lo": 1, "new_hi": 1,
         "src_lo": 500, "src_hi": 4100, "spans": False, "lens": 2},
        # whole prompts over long sources: the largest call, bound by the tensor cores
        {"name": "cross prompt long", "op": "cross", "dtype": "bf16", "H": 32, "K": 8, "d": 128, "page": 16, "requests": 4, "new_lo": 1024, "new_hi": 1024,
         "src_lo": 4096, "src_hi": 4096, "spans": False, "lens": 3},
        # prompts of odd lengths whose text stands between images (five query heads a kv head), some requests without any source
        {"name": "cross prompt spans", "op": "cross", "dtype": "bf16", "H": 40, "K": 8, "d": 128, "page": 32, "requests": 6, "new_lo": 17, "new_hi": 700,
         "src_lo": 0, "src_hi": 2500, "spans": True, "lens": 4},
        # short portions over a long recording: few rows, a long axis to split
        {"name": "cross portion long source", "op": "cross", "dtype": "bf16", "H": 16, "K": 8, "d": 64, "page": 64, "requests": 2, "new_lo": 9, "new_hi": 40,
         "src_lo": 16000, "src_hi": 20000, "spans": False, "lens": 5},
        # the 32-bit mode: a few requests of a small encoder-decoder, prompt portions and single tokens together
        {"name": "cross 32 bits", "op": "cross", "dtype": "f32", "H": 16, "K": 16, "d": 64, "page": 16, "requests": 5, "new_lo": 1, "new_hi": 150,
         "src_lo": 200, "src_hi": 900, "spans": False, "lens": 6},
        # a decode step's heads: eight tokens, three axes in sections
        {"name": "axes decode 8", "op": "axes", "dtype": "bf16", "H": 32, "K": 8, "d": 128, "page": 16, "tokens": 8, "padded": 0, "axes": 3, "spread": False,
         "rotary": 128, "interleaved": False, "norm": True, "first": 4000, "lens": 1},
        # long prompts with images among the text: bound by the bytes of the heads
        {"name": "axes prompt 8000", "op": "axes", "dtype": "bf16", "H": 32, "K": 8, "d": 128, "page": 16, "tokens": 8000, "padded": 7, "axes": 3, "spread": True,
         "rotary": 128, "interleaved": False, "norm": True, "first": 100000, "lens": 2},
        # an image encoder's heads in 32 bits: height and width, pairs side by side, no norm
        {"name": "axes image 32 bits", "op": "axes", "dtype": "f32", "H": 16, "K": 16, "d": 80, "page": 16, "tokens": 2501, "padded": 0, "axes": 2, "spread": False,
         "rotary": 80, "interleaved": True, "norm": False, "first": 0, "lens": 3},
        # a decode step of eight requests: latency alone
        {"name": "pages decode 8", "op": "pages", "requests": 8, "page": 16, "prompts": 0, "new_hi": 1, "have_hi": 4000, "ended": 1, "spare": 40, "lens": 1},
        # a mixed step: decodes, prompt portions, requests that ended
        {"name": "pages mixed 256", "op": "pages", "requests": 256, "page": 16, "prompts": 24, "new_hi": 600, "have_hi": 4000, "ended": 20, "spare": 1000, "lens": 2},
        # the largest: thousands of requests, a hundred thousand new tokens
        {"name": "pages many 4000", "op": "pages", "requests": 4000, "page": 32, "prompts": 400, "new_hi": 500, "have_hi": 2000, "ended": 150, "spare": 9000, "lens": 3},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["cross", "cross", "axes", "pages"])
    lens = rng.randrange(1 << 30)
    if op == "cross":
        dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
        H, K = rng.choice([(32, 8), (40, 8), (16, 8), (32, 4), (8, 8), (12, 4), (14, 2)])
        d = rng.choice([128, 128, 64, 80, 96])
        page = rng.choice([16, 32, 64])
        if rng.random() < 0.4:                                      # a decode step
            requests, src = _log(rng, 1, 64), _log(rng, 1, 4096)
            return {"op": op, "dtype": dtype, "H": H, "K": K, "d": d, "page": page, "requests": requests, "new_lo": 1, "new_hi": 1,
                    "src_lo": rng.choice([0, max(1, src // 8), src]), "src_hi": src, "spans": rng.random() < 0.25, "lens": lens}
        requests, new = _log(rng, 1, 4), _log(rng, 2, 700 if dtype == "bf16" else 300)
        src = _log(rng, 1, 4096 if new > 64 else 16000)
        return {"op": op, "dtype": dtype, "H": H, "K": K, "d": d, "page": page, "requests": requests, "new_lo": rng.choice([1, max(1, new // 4), new]), "new_hi": new,
                "src_lo": rng.choice([0, max(1, src // 8), src]), "src_hi": src, "spans": rng.random() < 0.4, "lens": lens}
    if op == "axes":
        dtype = rng.choice(["bf16", "bf16", "f32"])
        H, K = rng.choice([(32, 8), (40, 8), (16, 8), (16, 16), (14, 2), (5, 1)])
        d = rng.choice([128, 64, 80, 96])
        return {"op": op, "dtype": dtype, "H": H, "K": K, "d": d, "page": rng.choice([16, 32, 64]), "tokens": _log(rng, 1, 8000 if dtype == "bf16" else 2500),
                "padded": rng.choice([0, 0, 3, 16]), "axes": rng.choice([1, 2, 3]), "spread": rng.random() < 0.5, "rotary": rng.choice([d, d, d // 2]),
                "interleaved": rng.random() < 0.3, "norm": rng.random() < 0.6, "first": rng.choice([0, 1000, 300000]), "lens": lens}
    requests = _log(rng, 1, 3500)
    return {"op": op, "requests": requests, "page": rng.choice([16, 32, 64]), "prompts": rng.randrange(0, requests // 10 + 2), "new_hi": _log(rng, 1, 500),
            "have_hi": _log(rng, 20, 2000), "ended": rng.randrange(0, requests // 20 + 2), "spare": rng.choice([0, 200, 8000]), "lens": lens}


# ---- what a case's name stands for: lengths, from its own numbers alone ------------------------------------------------------

def _cross_lengths(case):
    """New tokens and source length of every request; requests of one token come first, as a step has them."""
    rng = random.Random(case["lens"])
    new = sorted((rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["requests"])), key=lambda n: n != 1)
    src = [rng.randint(case["src_lo"], case["src_hi"]) for _ in range(case["requests"])]
    if case["spans"] and case["src_lo"] == 0 and case["requests"] > 1:
        src[-1] = 0                                                 # a request without any source
    return new, src


IMAGES = 3


def _span(t, new, src):
    """The run of states that token t of `new` sees: the first of its portion's quarters none, each of the others one of three images."""
    part = min(IMAGES, (t * (IMAGES + 1)) // max(1, new)) if new > 1 else IMAGES
    return (0, 0) if part == 0 else (src * (part - 1) // IMAGES, src * part // IMAGES)


def _cross_spans(case):
    new, src = _cross_lengths(case)
    return [_span(t, n, s) if case["spans"] else (0, s) for n, s in zip(new, src) for t in range(n)]


def _page_lengths(case):
    """Lengths before and after the step: the first `prompts` requests bring a portion, the last `ended` give their pages back, one token each between."""
    rng = random.Random(case["lens"])
    n, ended = case["requests"], min(case["ended"], max(0, case["requests"] - 1))
    prompts = min(case["prompts"], n - ended)
    before = [rng.randint(0, case["have_hi"]) if r < prompts else rng.randint(1, case["have_hi"]) for r in range(n)]
    after = [b + rng.randint(1, case["new_hi"]) if r < prompts else (b + 1 if r < n - ended else rng.choice([0, 0, b // 2])) for r, b in enumerate(before)]
    order = list(range(n))
    rng.shuffle(order)
    return [before[i] for i in order], [after[i] for i in order]


def _pages_of(tokens, page):
    return -(-tokens // page)


def _dtype(case):
    return torch.bfloat16 if case.get("dtype") == "bf16" else torch.float32


def work(case):
    if case["op"] == "cross":
        new, src = _cross_lengths(case)
        spans = _cross_spans(case)
        starts = [sum(new[:r]) for r in range(len(new) + 1)]
        seen = [spans[a:b] for a, b in zip(starts, starts[1:])]
        keys = sum(max(hi for _, hi in s) - min([lo for lo, hi in s if hi > lo], default=0) for s in seen)
        size = 2 if case["dtype"] == "bf16" else 4
        pairs = sum(hi - lo for lo, hi in spans)
        return {"bytes": size * (2 * sum(new) * case["H"] * case["d"] + 2 * keys * case["K"] * case["d"]) + 4 * sum(_pages_of(s, case["page"]) for s in src),
                "flops": 4 * pairs * case["H"] * case["d"]}
    if case["op"] == "axes":
        T, size = case["tokens"], 2 if case["dtype"] == "bf16" else 4
        heads = case["H"] + 2 * case["K"]
        return {"bytes": (T + case["padded"]) * (2 * heads * case["d"] * size + 4 * case["axes"] + 4), "flops": 8 * T * heads * case["d"]}
    before, after = _page_lengths(case)
    tokens = sum(max(0, a - b) for a, b in zip(after, before))
    moved = sum(abs(_pages_of(a, case["page"]) - _pages_of(b, case["page"])) for a, b in zip(after, before))
    return {"bytes": 4 * (2 * len(before) + len(before) + 1 + 3 * tokens + 2 * moved), "flops": 8 * (tokens + len(before))}


# ---- inputs ---------------------------------------------------------------------------------------------------------------------

def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    host = random.Random(seed)
    if case["op"] == "cross":
        new, src = _cross_lengths(case)
        dt, H, K, d, page = _dtype(case), case["H"], case["K"], case["d"], case["page"]
        T, R = sum(new), len(new)
        counts = [_pages_of(s, page) for s in src]
        widest = max(1, max(counts))
        pool = torch.randperm(sum(counts) + 3, generator=g, device="cuda").to(torch.int32)            # pages lie anywhere in the pool
        starts = [sum(counts[:r]) for r in range(R)]
        at = torch.tensor(starts, device="cuda")[:, None] + torch.arange(widest, device="cuda")[None, :]
        mine = torch.arange(widest, device="cuda")[None, :] < torch.tensor(counts, device="cuda")[:, None]
        table = torch.where(mine, pool[at.clamp(max=pool.numel() - 1)], torch.zeros_like(pool[:1]))
        cu = [sum(new[:r]) for r in range(R + 1)]
        ctx = SimpleNamespace(num_tokens=T, num_requests=R, num_decode=sum(n == 1 for n in new), max_query_len=max(new), cu_tokens=_ints(cu),
                              req_index=_ints([r for r, n in enumerate(new) for _ in range(n)]))
        source = SimpleNamespace(block_table=table.contiguous(), lens=_ints(src), longest=max(src))
        q = torch.randn(T, H * d, generator=g, device="cuda").to(dt)
        k = torch.randn(pool.numel(), K, page, d, generator=g, device="cuda").to(dt)
        v = torch.randn(pool.numel(), K, page, d, generator=g, device="cuda").to(dt)
        return {"op": "cross", "q": q, "k": k, "v": v, "out": torch.zeros_like(q), "ctx": ctx, "source": source, "H": H, "K": K, "d": d, "scale": 1.0 / math.sqrt(d),
                "spans": _ints(_cross_spans(case)) if case["spans"] else None}
    if case["op"] == "axes":
        dt, H, K, d, page = _dtype(case), case["H"], case["K"], case["d"], case["page"]
        T, rotary, axes = case["tokens"] + case["padded"], case["rotary"], case["axes"]
        half = rotary // 2
        i = torch.arange(half, device="cuda")
        # sections: the first pairs turn with time, the next with height, the last with width; spread: the axes in turn
        axis_of = (i % axes if case["spread"] else i * axes // half).to(torch.int32)
        inv_freq = torch.pow(torch.tensor(THETA, dtype=torch.float64, device="cuda"), -2.0 * i.double() / rotary).float()
        t = torch.arange(T, device="cuda")
        # images of 16 by 16 among the text: time stands still over an image, height and width run
        grid = torch.stack([t // 256 * 16, t // 256 * 16 + t // 16 % 16, t // 256 * 16 + t % 16])[:axes]
        positions = (grid + case["first"] + host.randrange(1000)).to(torch.int32).contiguous()
        pages = _pages_of(case["tokens"], page) + 2
        order = torch.randperm(pages * page, generator=g, device="cuda")[:case["tokens"]].to(torch.int32)
        slots = torch.cat([order, torch.full((case["padded"],), -1, dtype=torch.int32, device="cuda")])
        weights = [(1.0 + 0.2 * torch.randn(d, generator=g, device="cuda")) if case["norm"] else None for _ in range(2)]
        return {"op": "axes", "rows": torch.randn(T, (H + 2 * K) * d, generator=g, device="cuda").to(dt), "q_out": torch.empty(T, H * d, device="cuda", dtype=dt),
                "q_weight": weights[0], "k_weight": weights[1], "positions": positions, "axis_of": axis_of, "inv_freq": inv_freq, "rotary": rotary,
                "interleaved": case["interleaved"], "slots": slots, "stored": case["tokens"], "k": torch.zeros(pages, K, page, d, device="cuda", dtype=dt),
                "v": torch.zeros(pages, K, page, d, device="cuda", dtype=dt), "H": H, "K": K, "d": d}
    before, after = _page_lengths(case)
    page = case["page"]
    held = [_pages_of(b, page) for b in before]
    needs = sum(max(0, _pages_of(a, page) - h) for a, h in zip(after, held))
    back = sum(max(0, h - _pages_of(a, page)) for a, h in zip(after, held))
    count = max(0, needs - back) + case["spare"]
    tokens = sum(max(0, a - b) for a, b in zip(after, before))
    columns = max(_pages_of(max(a, b), page) for a, b in zip(after, before)) + SPARE_PAGES
    pool = torch.randperm(sum(held) + count, generator=g, device="cuda").to(torch.int32)
    starts = torch.tensor(held, device="cuda").cumsum(0) - torch.tensor(held, device="cuda")
    at = starts[:, None] + torch.arange(columns, device="cuda")[None, :]
    mine = torch.arange(columns, device="cuda")[None, :] < torch.tensor(held, device="cuda")[:, None]
    table = torch.where(mine, pool[at.clamp(max=pool.numel() - 1)], torch.full_like(pool[:1], -1)).contiguous()
    free = torch.full((pool.numel(),), -1, dtype=torch.int32, device="cuda")
    free[:count] = pool[sum(held):]
    room = tokens + 5                                                # what a step's buffers hold is more than its tokens
    buffers = {n: torch.empty(s, dtype=torch.int32, device="cuda") for n, s in (("left", 2), ("cu", len(before) + 1), ("req", room), ("pos", room), ("slots", room))}
    return {"op": "pages", "before": _ints(before), "after": _ints(after), "table": table, "free": free, "count": _ints([count]), "page": page, **buffers}


# ---- the operators ------------------------------------------------------------------------------------------------------------

def _cross_plain(s):
    ctx, source, H, K, d = s["ctx"], s["source"], s["H"], s["K"], s["d"]
    page, R, L, S, T = s["k"].shape[2], ctx.num_requests, ctx.max_query_len, max(1, source.longest), ctx.num_tokens
    key = torch.arange(S, device="cuda")
    place = source.block_table[:, key // page].long()                               # [R, S]
    k = s["k"][place, :, key % page].float().permute(0, 2, 1, 3)                    # [R, K, S, d]
    v = s["v"][place, :, key % page].float().permute(0, 2, 1, 3)
    there = key[None, :] < source.lens[:, None]                                     # [R, S]
    v = torch.where(there[:, None, :, None], v, 0.0)
    token = (ctx.cu_tokens[:-1, None] + torch.arange(L, device="cuda")[None, :]).clamp(max=T - 1).long()      # [R, L]
    q = s["q"].view(T, H, d)[token].float().view(R, L, K, H // K, d).permute(0, 2, 3, 1, 4).reshape(R, K, H // K * L, d)
    scores = (q @ k.transpose(2, 3) * s["scale"]).view(R, K, H // K, L, S)
    seen = there[:, None, :]
    if s["spans"] is not None:
        lo, hi = s["spans"][:, 0][token], s["spans"][:, 1][token]
        seen = seen & (key >= lo[:, :, None]) & (key < hi[:, :, None])              # [R, L, S]
    scores = torch.where(seen[:, None, None], scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = (p.view(R, K, H // K * L, S) @ v).view(R, K, H // K, L, d) / torch.where(total == 0, 1.0, total)
    r = ctx.req_index.long()
    rows = o.permute(0, 3, 1, 2, 4).reshape(R, L, H * d)[r, torch.arange(T, device="cuda") - ctx.cu_tokens[r]]
    s["out"].copy_(rows)
    return s["out"]


def _axes_plain(s):
    H, K, d, half, n = s["H"], s["K"], s["d"], s["rotary"] // 2, s["stored"]
    T, page = s["rows"].shape[0], s["k"].shape[2]
    x = s["rows"].float().view(T, H + 2 * K, d)
    angle = s["positions"][s["axis_of"].long()].double().t() * s["inv_freq"].double()           # [T, half]: far positions need 64 bits
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def turned(part, weight):
        if weight is not None:
            part = part / torch.sqrt(part.square().mean(-1, keepdim=True) + EPS) * weight
        pair = (part[..., 0:2 * half:2], part[..., 1:2 * half:2]) if s["interleaved"] else (part[..., :half], part[..., half:2 * half])
        a, b = pair[0] * cos - pair[1] * sin, pair[1] * cos + pair[0] * sin
        whole = torch.stack([a, b], -1).flatten(-2) if s["interleaved"] else torch.cat([a, b], -1)
        return torch.cat([whole, part[..., 2 * half:]], -1)

    s["q_out"].copy_(turned(x[:, :H], s["q_weight"]).reshape(T, H * d))
    at = s["slots"][:n].long()
    s["k"][at // page, :, at % page] = turned(x[:, H:H + K], s["k_weight"])[:n].to(s["k"].dtype)
    s["v"][at // page, :, at % page] = s["rows"].view(T, H + 2 * K, d)[:n, H + K:]
    return s["q_out"], s["k"], s["v"]


def _pages_plain(s):
    before, after, table, page, R = s["before"], s["after"], s["table"], s["page"], s["before"].numel()
    room, columns, size = s["slots"].numel(), table.shape[1], s["free"].numel()
    held, wants = (before + page - 1) // page, (after + page - 1) // page
    new, taken, back = (after - before).clamp(min=0), (wants - held).clamp(min=0), (held - wants).clamp(min=0)
    upto = [torch.cat([torch.zeros_like(x[:1]), x.cumsum(0).int()]) for x in (new, taken, back)]
    n_new, n_taken, n_back = (u[-1] for u in upto)
    pool = s["count"][0] + n_back
    ok = (n_taken <= pool) & (n_new <= room) & (wants.max() <= columns)
    # the pages given back lie on top of the free list, in the order of requests and positions; pages are taken from its top
    i = torch.arange(size, device="cuda").int()
    k = (i - s["count"][0]).clamp(min=0)
    owner = (torch.searchsorted(upto[2], k, right=True) - 1).clamp(max=R - 1)
    given = table[owner, (wants[owner] + k - upto[2][owner]).clamp(0, columns - 1).long()]
    stack = torch.where((i >= s["count"][0]) & (i < pool), given, s["free"])
    column = torch.arange(columns, device="cuda").int()[None, :]
    fresh = (column >= held[:, None]) & (column < wants[:, None]) & ok
    from_top = upto[1][:-1, None] + column - held[:, None]
    table.copy_(torch.where(fresh, stack[(pool - 1 - from_top).clamp(0, size - 1).long()], table))
    s["free"].copy_(torch.where((i >= s["count"][0]) & (i < pool - n_taken) & ok, stack, s["free"]))
    s["left"].copy_(torch.stack([torch.where(ok, pool - n_taken, s["count"][0]), torch.where(ok, 0, torch.where(wants.max() > columns, 3, torch.where(n_new > room, 2, 1)))]))
    s["cu"].copy_(torch.where(ok, upto[0], 0))
    t = torch.arange(room, device="cuda").int()
    r = (torch.searchsorted(upto[0], t, right=True) - 1).clamp(max=R - 1)
    there = (t < n_new) & ok
    position = before[r] + t - upto[0][r]
    s["req"].copy_(torch.where(there, r, 0))
    s["pos"].copy_(torch.where(there, position, 0))
    s["slots"].copy_(torch.where(there, table[r, (position // page).clamp(0, columns - 1).long()] * page + position % page, -1))
    return table, s["free"], s["left"], s["cu"], s["req"], s["pos"], s["slots"]


def run(s):
    if own:
        from marin_b200.kernels import ops

        if s["op"] == "cross":
            ops.attention_cross(s["q"], s["k"], s["v"], s["out"], s["ctx"], s["source"], s["H"], s["K"], s["d"], s["scale"], s["spans"])
            return s["out"]
        if s["op"] == "axes":
            ops.qk_norm_axes_write(s["rows"], s["q_out"], s["q_weight"], s["k_weight"], EPS, s["positions"], s["axis_of"], s["inv_freq"], s["rotary"], s["interleaved"],
                                   s["slots"], s["k"], s["v"], s["H"], s["K"], s["d"])
            return s["q_out"], s["k"], s["v"]
        ops.page_step(s["before"], s["after"], s["table"], s["free"], s["count"], s["page"], s["left"], s["cu"], s["req"], s["pos"], s["slots"])
        return s["table"], s["free"], s["left"], s["cu"], s["req"], s["pos"], s["slots"]
    if s["op"] == "cross":
        return _cross_plain(s)
    if s["op"] == "axes":
        return _axes_plain(s)
    return _pages_plain(s)


# ---- the definitions in 64 bits, request by request and head by head --------------------------------------------------------

def _cross_exact(case, s):
    new, src = _cross_lengths(case)
    spans = _cross_spans(case)
    H, K, d, page, G = s["H"], s["K"], s["d"], case["page"], s["H"] // s["K"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for r, (n, length) in enumerate(zip(new, src)):
        if length > 0:
            pages = s["source"].block_table[r, :_pages_of(length, page)].long()
            limit = torch.tensor(spans[first:first + n], device="cuda")
            position = torch.arange(length, device="cuda")
            hidden = (position < limit[:, :1]) | (position >= limit[:, 1:])
            for h in range(H):
                keys = s["k"][pages, h // G].reshape(-1, d)[:length].double()
                values = s["v"][pages, h // G].reshape(-1, d)[:length].double()
                scores = (s["q"][first:first + n, h * d:(h + 1) * d].double() @ keys.t()) * s["scale"]
                weights = torch.softmax(scores.masked_fill(hidden, -math.inf), -1).nan_to_num(0.0)
                out[first:first + n, h * d:(h + 1) * d] = weights @ values
        first += n
    return out


def _axes_exact(case, s):
    H, K, d, page, half, T = s["H"], s["K"], s["d"], case["page"], s["rotary"] // 2, s["rows"].shape[0]
    heads = s["rows"].double().view(T, H + 2 * K, d)
    done = heads.clone()
    for h in range(H + K):
        x = heads[:, h]
        weight = s["q_weight"] if h < H else s["k_weight"]
        if weight is not None:
            x = x * torch.rsqrt(x.pow(2).sum(-1, keepdim=True) / d + EPS) * weight.double()
        y = x.clone()
        for i in range(half):
            turn = s["positions"][int(s["axis_of"][i])].double() * s["inv_freq"][i].double()
            a, b = (2 * i, 2 * i + 1) if s["interleaved"] else (i, half + i)
            y[:, a] = x[:, a] * turn.cos() - x[:, b] * turn.sin()
            y[:, b] = x[:, b] * turn.cos() + x[:, a] * turn.sin()
        done[:, h] = y
    k, v = (torch.zeros(s["k"].shape, dtype=torch.float64, device="cuda") for _ in range(2))
    slots = s["slots"][:case["tokens"]].long()
    k[slots // page, :, slots % page] = done[:case["tokens"], H:H + K]
    v[slots // page, :, slots % page] = done[:case["tokens"], H + K:]
    return done[:, :H].reshape(T, H * d), k, v


def _pages_exact(case, s):
    before, after = _page_lengths(case)
    page, room, columns = case["page"], s["slots"].numel(), s["table"].shape[1]
    table, free, count = s["table"].tolist(), s["free"].tolist(), int(s["count"])
    stack = free[:count]
    for row, b, a in zip(table, before, after):
        stack += row[_pages_of(a, page):_pages_of(b, page)]
    cu, req, pos, slots = [0], [], [], []
    for r, (row, b, a) in enumerate(zip(table, before, after)):
        for column in range(_pages_of(b, page), _pages_of(a, page)):
            row[column] = stack.pop()
        for p in range(b, a):
            req.append(r)
            pos.append(p)
            slots.append(row[p // page] * page + p % page)
        cu.append(len(req))
    for i in range(count, len(stack)):
        free[i] = stack[i]
    pad = room - len(req)
    return tuple(torch.tensor(x, dtype=torch.int32, device="cuda").view(-1, columns) if x is table else torch.tensor(x, dtype=torch.int32, device="cuda")
                 for x in (table, free, [len(stack), 0], cu, req + [0] * pad, pos + [0] * pad, slots + [-1] * pad))


def exact(case, seed):
    s = prepare(case, seed)
    return {"cross": _cross_exact, "axes": _axes_exact, "pages": _pages_exact}[case["op"]](case, s)
