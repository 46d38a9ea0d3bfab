"""A paged cache: the writes into it (exact: a copy, or one rounding) and the attention over it against the definition in 64 bits.

The attention's bound, of an output sum_j w_j v_j with S = sum_j w_j |v_j|: a weight is rounded to the cache's type (half a step, u) and comes from a
score whose fp32 sum of D products drops at most 2^-23 of the largest addend twice per tensor-core step of 16 (A = largest scale sum |q k|), and whose exponential's
argument, a number up to A log2(e) with the maximum's taken off, rounds three times: relative error of a weight e = u + 2 ceil(D / 16) 2^-23 A + 6 * 2^-24 (A + 1) + 2^-21 (exp2).
The weights' sum adds up to `len` terms (2^-24 each, with those errors but u), the values' sum likewise in fp32: |y - exact| <= (2 e + 3 len 2^-24) S, and
fp16 weights below 2^-31 of the largest may vanish: 2^-31 sum |v|; then half a step of the output's type."""
import math

import numpy as np
import pytest
import torch

import qwengine_b200 as q
from qwengine_b200 import api

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
KIND = {"f32": 0, "f16": 1, "bf16": 2}


@pytest.fixture(params=["by rule", "two tiles of rows"])
def tiles(ctx, request):
    """The variants with two tiles of rows together, which the rule takes for many rows only, at the sizes of these tests too."""
    ctx.debug_set_attention_two(1 if request.param.startswith("two") else 0)
    yield
    ctx.debug_set_attention_two(0)


class Text:
    """A batch of sequences in a cache: plan = [(new tokens, tokens in all)], their keys and values in 64 bits beside the pages that hold them.  Slots that no
    token has, and pages that no sequence has, hold NaN."""

    def __init__(self, plan, nk, D, page, dtype="bf16", seed=0, layout="page", spare_entries=2, bad=()):
        g = torch.Generator().manual_seed(seed)
        self.plan, self.nk, self.D, self.page, self.dtype = plan, nk, D, page, dtype
        need = [-(-max(total, 0) // page) for _, total in plan]
        pages = sum(need) + 3
        order = torch.randperm(pages, generator=g)
        table = torch.full((len(plan), max(need) + spare_entries), -7, dtype=torch.int32)
        at = 0
        for s, n in enumerate(need):
            table[s, :n] = order[at:at + n]
            at += n
        if spare_entries:
            table[:, -1] = 2 ** 31 - 1
        dt = DTYPES[dtype]
        self.keys = [torch.randn((max(t, 0), nk, D), generator=g).to(dt) for _, t in plan]
        self.values = [torch.randn((max(t, 0), nk, D), generator=g).to(dt) for _, t in plan]
        k, v = (torch.full((pages, page, nk, D), float("nan"), dtype=dt) for _ in range(2))
        for s, n in enumerate(need):
            for i in range(n):
                part = slice(i * page, min((i + 1) * page, plan[s][1]))
                k[table[s, i], :part.stop - part.start] = self.keys[s][part]
                v[table[s, i], :part.stop - part.start] = self.values[s][part]
        for s, i, number in bad:                        # entries that are no page's: the tokens there read as zeros
            table[s, i] = number
            part = slice(i * page, (i + 1) * page)
            self.keys[s][part], self.values[s][part] = 0, 0
        if layout == "head":                            # [page][head][slot][element]
            k, v = (t.transpose(1, 2).contiguous().cuda().transpose(1, 2) for t in (k, v))
        elif layout == "both":                          # keys and values of a slot side by side, padded
            room = torch.full((pages, page, 2, nk, D + 8), float("nan"), dtype=dt).cuda()
            room[:, :, 0, :, :D], room[:, :, 1, :, :D] = k.cuda(), v.cuda()
            k, v = room[:, :, 0, :, :D], room[:, :, 1, :, :D]
        else:
            k, v = k.cuda(), v.cuda()
        self.k, self.v, self.cache = k, v, q.PagedCache(k, v)
        self.table = table.cuda()
        self.lengths = torch.tensor([t for _, t in plan], dtype=torch.int32, device="cuda")
        self.begin = torch.tensor(np.concatenate([[0], np.cumsum([n for n, _ in plan])]), dtype=torch.int32, device="cuda")
        self.rows = sum(n for n, _ in plan)


def definition(text, x, scale, dtype_in):
    """(out, S, A, sum |v|, lse, len) of every row and head, float64."""
    x = x.to(DTYPES[text.dtype]).double().cpu()        # fp32 queries are rounded to the cache's type
    rows, nq, D = x.shape
    out, S, V = (torch.zeros((rows, nq, D), dtype=torch.float64) for _ in range(3))
    A, lse, count = torch.zeros((rows, nq)), torch.full((rows, nq), -math.inf, dtype=torch.float64), torch.zeros((rows, nq))
    row = 0
    for (new, total), keys, values in zip(text.plan, text.keys, text.values):
        for i in range(new):
            n = max(0, min(total - new + i + 1, total))
            for h in range(nq if n else 0):
                kv = h * text.nk // nq
                K, Vh = keys[:n, kv].double(), values[:n, kv].double()
                s = scale * (K @ x[row + i, h])
                w = torch.softmax(s, 0)
                out[row + i, h], S[row + i, h], V[row + i, h] = w @ Vh, w @ Vh.abs(), Vh.abs().sum(0)
                A[row + i, h] = float((scale * (K.abs() @ x[row + i, h].abs())).max())
                lse[row + i, h], count[row + i, h] = torch.logsumexp(s, 0), n
        row += new
    return out, S, A, V, lse, count


def half_step(dtype, value):
    f = torch.finfo(DTYPES[dtype])
    return f.eps / 2 * value.abs().clamp(min=f.smallest_normal)


def check(text, x, got, scale, lse=None):
    exact, S, A, V, want_lse, n = definition(text, x, scale, x.dtype)
    kind = {v: k for k, v in DTYPES.items()}[got.dtype]
    u = torch.finfo(DTYPES[text.dtype]).eps / 2
    e0 = (2 * -(-text.D // 16) * 2.0 ** -23 * A + 6 * 2.0 ** -24 * (A + 1) + 2.0 ** -21).double()
    e = (u + e0).unsqueeze(-1)
    tol = (2 * e + 3 * n.double().unsqueeze(-1) * 2.0 ** -24) * S + (2.0 ** -31 * V if text.dtype == "f16" else 0)
    tol = tol + (half_step(kind, exact.abs() + tol) if kind != "f32" else 2.0 ** -24 * exact.abs())
    got = got.double().cpu()
    bad = ~((got - exact).abs() <= tol)
    assert not bool(bad.any()), (bad.nonzero()[:4], got[bad][:4], exact[bad][:4], tol[bad][:4])
    assert bool((got[(n == 0)] == 0).all())
    if lse is not None:
        l = lse.double().cpu()
        seen = n > 0
        assert bool((l[~seen] == -math.inf).all())
        tol = 2 * e0 + n.double() * 2.0 ** -23 + 2.0 ** -22 * (1 + want_lse.abs())
        assert bool(((l - want_lse).abs()[seen] <= tol[seen]).all())


def run(ctx, plan, nq=6, nk=2, D=64, page=16, dtype="bf16", src=None, dst=None, layout="page", scale=None, seed=0, **kw):
    text = Text(plan, nk, D, page, dtype, seed, layout, **kw)
    g = torch.Generator().manual_seed(seed + 1)
    x = (torch.randn((text.rows, nq, D), generator=g) * torch.exp(0.5 * torch.randn((text.rows, nq, 1), generator=g))).to(DTYPES[src or dtype]).cuda()
    lse = torch.full((text.rows, nq), 5.0, device="cuda")
    got = ctx.attention(text.cache, x, text.table, text.lengths, text.begin, scale=scale, kind=KIND[dst or src or dtype], lse=lse)
    ctx.check()
    check(text, x, got, D ** -0.5 if scale is None else scale, lse)
    return text, x, got


@pytest.mark.parametrize("D", [8, 16, 40, 64, 72, 80, 96, 128, 136, 192, 200, 256])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_head_sizes(ctx, tiles, D, dtype):
    run(ctx, [(1, 1), (3, 200), (70, 70)], D=D, dtype=dtype)


@pytest.mark.parametrize("nq,nk", [(1, 1), (7, 1), (4, 4), (24, 4), (15, 5), (128, 1), (130, 1), (300, 1)])
@pytest.mark.parametrize("D", [64, 256])
def test_groups(ctx, tiles, nq, nk, D):
    run(ctx, [(1, 300), (5, 140)], nq=nq, nk=nk, D=D)


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256, 1024])
@pytest.mark.parametrize("D", [64, 96, 256])
def test_page_sizes(ctx, tiles, page, D):
    run(ctx, [(1, 1), (2, 129), (9, 300), (1, 1025)], page=page, D=D)


@pytest.mark.parametrize("total", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 700])
@pytest.mark.parametrize("new", [1, 2, 22, 43])
@pytest.mark.parametrize("D", [128, 256])
def test_lengths(ctx, tiles, total, new, D):
    run(ctx, [(new, total)], D=D, seed=total)     # some chunks are longer than their text: rows that see nothing


@pytest.mark.parametrize("n", [383, 384, 385, 1000])
def test_many_sequences(ctx, tiles, n):
    rng = np.random.default_rng(n)
    run(ctx, [(int(k), int(t)) for k, t in zip(rng.integers(0, 3, n), rng.integers(0, 60, n))], nq=2, nk=1, D=64)
    run(ctx, [(0, 5)] * (n - 1) + [(1, 300)], nq=2, nk=1, D=256)


def test_many_rows(ctx):
    """Enough rows for the rule to take two tiles of them together: several sequences, cuts inside tiles."""
    for D, nq, nk, dtype in ((256, 24, 4, "bf16"), (128, 48, 8, "f16"), (64, 48, 8, "bf16")):
        run(ctx, [(700, 900), (1, 300), (130, 131)], nq=nq, nk=nk, D=D, dtype=dtype)


def test_ragged_batches(ctx, tiles):
    run(ctx, [(0, 50), (1, 700), (0, 0), (33, 33), (5, 0), (1, 1), (2, 1), (64, 500), (0, 3)], D=256)
    run(ctx, [(0, 50), (1, 700), (0, 0), (33, 33), (5, 0), (1, 1), (2, 1), (64, 500), (0, 3)], D=96, dtype="f16", page=32)
    run(ctx, [(1, 1 + 37 * s % 400) for s in range(70)], D=128, nq=4, nk=2)


@pytest.mark.parametrize("src,dst", [("f32", "f32"), ("f32", "bf16"), ("bf16", "f32"), ("bf16", "f16")])
def test_types(ctx, tiles, src, dst):
    run(ctx, [(1, 90), (40, 150)], D=256, src=src, dst=dst)
    run(ctx, [(1, 90), (40, 150)], D=80, src=src, dst=dst)


@pytest.mark.parametrize("layout", ["head", "both"])
@pytest.mark.parametrize("nk", [1, 3])
def test_layouts(ctx, tiles, layout, nk):
    run(ctx, [(1, 90), (40, 150)], nq=2 * nk, nk=nk, D=128, layout=layout)
    run(ctx, [(3, 90)], nq=2 * nk, nk=nk, D=256, layout=layout, page=64)


@pytest.mark.parametrize("scale", [1e-3, 1.0, 20.0])
def test_scales(ctx, tiles, scale):
    run(ctx, [(1, 400), (30, 300)], D=64, scale=scale)
    run(ctx, [(1, 400), (30, 300)], D=256, scale=scale, dtype="f16")


def test_growing_scores(ctx, tiles):
    """Keys whose scores rise along the text, by steps small and large: the running maximum moves in every tile, or in some."""
    for rise in (0.01, 0.05, 0.4):
        for D in (64, 256):
            text = Text([(3, 900)], 1, D, 16, seed=3)
            x = torch.ones((3, 2, D), dtype=torch.bfloat16)
            ramp = (torch.arange(900).float() * rise / math.sqrt(D)).to(torch.bfloat16)
            text.keys[0][:, 0] = ramp[:, None] + 0 * text.keys[0][:, 0]
            page_of = text.table[0].long().cpu()
            for j in range(900):
                text.k[page_of[j // 16], j % 16, 0] = text.keys[0][j, 0].cuda()
            got = ctx.attention(text.cache, x.cuda(), text.table, text.lengths, text.begin)
            ctx.check()
            check(text, x, got, D ** -0.5)


def test_entries_that_are_no_pages(ctx, tiles):
    for D in (64, 256):
        run(ctx, [(2, 100), (1, 40)], D=D, bad=[(0, 2, -1), (1, 0, 1 << 30), (0, 5, 1000)])


def test_lengths_and_rows_past_their_ends(ctx, tiles):
    """Lengths past the table, rows past q, begins that fall: clamped, nothing outside is touched."""
    text = Text([(2, 64), (3, 64)], 2, 64, 16, spare_entries=0)
    text.k.nan_to_num_(0.5), text.v.nan_to_num_(0.25)
    x = torch.randn((5, 4, 64), device="cuda").bfloat16()
    full = ctx.attention(text.cache, x, text.table, torch.full_like(text.lengths, 64), text.begin)
    over = ctx.attention(text.cache, x, text.table, torch.full_like(text.lengths, 2 ** 31 - 1), text.begin)
    assert torch.equal(full, over)
    out = torch.full((9, 4, 64), 3.0, device="cuda", dtype=torch.bfloat16)
    lse = torch.full((9, 4), 3.0, device="cuda")
    big = torch.cat([x, torch.full((4, 4, 64), float("nan"), device="cuda", dtype=torch.bfloat16)])
    ctx.attention(text.cache, big, text.table, torch.full_like(text.lengths, 64), text.begin, out=out, lse=lse)
    assert torch.equal(out[:5], full) and bool((out[5:] == 3).all()) and bool((lse[5:] == 3).all()), "rows behind the last sequence"
    beyond = torch.tensor([0, 2, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    falling = torch.tensor([4, 2, -5], dtype=torch.int32, device="cuda")
    ctx.attention(text.cache, x, text.table, text.lengths, beyond)
    out.fill_(3.0)
    ctx.attention(text.cache, x, text.table, text.lengths, falling, out=out[:5])
    ctx.check()
    assert bool((out == 3).all())


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_what_a_row_does_not_see_has_no_influence(ctx, tiles, D, what):
    """NaN and infinities in keys and values of later tokens of the chunk itself."""
    plan, nq, nk = [(40, 150), (3, 10)], 4, 2
    text, x, got = run(ctx, plan, nq=nq, nk=nk, D=D)
    for first_spoilt in (111, 130, 149):       # (a token of the chunk: rows before it are as they were)
        for which in ("k", "v"):
            spoilt = Text(plan, nk, D, 16)
            pages = spoilt.table[0].long().cpu()
            for j in range(first_spoilt, 150):
                (spoilt.k if which == "k" else spoilt.v)[pages[j // 16], j % 16, :, j % D] = what
            again = ctx.attention(spoilt.cache, x, spoilt.table, spoilt.lengths, spoilt.begin)
            ctx.check()
            clean = first_spoilt - 110
            assert torch.equal(again[:clean], got[:clean]) and torch.equal(again[40:], got[40:])
            if which == "v":
                cols = [c for c in range(D) if c != first_spoilt % D]
                assert not bool(again[clean, :, first_spoilt % D].isfinite().any()) and bool(again[clean][:, cols].isfinite().all())


def test_the_same_bits_and_graphs(ctx):
    """A captured call follows the lengths, tables and rows that its tensors hold when it is replayed; two graphs and two streams at once."""
    plan = [(1, 500), (2, 77), (1, 1)]
    text = Text(plan, 2, 256, 16, seed=1)
    x = torch.randn((4, 12, 256), device="cuda").bfloat16()
    want = ctx.attention(text.cache, x, text.table, text.lengths, text.begin)
    for _ in range(5):
        assert torch.equal(ctx.attention(text.cache, x, text.table, text.lengths, text.begin), want)
    shorter = torch.tensor([300, 40, 1], dtype=torch.int32, device="cuda")
    want_shorter = ctx.attention(text.cache, x, text.table, shorter, text.begin)
    lengths = text.lengths.clone()
    ga, gb = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(ga):
        ya = ctx.attention(text.cache, x, text.table, lengths, text.begin)
    with torch.cuda.graph(gb):
        yb = ctx.attention(text.cache, x, text.table, shorter, text.begin)
    lengths.copy_(shorter)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(10):
        with torch.cuda.stream(a):
            ga.replay()
        with torch.cuda.stream(b):
            gb.replay()
            yc = ctx.attention(text.cache, x, text.table, text.lengths, text.begin)
        torch.cuda.synchronize()
        assert torch.equal(ya, want_shorter) and torch.equal(yb, want_shorter) and torch.equal(yc, want)
    ctx.check()


def test_strided_queries_and_outputs(ctx, tiles):
    """Queries beside their gates, outputs inside a larger tensor, at any alignment."""
    text = Text([(1, 90), (20, 60)], 2, 128, 16)
    base = torch.randn((21, 8 * 2 * 128 + 3), device="cuda").bfloat16()
    for off in (0, 1, 3):
        x = base[:, off:off + 8 * 256].unflatten(1, (8, 256))[:, :, :128]
        room = torch.full((21, 8, 130 + off), 2.0, device="cuda", dtype=torch.bfloat16)
        out = room[:, :, off:off + 128]
        ctx.attention(text.cache, x, text.table, text.lengths, text.begin, out=out)
        ctx.check()
        check(text, x, out, 128 ** -0.5)
        assert bool((room[:, :, :off] == 2).all()) and bool((room[:, :, off + 128:] == 2).all())


@pytest.mark.parametrize("D", [8, 40, 72, 136, 200])
def test_queries_of_any_alignment_in_padded_heads(ctx, tiles, D):
    """What lies behind a head's elements in shared memory (here: whatever a text of NaN left there) must not get into its scores."""
    spoilt = Text([(64, 64)], 1, 256, 16)
    spoilt.k.fill_(float("nan")), spoilt.v.fill_(float("nan"))
    for src in ("bf16", "f32"):
        ctx.attention(spoilt.cache, torch.full((64, 6, 256), float("nan"), device="cuda", dtype=torch.bfloat16), spoilt.table, spoilt.lengths, spoilt.begin)
        text = Text([(1, 90), (20, 60)], 2, D, 16)
        x = torch.randn((21, 8 * (D + 1) + 1), device="cuda").to(DTYPES[src])[:, 1:].unflatten(1, (8, D + 1))[:, :, :D]
        got = ctx.attention(text.cache, x, text.table, text.lengths, text.begin)
        ctx.check()
        check(text, x, got, D ** -0.5)


def test_far_pages(ctx):
    """Pages whose elements lie past 2^32 bytes from the first."""
    page_bytes = 5 << 30
    room = torch.empty(2 * page_bytes + (1 << 20), dtype=torch.uint8, device="cuda")
    k = room.view(torch.bfloat16).as_strided((3, 16, 2, 64), (page_bytes // 2, 128, 64, 1))
    v = room[1 << 19:].view(torch.bfloat16).as_strided((3, 16, 2, 64), (page_bytes // 2, 128, 64, 1))
    text = Text([(2, 40)], 2, 64, 16, seed=6)
    cache = q.PagedCache(k, v)
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
    k.zero_(), v.fill_(float("nan"))
    keys, values = text.keys[0].cuda(), text.values[0].cuda()
    begin = torch.tensor([0, 40], dtype=torch.int32, device="cuda")
    ctx.cache_append(cache, keys, values, table, text.lengths, begin)
    x = torch.randn((2, 4, 64), device="cuda").bfloat16()
    got = ctx.attention(cache, x, table, text.lengths, text.begin)
    ctx.check()
    check(text, x, got, 0.125)


def test_long_text(ctx, tiles):
    """70001 tokens, whose scores' maxima come late."""
    for D, nk in ((256, 1), (64, 2)):
        text = Text([(2, 70001)], nk, D, 64, seed=2)
        x = torch.randn((2, 6, D), generator=torch.Generator().manual_seed(3)).bfloat16()
        got = ctx.attention(text.cache, x.cuda(), text.table, text.lengths, text.begin)
        ctx.check()
        check(text, x, got, D ** -0.5)


# ---- the writes ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("src,dst", [("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("nk,D,page,layout", [(1, 8, 8, "page"), (4, 256, 16, "page"), (5, 96, 32, "head"), (3, 72, 64, "both"), (40, 128, 16, "page")])
def test_append(ctx, src, dst, nk, D, page, layout):
    plan = [(3, 40), (0, 9), (1, 1), (50, 50), (4, 2), (0, 0), (17, 100)]       # the fifth: two rows before its first token
    text = Text(plan, nk, D, page, dst, layout=layout, bad=[(6, 6, -1)] if page == 16 else ())
    rows = text.rows + 2                                                         # two rows that are nobody's
    g = torch.Generator().manual_seed(2)
    for off in (0, 1):
        both = torch.randn((rows, 2 * nk * D + off), generator=g).to(DTYPES[src]).cuda()
        both[5, off:off + 4] = torch.tensor([float("inf"), float("nan"), 1e30, -0.0], device="cuda").to(both.dtype)
        k, v = both[:, off:off + nk * D].unflatten(1, (nk, D)), both[:, off + nk * D:].unflatten(1, (nk, D))
        want_k, want_v = text.k.clone(), text.v.clone()
        table, row = text.table.cpu(), 0
        for s, (new, total) in enumerate(plan):
            for i in range(new):
                j = total - new + i
                if j >= 0 and 0 <= int(table[s, j // page]) < text.k.shape[0]:
                    want_k[table[s, j // page], j % page] = k[row + i].to(DTYPES[dst])
                    want_v[table[s, j // page], j % page] = v[row + i].to(DTYPES[dst])
            row += new
        ctx.cache_append(text.cache, k, v, text.table, text.lengths, text.begin)
        torch.cuda.synchronize()
        for got, want in ((text.k, want_k), (text.v, want_v)):
            same = (got == want) | (got.isnan() & want.isnan())
            assert bool(same.all())


def test_append_finds_rows_of_many_sequences(ctx):
    rng = np.random.default_rng(1)
    for n in (31, 32, 33, 1000, 1025, 3000):
        plan = [(int(k), int(k + rng.integers(0, 20))) for k in rng.integers(0, 3, n)]
        text = Text(plan, 1, 8, 8, seed=n)
        text.k.zero_(), text.v.zero_()
        k = (torch.arange(text.rows, device="cuda").float()[:, None, None] % 251 + 1).expand(-1, 1, 8).bfloat16().contiguous()
        ctx.cache_append(text.cache, k, 2 * k, text.table, text.lengths, text.begin)
        at = [(s, t - new + i) for s, (new, t) in enumerate(plan) for i in range(new)]
        table = text.table.cpu()
        page, slot = torch.tensor([int(table[s, j // 8]) for s, j in at]).cuda(), torch.tensor([j % 8 for _, j in at]).cuda()
        assert torch.equal(text.k[page, slot], k) and torch.equal(text.v[page, slot], 2 * k)
        assert int((text.k != 0).sum()) == text.rows * 8


def test_the_wrappers_work_area_is_the_librarys(ctx):
    """The wrapper counts its bytes itself: less would be refused, more is not needed."""
    for D, nq, nk, rows in ((64, 4, 2, 1), (8, 1, 1, 7), (128, 48, 8, 300), (136, 6, 6, 9), (256, 24, 4, 3), (256, 24, 4, 5000)):
        asked = []
        text = Text([(0, 5)], nk, D, 16)
        real, ctx_lib = api._empty, ctx.lib
        api._empty = lambda shape, *a, **kw: (asked.append(shape), real(shape, *a, **kw))[1]
        try:
            ctx.attention(text.cache, torch.zeros((rows, nq, D), dtype=torch.bfloat16, device="cuda"), text.table, text.lengths, text.begin)
        finally:
            api._empty = real
        assert asked[-1] == (ctx_lib.q38b_attention_work_bytes(ctx.h, nq, nk, D, rows),)


def test_wrapper_refusals(ctx):
    text = Text([(1, 20)], 2, 64, 16)
    x = torch.randn((1, 4, 64), device="cuda").bfloat16()
    call = lambda x=x, table=text.table, lengths=text.lengths, begin=text.begin, **kw: ctx.attention(text.cache, x, table, lengths, begin, **kw)   # noqa: E731
    k = x[:, :2]
    append = lambda k=k, v=k, begin=text.begin: ctx.cache_append(text.cache, k, v, text.table, text.lengths, begin)   # noqa: E731
    for bad in (lambda: call(x=x[:, :, :32]), lambda: call(x=x.double()), lambda: call(x=x.cpu()), lambda: call(table=text.table.long()), lambda: call(lengths=text.lengths[:0]),
                lambda: call(begin=text.begin[:1]), lambda: call(begin=text.begin.cpu()), lambda: call(out=torch.empty((1, 4, 32), device="cuda")), lambda: call(lse=torch.empty((1, 3), device="cuda")),
                lambda: append(k=x), lambda: append(v=k.float()), lambda: append(k=k.cpu()), lambda: append(begin=text.begin.long()),
                lambda: q.PagedCache(text.k, text.v[:1]), lambda: q.PagedCache(text.k.float(), text.v.float()), lambda: q.PagedCache(text.k[..., ::2], text.v[..., ::2])):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: call(x=torch.randn((1, 3, 64), device="cuda").bfloat16()), lambda: call(x=x.half()), lambda: call(scale=0.0), lambda: append(k=k.half(), v=k.half())):
        with pytest.raises(api.Q38BError):
            bad()
    assert call(x=x[:0]).shape == (0, 4, 64) and append(k=k[:0], v=k[:0]) is None


# ---- batches of at most 8 rows a key head, which warps work on by themselves ----
@pytest.mark.parametrize("nq,nk", [(1, 1), (6, 3), (8, 1), (4, 2), (7, 7)])
@pytest.mark.parametrize("D", [8, 64, 72, 128, 192, 256])
@pytest.mark.parametrize("src,cache,dst", [("bf16", "bf16", "bf16"), ("f32", "f16", "f32"), ("f16", "f16", "bf16")])
def test_few_rows(ctx, nq, nk, D, src, cache, dst):
    """Sequences of 0 to 8 / group new tokens of none to 700, some that see nothing, cut into parts and not."""
    most = 8 // (nq // nk)
    run(ctx, [(1, 1), (most, 700), (0, 40), (most, most), (1, 128), (min(2, most), 0), (1, 129), (most, 16 + most), (1, 0)], nq=nq, nk=nk, D=D, dtype=cache, src=src, dst=dst)


@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("page,layout", [(8, "page"), (64, "head"), (256, "both")])
def test_few_rows_of_many_and_of_long_sequences(ctx, D, page, layout):
    run(ctx, [(1, 1 + 7 * s % 400) for s in range(300)], nq=3, nk=1, D=D, page=page, layout=layout)
    run(ctx, [(1, 9000), (2, 3), (1, 20011)], nq=8, nk=2, D=D, page=page, layout=layout)


@pytest.mark.parametrize("D", [64, 128, 192, 256])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_few_rows_what_a_row_does_not_see_has_no_influence(ctx, D, dtype, what):
    plan, nq, nk = [(4, 150), (3, 10)], 4, 2
    text, x, got = run(ctx, plan, nq=nq, nk=nk, D=D, dtype=dtype)
    for first_spoilt in (147, 148, 149):
        for which in ("k", "v"):
            spoilt = Text(plan, nk, D, 16, dtype)
            pages = spoilt.table[0].long().cpu()
            for j in range(first_spoilt, 150):
                (spoilt.k if which == "k" else spoilt.v)[pages[j // 16], j % 16, :, j % D] = what
            again = ctx.attention(spoilt.cache, x, spoilt.table, spoilt.lengths, spoilt.begin)
            ctx.check()
            clean = first_spoilt - 146
            assert torch.equal(again[:clean], got[:clean]) and torch.equal(again[4:], got[4:])
            if which == "v":       # every row from there on has its weight times the infinity (or a NaN) in each spoilt column that it sees, and what it had in all others
                for row in range(clean, 4):
                    columns = [j % D for j in range(first_spoilt, 147 + row)]
                    others = [c for c in range(D) if c not in columns]
                    assert bool(torch.isnan(again[row][:, columns]).all() if math.isnan(what) else (again[row][:, columns] == what).all())
                    assert torch.equal(again[row][:, others], got[row][:, others])


@pytest.mark.parametrize("D", [8, 40, 72, 128, 256])
def test_few_rows_of_any_stride_and_alignment(ctx, D):
    text = Text([(1, 90), (2, 60), (1, 300)], 2, D, 16)
    g = torch.Generator().manual_seed(3)
    for src in ("bf16", "f32"):
        for offset in (0, 1, 8):
            room = torch.randn((4, 8, D + 11), generator=g).to(DTYPES[src]).cuda()
            x = room[:, :, offset:offset + D]
            back = torch.full((4, 8, D + 9), 7.0, device="cuda", dtype=DTYPES[src])
            out = back[:, :, offset:offset + D] if offset < 9 else None
            ctx.attention(text.cache, x, text.table, text.lengths, text.begin, out=out)
            ctx.check()
            check(text, x, out, D ** -0.5)
            assert bool((back[:, :, :offset] == 7).all()) and bool((back[:, :, offset + D:] == 7).all())


def test_few_rows_growing_scores(ctx):
    """Maxima that grow from tile to tile and from warp to warp, by more and by less than what the running maximum may lag behind, up and down."""
    for seed, step in enumerate((0.02, 0.3, -0.3)):
        text = Text([(2, 900), (1, 400)], 2, 64, 16, seed=seed)
        x = torch.randn((3, 8, 64), generator=torch.Generator().manual_seed(seed)).bfloat16().cuda()
        for s, (_, total) in enumerate(text.plan):     # keys along the first query's direction, longer and longer
            for kv in range(2):
                d = x[2 * s, 4 * kv].float().cpu()
                d = d / (d @ d)
                grow = (torch.arange(total).float() * step if step > 0 else (torch.arange(total).float() - total) * step).unsqueeze(1) * d
                text.keys[s][:, kv] = (text.keys[s][:, kv].float() * 0.1 + grow).bfloat16()
            for i in range(-(-total // 16)):
                part = slice(i * 16, min((i + 1) * 16, total))
                text.k[text.table[s, i].long(), :part.stop - part.start] = text.keys[s][part].cuda()
        got = ctx.attention(text.cache, x, text.table, text.lengths, text.begin, scale=1.0)
        ctx.check()
        check(text, x, got, 1.0)


def test_a_captured_call_takes_few_rows_and_many(ctx):
    """Which way a batch goes is found out when the kernel runs: twelve sequences of a token each, then one of twelve."""
    text = Text([(1, 100 + s) for s in range(12)], 2, 128, 16)
    x = torch.randn((12, 8, 128), generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
    begin, lengths = text.begin.clone(), text.lengths.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ctx.attention(text.cache, x, text.table, lengths, begin)
    graph.replay()
    check(text, x, got, 128 ** -0.5)
    begin[1:] = 12
    graph.replay()
    ctx.check()
    one = Text.__new__(Text)
    one.plan, one.keys, one.values, one.nk, one.D, one.dtype = [(12, 100)], text.keys[:1], text.values[:1], 2, 128, "bf16"
    check(one, x, got, 128 ** -0.5)
    begin.copy_(text.begin)
    graph.replay()
    ctx.check()
    check(text, x, got, 128 ** -0.5)
