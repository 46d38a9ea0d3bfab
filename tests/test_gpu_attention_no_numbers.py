"""Scores that are no numbers, where they are seen: outputs and logarithms of sums are what the formula gives, of these rows and of no others."""
import math

import pytest
import torch

from test_gpu_cache import Text, tiles   # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu

SHAPES = [(1, 4, 2), (40, 8, 2), (150, 4, 1)]      # new tokens, heads, key heads: the warps' own products, the tensor core's, more than one tile of rows


@pytest.mark.parametrize("D", [64, 128, 192, 256])
@pytest.mark.parametrize("new,nq,nk", SHAPES)
@pytest.mark.parametrize("total", [1, 100, 129, 700])
def test_queries(ctx, tiles, D, new, nq, nk, total):   # noqa: F811
    text = Text([(new, total + new), (2, 90)], nk, D, 16)
    g = torch.Generator().manual_seed(1)
    x = torch.randn((text.rows, nq, D), generator=g).bfloat16().cuda()
    lse, again_lse = (torch.empty((text.rows, nq), device="cuda") for _ in range(2))
    got = ctx.attention(text.cache, x, text.table, text.lengths, text.begin, lse=lse)
    bad = torch.zeros((text.rows, nq), dtype=torch.bool, device="cuda")
    bad[0, 1], bad[new // 2, nq - 1], bad[new, 0] = True, True, True
    spoilt = x.clone()
    spoilt[..., D // 3][bad] = float("nan")
    again = ctx.attention(text.cache, spoilt, text.table, text.lengths, text.begin, lse=again_lse)
    ctx.check()
    assert torch.equal(again[~bad], got[~bad]) and torch.equal(again_lse[~bad], lse[~bad])
    assert bool(again[bad].isnan().all()) and bool(again_lse[bad].isnan().all())


@pytest.mark.parametrize("D", [64, 128, 192, 256])
@pytest.mark.parametrize("new,nq,nk", SHAPES)
@pytest.mark.parametrize("first,last", [(0, 1), (0, 128), (0, 300), (128, 256), (200, 201), (256, 300)])
def test_keys(ctx, tiles, D, new, nq, nk, first, last):   # noqa: F811
    """Keys of the first head from token `first` on are NaN: all rows of that head see some."""
    total = 300
    text = Text([(new, total + new), (2, 90)], nk, D, 16)
    x = torch.randn((text.rows, nq, D), generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    lse, again_lse = (torch.empty((text.rows, nq), device="cuda") for _ in range(2))
    got = ctx.attention(text.cache, x, text.table, text.lengths, text.begin, lse=lse)
    for j in range(first, last):
        text.k[text.table[0, j // 16].long(), j % 16, 0, 1] = float("nan")
    again = ctx.attention(text.cache, x, text.table, text.lengths, text.begin, lse=again_lse)
    ctx.check()
    bad = torch.zeros((text.rows, nq), dtype=torch.bool, device="cuda")
    bad[:new, :nq // nk] = True
    assert torch.equal(again[~bad], got[~bad]) and torch.equal(again_lse[~bad], lse[~bad])
    assert bool(again[bad].isnan().all()) and bool(again_lse[bad].isnan().all())


@pytest.mark.parametrize("D", [64, 128, 192, 256])
@pytest.mark.parametrize("new,nq,nk", SHAPES)
@pytest.mark.parametrize("last", [128, 200, None])
def test_scores_of_minus_infinity(ctx, tiles, D, new, nq, nk, last):   # noqa: F811
    """The first `last` tokens' scores are minus infinity: their weights are zeros.  None: all are, and there is nothing to divide by."""
    total = 300 + new
    text = Text([(new, total)], nk, D, 16)
    x = torch.rand((new, nq, D), generator=torch.Generator().manual_seed(3)).bfloat16() + 0.5
    bound = last or total
    for j in range(bound):
        text.k[text.table[0, j // 16].long(), j % 16, :, 0] = -math.inf
    lse = torch.empty((new, nq), device="cuda")
    got = ctx.attention(text.cache, x.cuda(), text.table, text.lengths, text.begin, kind=0, lse=lse)
    ctx.check()
    if last is None:
        assert bool(got.isnan().all()) and bool((lse == -math.inf).all())
        return
    # what is left is the attention over the tokens behind them
    from test_gpu_cache import check
    left = Text.__new__(Text)
    left.plan, left.keys, left.values, left.nk, left.D, left.dtype = [(new, total - bound)], [text.keys[0][bound:]], [text.values[0][bound:]], nk, D, "bf16"
    check(left, x.float(), got, D ** -0.5, lse)
