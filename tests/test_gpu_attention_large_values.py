"""Finite values near the end of their type: what is added up before the division must not pass fp32 while the outputs do not."""
import math

import pytest
import torch

from test_gpu_cache import Text, check, tiles   # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128, 192, 256])
@pytest.mark.parametrize("new,nq,nk", [(1, 4, 2), (3, 6, 1), (200, 4, 1)])
def test_maxima_that_lag_behind(ctx, tiles, D, new, nq, nk):   # noqa: F811
    """Scores 2^0 at the first token, 2^7.8 of a weight more at a few in later tiles (the running maximum may stay), 2^-40 elsewhere: the outputs are means of a few values of
    2^120 to 2^126.  With n tokens of weight 1 and a value of v each, v n < 2^127 is what is allowed."""
    total = 700 + new
    text = Text([(new, total)], nk, D, 16, seed=D)
    g = torch.Generator().manual_seed(D + new)
    log2 = torch.full((total,), -40.0)
    log2[0], log2[[150, 290, 400, 690]] = 0.0, 7.75
    text.keys[0] = torch.zeros_like(text.keys[0])
    text.keys[0][:, :, 0] = (log2 / 16).bfloat16().unsqueeze(1)                       # exact: a few bits each
    text.values[0] = torch.ldexp(torch.randn((total, nk, D), generator=g).clamp(-2, 2), torch.tensor(122)).bfloat16()
    text.values[0][[150, 400]] = 2.0 ** 124
    flat_k, flat_v = (torch.nn.functional.pad(t[0], (0, 0, 0, 0, 0, -total % 16)).unflatten(0, (-1, 16)) for t in (text.keys, text.values))
    n = flat_k.shape[0]
    text.k[text.table[0, :n].long()], text.v[text.table[0, :n].long()] = flat_k.cuda(), flat_v.cuda()
    x = torch.zeros((new, nq, D), dtype=torch.bfloat16)
    x[:, :, 0] = 16.0
    lse = torch.empty((new, nq), device="cuda")
    got = ctx.attention(text.cache, x.cuda(), text.table, text.lengths, text.begin, scale=math.log(2.0), kind=0, lse=lse)
    ctx.check()
    check(text, x.float(), got, math.log(2.0), lse)
    assert bool((got.abs() > 2.0 ** 121).any())


def test_small_values_and_sums_of_logarithms(ctx, tiles):   # noqa: F811
    """Values far below 1 (2^-100) keep their bits; a single token's logarithm is its score, small ones included."""
    text = Text([(20, 300), (1, 1), (9, 9)], 2, 64, 16, seed=4)
    text.v *= 2.0 ** -100
    text.values = [v * 2.0 ** -100 for v in text.values]
    x = torch.randn((text.rows, 8, 64), generator=torch.Generator().manual_seed(4)).bfloat16()
    lse = torch.empty((text.rows, 8), device="cuda")
    for scale in (1e-4, 0.125):
        got = ctx.attention(text.cache, x.cuda(), text.table, text.lengths, text.begin, scale=scale, kind=0, lse=lse)
        ctx.check()
        check(text, x.float(), got, scale, lse)
