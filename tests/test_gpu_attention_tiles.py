"""Attention where a CTA goes through several tiles of rows one behind the other: what one tile leaves must not reach the next, whatever the values hold."""
import pytest
import torch

from test_gpu_cache import Text, check

pytestmark = pytest.mark.gpu

# 48 sequences x 4 key heads, 320 (token, head) rows each: 576 tiles of 128 rows or 384 of 256, three and more a CTA (five a pair), every one with tokens of the chunk in it
PLAN = [(40, 40 + 7 * s % 31) for s in range(48)]
NQ, NK = 32, 4


@pytest.fixture(params=[-1, 0, 1], ids=["single tiles", "by rule", "two tiles"])
def two(ctx, request):
    ctx.debug_set_attention_two(request.param)
    yield request.param
    ctx.debug_set_attention_two(0)


_clean = {}


def clean_run(ctx, D, dtype, two):
    """The batch with ordinary numbers, checked against the definition (once for each way)."""
    key = (D, dtype, two)
    if key not in _clean:
        text = Text(PLAN, NK, D, 16, dtype, seed=D)
        x = torch.randn((text.rows, NQ, D), generator=torch.Generator().manual_seed(D)).to(text.k.dtype).cuda()
        lse = torch.empty((text.rows, NQ), device="cuda")
        got = ctx.attention(text.cache, x, text.table, text.lengths, text.begin, lse=lse)
        ctx.check()
        if two == 0:
            check(text, x, got, D ** -0.5, lse)
        _clean[key] = x, got, lse
    return _clean[key]


@pytest.mark.parametrize("D,dtype", [(64, "bf16"), (96, "f16"), (128, "bf16"), (192, "bf16"), (256, "bf16"), (256, "f16")])
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
def test_values_that_are_no_numbers_stay_in_their_tile(ctx, two, D, dtype, what):
    """A value of a late token of the chunk, in the upper half of its head's elements, is no number, in every third sequence and one key head of it: rows in front of that token, other heads,
    other elements and other sequences are what they were, bit for bit."""
    x, want, want_lse = clean_run(ctx, D, dtype, two)
    text = Text(PLAN, NK, D, 16, dtype, seed=D)
    table = text.table.long().cpu()
    spoilt = torch.zeros(want.shape, dtype=torch.bool)
    for s, (new, total) in enumerate(PLAN):
        if s % 3:
            continue
        kv, first = s // 3 % NK, 21 + s % 11                   # tokens `first` to first + 2 of the chunk
        for i in range(first, first + 3):
            j, e = total - new + i, D // 2 + (5 * s + 9 * i) % (D - D // 2)
            text.v[table[s, j // 16], j % 16, kv, e] = what
            group = NQ // NK
            spoilt[40 * s + i:40 * (s + 1), kv * group:(kv + 1) * group, e] = True
    for _ in range(3):
        lse = torch.empty_like(want_lse)
        got = ctx.attention(text.cache, x, text.table, text.lengths, text.begin, lse=lse)
        ctx.check()
        got, lse = got.cpu(), lse.cpu()
        assert torch.equal(got[~spoilt], want.cpu()[~spoilt]) and torch.equal(lse, want_lse.cpu())
        assert not bool(got[spoilt].isfinite().any())
