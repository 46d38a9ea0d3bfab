"""Begins that fall, which no batch has: sequences of rows over and over.  The calls end and touch nothing outside their rows, also where the work so made up passes what 32 bits count."""
import pytest
import torch

import qwengine_b200 as q

pytestmark = pytest.mark.gpu


def falling(ctx, rows, n_seqs, D, tokens):
    page, guard = 8, 1000
    cache = q.PagedCache(*(torch.randn((tokens // page, page, 1, D), device="cuda").bfloat16() for _ in range(2)))
    table = torch.arange(tokens // page, dtype=torch.int32, device="cuda").expand(n_seqs, -1).contiguous()
    lengths = torch.full((n_seqs,), tokens, dtype=torch.int32, device="cuda")
    begin = torch.zeros(n_seqs + 1, dtype=torch.int32, device="cuda")
    begin[1::2] = rows                                  # 0, rows, 0, rows, ..: every other sequence is all of the rows
    x = torch.randn((rows, 1, D), device="cuda").bfloat16()
    room, lse = torch.full((rows + 2 * guard, 1, D), 3.0, device="cuda", dtype=torch.bfloat16), torch.full((rows + 2 * guard, 1), 3.0, device="cuda")
    ctx.attention(cache, x, table, lengths, begin, out=room[guard:-guard], lse=lse[guard:-guard])
    ctx.check()
    for t in (room, lse):
        assert bool((t[:guard] == 3).all()) and bool((t[-guard:] == 3).all())


@pytest.mark.parametrize("two", [-1, 0, 1])
@pytest.mark.parametrize("D", [64, 256])
def test_rows_over_and_over(ctx, two, D):
    ctx.debug_set_attention_two(two)
    try:
        for rows, n_seqs in ((5, 7), (300, 12), (1000, 100)):
            falling(ctx, rows, n_seqs, D, 256)
    finally:
        ctx.debug_set_attention_two(0)


@pytest.mark.parametrize("tiles", [32766, 32770])
def test_work_past_32_bits(ctx, tiles):
    """32767 sequences of `tiles` tiles of 128 rows, four units each: 2^32 - 393208, and 2^32 + 131064, which in 32 bits is 131064 again and again."""
    assert 32767 * 4 * 32770 == 2 ** 32 + 131064 and 32767 * 4 * 32766 == 2 ** 32 - 393208
    ctx.debug_set_attention_two(-1)
    try:
        falling(ctx, tiles * 128, 65534, 8, 128)
    finally:
        ctx.debug_set_attention_two(0)
