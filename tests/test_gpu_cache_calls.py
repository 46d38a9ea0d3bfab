"""Calls of the cache and the attention that a host may make and that are easily forgotten: captured appends, rows in front of the first sequence, a text twice in a batch, shared
queries, pages far apart under many rows."""
import pytest
import torch

import qwengine_b200 as q

from test_gpu_cache import Text, check, tiles   # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def test_captured_appends_on_two_streams(ctx):
    """Two graphs, replayed at once on streams of their own, each into its own pages of one cache, as the lengths move on."""
    page, nk, D, steps = 16, 2, 64, 40
    k, v = (torch.zeros((8, page, nk, D), device="cuda", dtype=torch.bfloat16) for _ in range(2))
    cache = q.PagedCache(k, v)
    tables = [torch.tensor([t], dtype=torch.int32, device="cuda") for t in ([5, 0, 3], [2, 7, 1])]
    lengths = [torch.zeros(1, dtype=torch.int32, device="cuda") for _ in range(2)]
    begin = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    rows = [torch.zeros((1, nk, D), device="cuda") for _ in range(2)]
    graphs, streams = [torch.cuda.CUDAGraph() for _ in range(2)], [torch.cuda.Stream() for _ in range(2)]
    for i in range(2):
        with torch.cuda.graph(graphs[i]):
            ctx.cache_append(cache, rows[i], -rows[i], tables[i], lengths[i], begin)
    torch.cuda.synchronize()
    for j in range(steps):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                rows[i].fill_(1000 * i + j + 1)
                lengths[i].fill_(j + 1)
                graphs[i].replay()
    torch.cuda.synchronize()
    for i in range(2):
        want = (1000.0 * i + 1 + torch.arange(steps, device="cuda")).bfloat16().view(-1, 1, 1).expand(-1, nk, D)
        assert torch.equal(k[tables[i][0].long()].flatten(0, 1)[:steps], want) and torch.equal(v[tables[i][0].long()].flatten(0, 1)[:steps], -want)
    assert bool((k[[4, 6]] == 0).all()) and bool((k[3, 8:] == 0).all())


@pytest.mark.parametrize("D", [64, 128, 256])
def test_rows_in_front_of_the_first_sequence(ctx, tiles, D):   # noqa: F811
    """begin[0] above 0: the rows in front are nobody's."""
    text = Text([(1, 70), (30, 200)], 2, D, 16)
    x = torch.randn((text.rows, 8, D), generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    front = 7
    big = torch.cat([torch.full((front, 8, D), float("nan"), device="cuda", dtype=torch.bfloat16), x])
    out, lse = torch.full_like(big, 3.0), torch.full((front + text.rows, 8), 3.0, device="cuda")
    ctx.attention(text.cache, big, text.table, text.lengths, text.begin + front, out=out, lse=lse)
    ctx.check()
    assert bool((out[:front] == 3).all()) and bool((lse[:front] == 3).all())
    check(text, x, out[front:], D ** -0.5, lse[front:])
    before = text.k.clone(), text.v.clone()
    new = torch.randn((front + text.rows, 2, D), device="cuda").bfloat16()
    ctx.cache_append(text.cache, new, new, text.table, text.lengths, text.begin + front)
    at = text.table[0, 69 // 16].long(), 69 % 16
    assert torch.equal(text.k[at], new[front]) and torch.equal(text.v[at], new[front])
    for pages, was in zip((text.k, text.v), before):
        changed = ((pages != was) & ~(pages.isnan() & was.isnan())).flatten(2).any(2)
        assert int(changed.sum()) == text.rows


@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("new", [1, 40])
def test_a_text_twice_in_a_batch_and_one_query_for_all_heads(ctx, tiles, D, new):   # noqa: F811
    """Two entries of a batch name the same pages (several continuations of one text are read so), every head has the same query (a head stride of 0), keys are their own values."""
    text = Text([(new, 150)], 2, D, 16)
    cache = q.PagedCache(text.k, text.k)
    table, lengths = text.table.expand(2, -1).contiguous(), text.lengths.expand(2).contiguous()
    begin = torch.tensor([0, new, 2 * new], dtype=torch.int32, device="cuda")
    x = torch.randn((2 * new, 1, D), generator=torch.Generator().manual_seed(2)).bfloat16().cuda().expand(-1, 8, -1)
    got = ctx.attention(cache, x, table, lengths, begin)
    ctx.check()
    text.plan, text.keys, text.values = text.plan * 2, text.keys * 2, text.keys * 2
    check(text, x, got, D ** -0.5)


@pytest.mark.parametrize("D,nq,two", [(64, 8, -1), (64, 8, 1), (256, 24, -1), (256, 24, 1)])
def test_far_pages_of_many_rows(ctx, D, nq, two):
    """Pages past 2^32 bytes from the first under tiles of rows, values that are no numbers among them."""
    nk, page_bytes, new, total = 2, 5 << 30, 40, 45
    slot = nk * D
    room = torch.empty(2 * page_bytes + (1 << 21), dtype=torch.uint8, device="cuda")
    k = room.view(torch.bfloat16).as_strided((3, 16, nk, D), (page_bytes // 2, slot, D, 1))
    v = room[1 << 20:].view(torch.bfloat16).as_strided((3, 16, nk, D), (page_bytes // 2, slot, D, 1))
    text = Text([(new, total)], nk, D, 16, seed=6)
    cache = q.PagedCache(k, v)
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
    begin = torch.tensor([0, total], dtype=torch.int32, device="cuda")
    k.zero_(), v.fill_(float("nan"))
    ctx.cache_append(cache, text.keys[0].cuda(), text.values[0].cuda(), table, text.lengths, begin)
    x = torch.randn((new, nq, D), generator=torch.Generator().manual_seed(7)).bfloat16().cuda()
    ctx.debug_set_attention_two(two)
    try:
        got = ctx.attention(cache, x, table, text.lengths, text.begin)
        ctx.check()
        check(text, x, got, D ** -0.5)
        v[1, 8, 0, D - 1], v[0, 3, 1, 2] = float("inf"), float("nan")        # tokens 40 and 19: rows 35 and 14 on
        again = ctx.attention(cache, x, table, text.lengths, text.begin)
        ctx.check()
    finally:
        ctx.debug_set_attention_two(0)
    spoilt = torch.zeros_like(got, dtype=torch.bool)
    spoilt[35:, :nq // 2, D - 1] = True
    spoilt[14:, nq // 2:, 2] = True
    assert torch.equal(again[~spoilt], got[~spoilt]) and not bool(again[spoilt].isfinite().any())
