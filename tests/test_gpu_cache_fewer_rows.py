"""Calls for fewer rows than the batch's lists say: a call that ends inside a sequence writes and attends as a call for all rows does for those it has."""
import pytest
import torch

import qwengine_b200 as q

from test_gpu_cache import Text, check, tiles   # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def shortened(text, rows):
    """The same sequences with the rows that a call for `rows` of them has."""
    one = Text.__new__(Text)
    one.plan, at = [], 0
    for new, total in text.plan:
        there = max(0, min(new, rows - at))
        one.plan.append((there, total - new + there))
        at += new
    one.keys, one.values, one.nk, one.D, one.dtype = text.keys, text.values, text.nk, text.D, text.dtype
    return one


@pytest.mark.parametrize("D", [64, 128, 192, 256])
@pytest.mark.parametrize("nq,nk,plan", [(2, 2, [(4, 100), (1, 7), (3, 60)]), (6, 2, [(45, 200), (7, 90), (60, 61)]), (4, 2, [(5, 3), (40, 30), (9, 200)])])
def test_attention(ctx, tiles, D, nq, nk, plan):   # noqa: F811
    text = Text(plan, nk, D, 16)
    x = torch.randn((text.rows, nq, D), generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    for rows in {1, 2, plan[0][0] - 1, plan[0][0], plan[0][0] + 1, text.rows - 2, text.rows - 1, text.rows}:
        out, lse = torch.full((text.rows + 1, nq, D), 3.0, device="cuda", dtype=torch.bfloat16), torch.full((text.rows + 1, nq), 3.0, device="cuda")
        ctx.attention(text.cache, x[:rows], text.table, text.lengths, text.begin, out=out[:rows], lse=lse[:rows])
        ctx.check()
        check(shortened(text, rows), x[:rows], out[:rows], D ** -0.5, lse[:rows])
        assert bool((out[rows:] == 3).all()) and bool((lse[rows:] == 3).all())


def test_append(ctx):
    plan = [(4, 100), (0, 5), (30, 40), (3, 2), (6, 6)]
    text = Text(plan, 2, 64, 16)
    k, v = (torch.randn((text.rows, 2, 64), generator=torch.Generator().manual_seed(s)).bfloat16().cuda() for s in (1, 2))
    table = text.table.long().cpu()
    for rows in range(1, text.rows + 1):
        text.k.zero_(), text.v.zero_()
        want_k, want_v, row = text.k.clone(), text.v.clone(), 0
        for s, (new, total) in enumerate(plan):
            for i in range(new):
                j = total - new + i
                if row < rows and j >= 0:
                    want_k[table[s, j // 16], j % 16], want_v[table[s, j // 16], j % 16] = k[row], v[row]
                row += 1
        ctx.cache_append(text.cache, k[:rows], v[:rows], text.table, text.lengths, text.begin)
        assert torch.equal(text.k, want_k) and torch.equal(text.v, want_v)


def test_a_pass_for_fewer_columns_than_a_sequence_has(ctx):
    nq, nk, D, new, total = 4, 2, 64, 5, 60
    text = Text([(new, total)], nk, D, 16)
    ps = q.Pass(ctx, max_nb=new)
    heads, kv, mixed = ps.buffer_f32(nq * D), ps.buffer_f32(2 * nk * D), ps.buffer_f32(nq * D)
    batch = (text.table, text.lengths, text.begin)
    ps.cache_append(text.cache, dict(buf=kv), dict(buf=kv, off=nk * D), *batch)
    ps.attention(text.cache, dict(buf=heads, n_heads=nq), dict(buf=mixed), *batch)
    x, rows = torch.randn((new, nq, D), device="cuda"), torch.randn((new, 2, nk, D), device="cuda")
    ps.buffer_tensor(heads).copy_(x.flatten(1)), ps.buffer_tensor(kv).copy_(rows.flatten(1))
    before = text.keys[0].clone(), text.values[0].clone()
    for nb in (1, 2, 4, 5):
        text.keys[0], text.values[0] = before[0].clone(), before[1].clone()
        for i in range(nb):
            text.keys[0][total - new + i], text.values[0][total - new + i] = rows[i, 0].bfloat16().cpu(), rows[i, 1].bfloat16().cpu()
        ps.run(nb)
        ctx.check()
        for pages, held in ((text.k, text.keys[0]), (text.v, text.values[0])):
            flat = pages[text.table[0, :4].long()].flatten(0, 1)
            assert torch.equal(flat[:total].cpu(), held)
            flat[total - new:total] = (before[0] if pages is text.k else before[1])[total - new:].cuda()      # as they were, for the next run
            pages[text.table[0, :4].long()] = flat.unflatten(0, (4, 16))
        check(shortened(text, nb), x[:nb], ps.buffer_tensor(mixed)[:nb].unflatten(1, (nq, D)), D ** -0.5)
    ps.close()
