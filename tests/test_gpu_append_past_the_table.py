"""Lengths that pass the table's last entry: rows behind it go nowhere, rows in front of it to their places, and nothing that is there is written over."""
import pytest
import torch

from test_gpu_cache import Text

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page", [8, 16, 64])
@pytest.mark.parametrize("over", [0, 1, 3, 4, 5, 1000, 2 ** 31 - 1])
def test_append(ctx, page, over):
    entries, new = 3, 4
    room = entries * page
    text = Text([(new, room), (2, 9)], 2, 64, page, spare_entries=0)
    length = min(room + over, 2 ** 31 - 1)
    lengths = torch.tensor([length, 9], dtype=torch.int32, device="cuda")
    k, v = (torch.randn((new + 2, 2, 64), generator=torch.Generator().manual_seed(s)).bfloat16().cuda() for s in (1, 2))
    want_k, want_v, table = text.k.clone(), text.v.clone(), text.table.long().cpu()
    for i in range(new):
        j = length - new + i
        if j < room:
            want_k[table[0, j // page], j % page], want_v[table[0, j // page], j % page] = k[i], v[i]
    for i in range(2):
        want_k[table[1, (7 + i) // page], (7 + i) % page], want_v[table[1, (7 + i) // page], (7 + i) % page] = k[new + i], v[new + i]
    ctx.cache_append(text.cache, k, v, text.table, lengths, text.begin)
    for got, want in ((text.k, want_k), (text.v, want_v)):
        assert bool(((got == want) | (got.isnan() & want.isnan())).all())
