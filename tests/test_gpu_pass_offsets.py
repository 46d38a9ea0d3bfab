"""Recorded logit rules on a shard of a head: the tokens of the pass's logits begin at an offset, as in the direct call."""
import numpy as np
import pytest
import torch

import qwengine_b200 as q
from qwengine_b200 import api

from test_gpu_logits import check, definition

pytestmark = pytest.mark.gpu


def rules(nb, vocab, seed):
    """A text, biases and masks over a vocabulary of `vocab` tokens: device tensors, and the definition's arguments."""
    rng = np.random.default_rng(seed)
    text = rng.integers(0, vocab, (nb, 50)).astype(np.int32)
    ids = rng.integers(0, vocab, (nb, 9)).astype(np.int32)
    values = rng.standard_normal((nb, 9)).astype(np.float32)
    masks = rng.integers(0, 2 ** 32, (nb, (vocab + 31) // 32), dtype=np.uint32)
    penalties = np.tile(np.float32([1.25, 0.5, 0.25]), (nb, 1))
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()   # noqa: E731
    begin = lambda n: torch.arange(nb + 1, device="cuda") * n          # noqa: E731
    r = dict(penalties=dev(penalties), history=dev(text.reshape(-1)), history_begin=begin(50), prompt_len=torch.full((nb,), 20, dtype=torch.int32, device="cuda"),
             bias_ids=dev(ids.reshape(-1)), bias_values=dev(values.reshape(-1)), bias_begin=begin(9), masks=dev(masks.view(np.int32)))
    d = dict(penalties=penalties, history=[t.tolist() for t in text], prompt=[20] * nb, biases=[list(zip(i.tolist(), v.tolist())) for i, v in zip(ids, values)], masks=masks)
    return r, d


@pytest.mark.parametrize("nb", [1, 3])
@pytest.mark.parametrize("first,n", [(0, 700), (1, 700), (300, 700), (997, 3), (512, 488)])
@pytest.mark.parametrize("in_place", [True, False])
def test_recorded_rules_begin_at_their_token(ctx, nb, first, n, in_place):
    vocab = 1000
    r, d = rules(nb, vocab, first + nb)
    x = torch.randn((nb, vocab), generator=torch.Generator().manual_seed(first)).cuda()
    want = ctx.adjust_logits(x[:, first:first + n], index_offset=first, **r)
    whole, bound = definition(x.cpu().numpy(), **d)
    check(want, whole[:, first:first + n], bound[:, first:first + n])
    ps = q.Pass(ctx, max_nb=nb)
    src, dst = ps.buffer_f32(n + 4), ps.buffer_f32(n)
    ps.adjust_logits(src, 4, n, dst=None if in_place else dst, index_offset=first, **r)
    for _ in range(2):                       # recorded once, replayed
        ps.buffer_tensor(src)[:, 4:] = x[:, first:first + n]
        ps.run(nb)
        ctx.check()
        assert torch.equal(ps.buffer_tensor(src)[:, 4:] if in_place else ps.buffer_tensor(dst), want)
    ps.close()


def test_refusals(ctx):
    ps = q.Pass(ctx, max_nb=2)
    a = ps.buffer_f32(64)
    masks = torch.zeros((2, 4), dtype=torch.int32, device="cuda")       # 128 tokens
    with pytest.raises(ValueError):
        ps.adjust_logits(a, 0, 64, masks=masks, index_offset=65)
    for off in (-1, 2 ** 31 - 64):
        with pytest.raises(api.Q38BError):
            ps.adjust_logits(a, 0, 64, index_offset=off)
    ps.adjust_logits(a, 0, 64, masks=masks, index_offset=64)
    ps.run(2)
    ctx.check()
    assert torch.isneginf(ps.buffer_tensor(a)).all()                    # no token of these masks is allowed
    ps.close()


def test_without_an_offset_logits_begin_at_token_zero(ctx):
    """q38b_pass_op_adjust_logits records what the call with an offset of nothing does."""
    r, _ = rules(2, 300, 5)
    x = torch.randn((2, 300), generator=torch.Generator().manual_seed(6)).cuda()
    ps = q.Pass(ctx, max_nb=2)
    a = ps.buffer_f32(300)
    assert ps.lib.q38b_pass_op_adjust_logits(ps.h, a, 0, 300, ctx.logit_rules(2, 300, **r), a, 0) == 0
    ps.buffer_tensor(a).copy_(x)
    ps.run(2)
    ctx.check()
    assert torch.equal(ps.buffer_tensor(a), ctx.adjust_logits(x, **r))
    ps.close()


def test_more_logits_than_a_call_takes_are_not_recorded(ctx):
    ps = q.Pass(ctx, max_nb=1)
    a = ps.buffer_f32((1 << 30) + 1)
    with pytest.raises(api.Q38BError) as e:
        ps.adjust_logits(a, 0, (1 << 30) + 1)
    assert e.value.status == -2
    ps.adjust_logits(a, 1, 1 << 30)
    ps.close()
