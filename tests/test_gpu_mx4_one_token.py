"""One token's product in every number of parts that two CTAs of an SM take: sums of whole numbers, exact whatever the cut, in one launch and in two."""
import pytest
import torch

import qwengine_b200 as q   # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,K", [(10700, 10240), (9216, 5120), (7680, 4096), (8100, 6144), (6144, 10240), (4608, 10240), (2560, 6144),    # 3, 3, 4, 4, 5 and 6 parts in one wave, 6 of whole SMs
                                 (24576, 10240), (20480, 7168), (12288, 10240)])                                                            # more CTAs than places
def test_whole_number_products(ctx, M, K):
    gen = torch.Generator("cuda").manual_seed(M + K)
    x, w = (torch.randint(-4, 5, (n, K), generator=gen, device="cuda").float() for n in (1, M))
    x[:, ::32], w[:, ::32] = 4, -4                # every block scaled by one: whole numbers up to 4 are E2M1 values, sums stay below 2^24
    x[0, 64:96] = 0                               # ... but for a block of nothing
    whole = torch.full((M + 6,), 3.0, device="cuda")
    y = whole[3:M + 3].unsqueeze(0)
    W = ctx.quantize_mx4(w)
    ctx.gemm_mx4(W, x, out=y)
    ctx.check()
    assert torch.equal(y, (x.double() @ w.double().t()).float())
    assert torch.equal(y, ctx.gemm_mx4(W, ctx.quantize_mx4(x)))
    for _ in range(3):
        assert torch.equal(y, ctx.gemm_mx4(W, x))
    ctx.check()
    assert (whole[:3] == 3.0).all() and (whole[M + 3:] == 3.0).all()
