"""The new operators where offsets pass 32 bits, and called on two streams at once."""
import pytest
import torch

import qwengine_b200 as q   # noqa: F401

pytestmark = pytest.mark.gpu

FAR = 1 << 30      # elements between rows: the third begins at 2^31


@pytest.fixture
def flat(request):
    t = torch.empty(2 * FAR + 50000, dtype=request.param, device="cuda")
    yield t
    del t
    torch.cuda.empty_cache()


def normal(*shape, dtype=torch.float32, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.mark.parametrize("flat", [torch.bfloat16], indirect=True)
def test_heads(ctx, flat):
    x = flat.as_strided((3, 4, 128), (FAR, 256, 1))
    x.copy_(normal(3, 4, 128, dtype=torch.bfloat16))
    pos, f = torch.arange(3, dtype=torch.int32, device="cuda"), 1e4 ** (-torch.arange(0, 64, 2, dtype=torch.float64, device="cuda") / 64)
    want = ctx.qk_norm_rope(x.contiguous(), None, pos, f)[0]
    assert torch.equal(ctx.qk_norm_rope(x, None, pos, f)[0], want)
    ctx.qk_norm_rope(x, None, pos, f, q_out=x)
    assert torch.equal(x, want)


@pytest.mark.parametrize("flat", [torch.float32], indirect=True)
def test_logits(ctx, flat):
    x = flat.as_strided((3, 5003), (FAR, 1))
    x.copy_(normal(3, 5003))
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")   # noqa: E731
    rules = dict(penalties=torch.tensor([[1.5, 0.2, 0.1]] * 3, device="cuda"), history=i32(5, 5, 7, 9, 9, 5002), history_begin=torch.tensor([0, 2, 4, 6], device="cuda"), prompt_len=i32(1, 0, 1))
    want = ctx.adjust_logits(x.contiguous(), **rules)
    assert torch.equal(ctx.adjust_logits(x, **rules), want)
    ctx.adjust_logits(x, out=x, **rules)
    assert torch.equal(x, want)


@pytest.mark.parametrize("flat", [torch.float32], indirect=True)
def test_microscaled(ctx, flat):
    x = flat.as_strided((3, 512), (FAR, 1))
    x.copy_(normal(3, 512))
    X = ctx.quantize_mx4(x)
    assert torch.equal(X.codes, ctx.quantize_mx4(x.contiguous()).codes)
    for M in (70, 300):
        W = ctx.quantize_mx4(normal(M, 512, seed=M))
        want = ctx.gemm_mx4(W, X)
        assert torch.equal(ctx.gemm_mx4(W, x), want)
        y = flat.as_strided((3, M), (FAR, 1), 1000)
        ctx.gemm_mx4(W, X, out=y)
        assert torch.equal(y, want)
    try:                                                  # the tiled kernel of many tokens, with TMA stores
        ctx.debug_set_mx4_pairs(64)
        y = flat.as_strided((3, 300), (FAR, 1), 1000)
        y.zero_()
        ctx.gemm_mx4(W, X, out=y)
        ctx.check()
        assert torch.allclose(y, want, rtol=0, atol=1e-4)
    finally:
        ctx.debug_set_mx4_pairs(0)


def test_two_streams_at_once(ctx):
    """None of these calls has a work area in the context: whatever overlaps, each gives its own result."""
    W = [ctx.quantize_mx4(normal(M, K, seed=M)) for M, K in ((640, 4096), (3000, 1024))]
    xs = [normal(1, 4096, seed=1), normal(300, 1024, seed=2)]
    logits = [normal(2, 30000, seed=3), normal(9, 5001, seed=4)]
    mask = torch.randint(-2 ** 31, 2 ** 31, (9, 1000), device="cuda").to(torch.int32)
    heads = [normal(2, 8, 256, seed=5), normal(70, 3, 96, seed=6)]
    pos, f = torch.arange(70, dtype=torch.int32, device="cuda"), 1e4 ** (-torch.arange(0, 64, 2, dtype=torch.float64, device="cuda") / 64)

    def run(i):
        h = heads[i]
        return (ctx.gemm_mx4(W[i], xs[i]), ctx.adjust_logits(logits[i], masks=mask), ctx.qk_norm_rope(h, None, pos[:h.shape[0]], f)[0], ctx.dequant_mx4(ctx.quantize_mx4(xs[i])))

    want = [run(0), run(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i].append(run(i))
    torch.cuda.synchronize()
    ctx.check()
    for i in (0, 1):
        for r in got[i]:
            assert all(torch.equal(a.view(torch.int32), b.view(torch.int32)) for a, b in zip(r, want[i]))
