"""8-bit integers with one scale a row (quantize_i8, gemm_i8) against the definition in 64 bits.

Codes are exact, and scales are one division rounded once: equal, bit for bit.  Sums are whole numbers below 2^31: exact.  A result then rounds three times in
fp32 (the sum to fp32, times either scale: half a step of 2^-24 each, 3.01 * 2^-24 together), accumulating rounds the sum with the old value once
more (2^-24 of it), then half a step of the output's type, or half of its smallest step where it is subnormal."""
import numpy as np
import pytest
import torch

import qwengine_b200 as q
from qwengine_b200 import api

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
KIND = {"f32": 0, "f16": 1, "bf16": 2}
TINY = 2.0 ** -126


def definition(x):
    """x float64 [rows, K] -> codes (int64) and scales (float32)."""
    top = np.abs(x).max(-1)
    with np.errstate(invalid="ignore"):
        scale = np.where(np.isfinite(top), np.maximum((top / 127).astype(np.float32), np.float32(TINY)), np.float32(np.nan)).astype(np.float32)
        code = np.where(np.isfinite(scale)[:, None], np.round(x / scale.astype(np.float64)[:, None]), 0.0)
    return code.astype(np.int64), scale


def half_step(kind, value):
    f = torch.finfo(DTYPES[kind])
    return f.eps / 2 * np.maximum(np.abs(value), f.smallest_normal)


def check_product(y, xc, xs, wc, ws, kind, before=None):
    exact = (xc @ wc.T) * xs.astype(np.float64)[:, None] * ws.astype(np.float64)[None]
    tol = 3.01 * 2.0 ** -24 * np.abs(exact)
    if before is not None:
        exact = exact + before
        tol = tol + 2.0 ** -24 * (np.abs(exact) + tol)
    if kind != "f32":
        tol = tol + half_step(kind, np.abs(exact) + tol)
    got = y.double().cpu().numpy()
    # rounding to the type gives an infinity from half a step past its largest number on (eps / 4 of it, or a little more)
    edge = torch.finfo(DTYPES[kind]).max * (1 + torch.finfo(DTYPES[kind]).eps / 4)
    infinite = np.isinf(got) & (np.sign(got) == np.sign(exact)) & (np.abs(exact) + tol >= edge)
    bad = ~infinite & ~(np.abs(got - exact) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], exact[bad][:4])


def rand(rows, K, seed, dtype="f32", spread=1.0):
    g = np.random.default_rng(seed)
    x = g.standard_normal((rows, K)) * np.exp(spread * g.standard_normal((rows, 1)))
    return torch.from_numpy(x.astype(np.float32)).to(DTYPES[dtype])


@pytest.mark.parametrize("rows,K", [(1, 1), (1, 5120), (3, 17), (2, 8193), (129, 160), (77, 5120), (300, 1000), (2, 131071)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_codes_and_scales(ctx, rows, K, dtype):
    x = rand(rows, K, rows + K, dtype)
    codes, scales = definition(x.double().numpy())
    m = ctx.quantize_i8(x.cuda())
    assert m.rows == rows and m.K == K and m.ld % 16 == 0
    assert np.array_equal(m.codes.cpu().numpy(), codes) and np.array_equal(m.scales.cpu().numpy(), scales)


def test_halves_extremes_and_what_is_no_number(ctx):
    K = 600
    g = np.random.default_rng(4)
    x = np.zeros((14, K), np.float32)
    halves = np.arange(-127, 127) + 0.5
    x[0, :254], x[0, 254] = halves, 127                                    # scale 1: every tie
    x[1, :254], x[1, 254] = np.nextafter(halves.astype(np.float32), np.float32(np.inf)), 127
    x[2, :254], x[2, 254] = np.nextafter(halves.astype(np.float32), np.float32(-np.inf)), 127
    scale = np.float32(np.float32(3.3) / 127)                               # ties of a scale that is no power of two, and their neighbours
    near = (halves * np.float64(scale)).astype(np.float32)
    x[3, :254], x[3, 254] = near, 3.3
    x[4, :254], x[4, 254] = np.nextafter(near, np.float32(np.inf)), 3.3
    x[5, :254], x[5, 254] = np.nextafter(near, np.float32(-np.inf)), 3.3
    x[6, :3] = [3.4028235e38, -3.4028235e38, 1e38]
    x[7, :4] = [1e-45, -1e-45, 3e-39, -1e-38]                               # below the least scale
    x[8, :5] = [TINY * 127, TINY * 0.5, TINY * 1.5, -TINY * 2.5, TINY * 126.5]
    x[9, 5] = np.nan
    x[10, 5], x[10, 6] = np.inf, np.nan
    x[11, 599] = -np.inf
    x[13] = g.standard_normal(K) * 1e-30                                    # row 12: zeros
    codes, scales = definition(x.astype(np.float64))
    m = ctx.quantize_i8(torch.from_numpy(x).cuda())
    assert np.array_equal(m.scales.cpu().numpy(), scales, equal_nan=True)
    assert np.array_equal(m.codes.cpu().numpy(), codes)


def test_rows_of_any_stride_and_alignment(ctx):
    base = rand(40, 1111, 9)
    for dtype in DTYPES:
        for off, width in ((0, 1111), (1, 1000), (3, 801), (8, 160)):
            v = base.to(DTYPES[dtype]).cuda()[:, off:off + width]
            codes, scales = definition(v.double().cpu().numpy())
            m = ctx.quantize_i8(v[::3])
            assert np.array_equal(m.codes.cpu().numpy(), codes[::3]) and np.array_equal(m.scales.cpu().numpy(), scales[::3])


def test_bytes_behind_a_row_stay(ctx):
    x = rand(5, 37, 3).cuda()
    codes, scales = torch.full((5, 64), 77, dtype=torch.int8, device="cuda"), torch.zeros(5, device="cuda")
    assert ctx.lib.q38b_quantize_i8(ctx.h, x.data_ptr(), 0, 37, 37, 5, codes.data_ptr(), 64, scales.data_ptr(), None) == 0
    assert bool((codes[:, 37:] == 77).all()) and np.array_equal(codes[:, :37].cpu().numpy(), definition(x.double().cpu().numpy())[0])


SHAPES = [(1, 1, 1), (1, 128, 256), (1, 1000, 5120), (2, 130, 17), (5, 33, 1000), (7, 300, 4099), (16, 257, 640), (17, 128, 32), (33, 640, 2048), (64, 513, 96), (77, 384, 1029), (129, 1000, 512),
          (200, 96, 5120), (256, 300, 300), (257, 256, 1280), (333, 520, 777), (1000, 600, 384)]


@pytest.mark.parametrize("B,M,K", SHAPES)
@pytest.mark.parametrize("src,dst", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16")])
def test_products(ctx, B, M, K, src, dst):
    x, w = rand(B, K, B + 7 * K, src), rand(M, K, M + K, "f32")
    W = ctx.quantize_i8(w.cuda())
    y = ctx.gemm_i8(W, x.cuda(), kind=KIND[dst])
    xc, xs = definition(x.double().numpy())
    wc, ws = definition(w.double().numpy())
    check_product(y, xc, xs, wc, ws, dst)
    X = ctx.quantize_i8(x.cuda())
    assert torch.equal(ctx.gemm_i8(W, X, kind=KIND[dst]), y), "one call and two"
    ctx.check()


def codes(rows, K, seed, room=0):
    """Every code, -128 among them, behind each row whatever (which no product may take up)."""
    g = torch.Generator().manual_seed(seed)
    ld = (K + 15) // 16 * 16 + room
    whole = torch.randint(-128, 128, (rows, ld), generator=g, dtype=torch.int8)
    return whole[:, :K], (torch.rand(rows, generator=g) + 0.5) * 0.01


@pytest.mark.parametrize("B,M,K", [(1, 200, 5121), (3, 129, 100), (70, 300, 1000), (300, 515, 2050), (1, 64, 131071), (40, 70, 131071)])
def test_any_codes(ctx, B, M, K):
    (xc, xs), (wc, ws) = codes(B, K, 1, 16), codes(M, K, 2, 32)
    if K > 100000:
        xc[0], wc[0] = -128, -128        # the largest sum there is: 131071 * 2^14
        wc[-1] = 127
    def dev(c, s):
        room = torch.empty((c.shape[0], c.stride(0)), dtype=torch.int8, device="cuda").random_(-128, 128)
        room[:, :c.shape[1]] = c.cuda()
        return q.I8(room[:, :c.shape[1]], s.cuda())

    X, W = dev(xc, xs), dev(wc, ws)
    y = ctx.gemm_i8(W, X)
    check_product(y, xc.numpy().astype(np.int64), xs.numpy(), wc.numpy().astype(np.int64), ws.numpy(), "f32")


@pytest.mark.parametrize("B,M,K", [(1, 300, 512), (9, 200, 700), (150, 400, 384), (600, 512, 256)])
@pytest.mark.parametrize("dst", ["f32", "bf16", "f16"])
def test_accumulates_into_strided_outputs(ctx, B, M, K, dst):
    (xc, xs), (wc, ws) = codes(B, K, 5), codes(M, K, 6)
    for width, off in ((M + 24, 8), (M + 5, 3)):
        big = torch.randn((B + 2, width), device="cuda").to(DTYPES[dst])
        keep = big.clone()
        out = big[1:B + 1, off:off + M]
        before = out.double().cpu().numpy()
        W, X = ctx.quantize_i8(wc.float().cuda()), ctx.quantize_i8(xc.float().cuda())
        got = ctx.gemm_i8(W, X, out=out, accumulate=True)
        assert got is out
        a, b = definition(xc.double().numpy()), definition(wc.double().numpy())
        check_product(out, *a, *b, dst, before)
        keep[1:B + 1, off:off + M] = out
        assert torch.equal(big, keep), "nothing beside the outputs"


def test_a_token_that_is_no_number_spoils_its_own_row_only(ctx):
    x = rand(6, 320, 1)
    x[2, 100] = float("inf")
    W = ctx.quantize_i8(rand(200, 320, 2).cuda())
    y = ctx.gemm_i8(W, x.cuda())
    assert bool(y[2].isnan().all()) and bool(y[[0, 1, 3, 4, 5]].isfinite().all())


def test_same_bits_whatever_runs_beside(ctx):
    """Two streams at once, and a captured graph replayed on other inputs."""
    x1, x2 = rand(40, 1024, 1).cuda(), rand(40, 1024, 2).cuda()
    W = ctx.quantize_i8(rand(700, 1024, 3).cuda())
    want1, want2 = ctx.gemm_i8(W, x1), ctx.gemm_i8(W, x2)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(20):
        with torch.cuda.stream(a):
            y1 = ctx.gemm_i8(W, x1)
        with torch.cuda.stream(b):
            y2 = ctx.gemm_i8(W, x2)
        torch.cuda.synchronize()
        assert torch.equal(y1, want1) and torch.equal(y2, want2)
    held = x1.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ctx.gemm_i8(W, held)
    held.copy_(x2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want2)
    ctx.check()


def test_wrapper_refusals(ctx):
    W = ctx.quantize_i8(torch.randn((64, 64), device="cuda"))
    for bad in (lambda: ctx.gemm_i8(W, torch.randn((2, 65), device="cuda")), lambda: ctx.gemm_i8(W, torch.randn((2, 64), device="cuda").double()), lambda: ctx.gemm_i8(W, torch.randn((2, 64))),
                lambda: ctx.gemm_i8(W, torch.randn((2, 64), device="cuda"), accumulate=True), lambda: ctx.gemm_i8(W, torch.randn((2, 64), device="cuda"), out=torch.empty((2, 63), device="cuda")),
                lambda: ctx.gemm_i8(W, torch.randn((0, 64), device="cuda")), lambda: ctx.quantize_i8(torch.randn((2, 64))), lambda: ctx.quantize_i8(torch.randn((64, 2), device="cuda").t()),
                lambda: q.I8(W.codes[:, ::2], W.scales), lambda: q.I8(W.codes.float(), W.scales), lambda: q.I8(W.codes, W.scales[:5]),
                lambda: q.I8(torch.zeros((3, 20), dtype=torch.int8, device="cuda"), torch.zeros(3, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: ctx.quantize_i8(torch.empty((0, 64), device="cuda")), lambda: ctx.quantize_i8(torch.empty((1, 131072), device="cuda"))):
        with pytest.raises(api.Q38BError):
            bad()


@pytest.mark.parametrize("mode", [64, 128, 192, 256, -10, -20, -1, -2, -3, -4, -5, -6, -7, -8, -12, -22, -23, -25, -28])
def test_every_cut_gives_the_same_sums(ctx, mode):
    """Pairs of CTAs with every tile, single CTAs with K in every number of parts: exact sums, so the same bits."""
    for B, M, K in ((1, 700, 2000), (20, 300, 1300), (60, 130, 4096), (200, 513, 1111), (520, 256, 640)):
        if mode // 10 == -2 or -mode // 10 == 2:
            if B > 64:
                continue
        (xc, xs), (wc, ws) = codes(B, K, B), codes(M, K, M)
        X = ctx.quantize_i8(torch.zeros((B, K), device="cuda"))
        W = ctx.quantize_i8(torch.zeros((M, K), device="cuda"))
        X.codes.copy_(xc.cuda()), X.scales.copy_(xs.cuda()), W.codes.copy_(wc.cuda()), W.scales.copy_(ws.cuda())
        for kind in (0, 2):
            want = ctx.gemm_i8(W, X, kind=kind)
            room = torch.full((B, M + 3), 7.0, device="cuda", dtype=want.dtype)
            ctx.debug_set_i8_cut(mode)
            try:
                got = ctx.gemm_i8(W, X, kind=kind)
                ctx.gemm_i8(W, X, out=room[:, 1:M + 1])
            finally:
                ctx.debug_set_i8_cut(0)
            ctx.check()
            assert torch.equal(got, want) and torch.equal(room[:, 1:M + 1], want) and bool((room[:, 0] == 7).all()) and bool((room[:, M + 1:] == 7).all())
            if kind == 0:
                check_product(want, xc.numpy().astype(np.int64), xs.numpy(), wc.numpy().astype(np.int64), ws.numpy(), "f32")
