"""Microscaled 4-bit floating point (quantize_mx4, pack_mx4, dequant_mx4, gemm_mx4) against the definition in 64 bits.

Quantizer and dequantizer are exact: equal values, bit for bit.  Products of two elements are multiples of 1/4 up to 36 and
scales are powers of two, so only the sum rounds.  Its bound: a tensor-core step adds 64 products to the fp32 accumulator and may
drop what lies below 2^-23 of the largest addend, twice (products among themselves, then with the accumulator), which is at most
2 * 2^-23 of the sum of magnitudes S per step; K split over up to 8 CTAs adds 8 fp32 additions of 2^-24 S:
|y - exact| <= (2 ceil(K / 64) 2^-23 + 8 * 2^-24) S, then half a step of the output's type."""
import numpy as np
import pytest
import torch

import qwengine_b200 as q
from qwengine_b200 import api

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
KIND = {"f32": 0, "f16": 1, "bf16": 2}


def mx_values(x):
    """The definition: x float64 [rows, K] -> the values its codes and scales stand for, and the scale exponents."""
    b = x.reshape(x.shape[0], -1, 32)
    top = np.abs(b).max(-1, keepdims=True)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.where(top > 0, np.frexp(np.where(np.isfinite(top), top, 1.0))[1] - 1, -200) - 2
    e = np.maximum(e, -127)
    p = np.ldexp(1.0, e)
    with np.errstate(invalid="ignore"):
        a = np.abs(b / p)
        step = np.where(a < 2, 0.5, np.where(a < 4, 1.0, 2.0))
        v = np.copysign(np.minimum(np.round(a / step) * step, 6.0), b) * p
    v = np.where(np.isfinite(top), v, np.nan)
    return v.reshape(x.shape), e[..., 0]


def bound(xv, wv, K, out):
    S = np.abs(xv) @ np.abs(wv).T
    return (2 * -(-K // 64) * 2.0 ** -23 + 8 * 2.0 ** -24) * S


def check_product(y, xv, wv, K, kind):
    exact = xv @ wv.T
    y = y.double().cpu().numpy()
    tol = bound(xv, wv, K, kind)
    half = torch.finfo(DTYPES[kind]).eps / 2
    tol = tol + (half * (np.abs(exact) + tol) + torch.finfo(DTYPES[kind]).smallest_normal * half * 2 if kind != "f32" else 0)
    bad = np.abs(y - exact) > tol
    assert not bad.any(), (np.argwhere(bad)[:4], np.abs(y - exact).max(), tol.max())


def rand(rows, K, seed, dtype="f32", spread=1.0):
    g = np.random.default_rng(seed)
    x = g.standard_normal((rows, K)) * np.exp(spread * g.standard_normal((rows, 1)))
    return torch.from_numpy(x.astype(np.float32)).to(DTYPES[dtype])


@pytest.mark.parametrize("rows,K", [(1, 32), (1, 5120), (3, 96), (129, 160), (77, 5120), (128, 128), (300, 1056)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_rows_to_mx4_and_back(ctx, rows, K, dtype):
    x = rand(rows, K, rows + K, dtype)
    want, e = mx_values(x.double().numpy())
    m = ctx.quantize_mx4(x.cuda())
    got = ctx.dequant_mx4(m)
    assert np.array_equal(got.double().cpu().numpy(), want)
    tiles = m.scales.cpu().numpy().reshape(-(-rows // 128), -(-K // 128), 32, 4, 4)   # [i][j][r % 32][r / 32][b]
    plain = tiles.transpose(0, 3, 2, 1, 4).reshape(-(-rows // 128) * 128, -1)
    assert np.array_equal(plain[:rows, :K // 32], (e + 127).astype(np.uint8))
    assert not plain[rows:].any() and not plain[:, K // 32:].any()
    for kind in ("f16", "bf16"):
        assert torch.equal(ctx.dequant_mx4(m, KIND[kind]), got.to(DTYPES[kind]))


def test_quantizer_at_its_edges(ctx):
    """Every tie, saturation, zeros of both signs, subnormal blocks, the largest floats, NaN and infinity."""
    K = 32 * 12
    x = np.zeros((2, K), np.float32)
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.2500001, 0.7499999, 1.2500001, 2.4999998, 3.5000002, 4.9999995, 5.0000005, 6.0, 7.9999995], np.float32)
    x[0, :16], x[0, 16:32] = ties, -ties
    x[0, 32:48], x[0, 48:64] = ties * 2.0 ** 60, -ties * 2.0 ** -60
    x[0, 64:96] = -0.0
    x[0, 96:128] = np.float32(2.0) ** -np.arange(118, 150)                 # down through the subnormals
    x[0, 128:160] = np.ldexp(np.float32(1.0), -149) * np.arange(32)        # nothing but subnormals
    x[0, 160:192] = np.finfo(np.float32).max * np.linspace(-1, 1, 32, dtype=np.float32)
    x[0, 192:224] = 1.0
    x[0, 200] = np.nan
    x[0, 224:256] = 2.0
    x[0, 231] = -np.inf
    x[0, 256] = 1.0                                                         # a block of one value
    x[1] = np.random.default_rng(1).standard_normal(K)
    want, _ = mx_values(x.astype(np.float64))
    m = ctx.quantize_mx4(torch.from_numpy(x).cuda())
    got = ctx.dequant_mx4(m).cpu().numpy()
    assert np.array_equal(got.astype(np.float64), want, equal_nan=True)
    assert np.isnan(got[0, 192:256]).all() and np.isfinite(got[0, :192]).all()


@pytest.mark.parametrize("ld,off", [(200, 0), (201, 0), (201, 3), (164, 4)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_quantizer_takes_any_row_stride_and_offset(ctx, ld, off, dtype):
    flat = rand(1, 7 * ld + off, 5, dtype)[0].cuda()
    x = flat[off:].as_strided((7, 160), (ld, 1), flat.storage_offset() + off)
    assert torch.equal(ctx.dequant_mx4(ctx.quantize_mx4(x)), ctx.dequant_mx4(ctx.quantize_mx4(x.contiguous())))


def test_other_producers_scales_and_strided_codes(ctx):
    rows, K = 200, 288
    x = rand(rows, K, 8).cuda()
    m = ctx.quantize_mx4(x)
    _, e = mx_values(x.double().cpu().numpy())
    scales = torch.full((rows, K // 32 + 3), 7, dtype=torch.uint8, device="cuda")
    scales[:, :K // 32] = torch.from_numpy((e + 127).astype(np.uint8)).cuda()
    wide = torch.full((rows, K // 2 + 16), 0x77, dtype=torch.uint8, device="cuda")
    wide[:, :K // 2] = m.codes
    p = ctx.pack_mx4(wide[:, :K // 2], scales[:, :K // 32])
    assert torch.equal(p.scales, m.scales)
    assert torch.equal(ctx.dequant_mx4(p), ctx.dequant_mx4(m))
    assert torch.equal(ctx.gemm_mx4(p, p), ctx.gemm_mx4(m, m))


SHAPES = [(1, 128, 256), (1, 1, 32), (2, 5, 64), (1, 640, 2560), (7, 300, 1056), (16, 129, 96), (17, 128, 4096), (33, 257, 288), (128, 384, 512), (129, 130, 320),
          (255, 64, 160), (256, 256, 1024), (257, 200, 1024), (300, 1000, 736), (513, 136, 2048), (1, 1280, 17408)]


@pytest.mark.parametrize("B,M,K", SHAPES)
def test_product(ctx, B, M, K):
    x, w = rand(B, K, B + K), rand(M, K, M + K + 1, "bf16")
    xv, wv = mx_values(x.double().numpy())[0], mx_values(w.double().numpy())[0]
    W = ctx.quantize_mx4(w.cuda())
    X = ctx.quantize_mx4(x.cuda())
    y = ctx.gemm_mx4(W, X)
    ctx.check()
    check_product(y, xv, wv, K, "f32")
    assert torch.equal(y, ctx.gemm_mx4(W, x.cuda())), "quantized within the call"
    assert torch.equal(y, ctx.gemm_mx4(W, X)), "the same bits again"
    for kind in ("f16", "bf16"):
        check_product(ctx.gemm_mx4(W, X, kind=KIND[kind]), xv, wv, K, kind)
        assert torch.equal(ctx.gemm_mx4(W, x.to(DTYPES[kind]).cuda()), ctx.gemm_mx4(W, ctx.quantize_mx4(x.to(DTYPES[kind]).cuda())))
    ctx.check()


@pytest.mark.parametrize("tile", [64, 128, 192, 256])
@pytest.mark.parametrize("B,M,K", [(1, 1, 32), (5, 130, 96), (200, 257, 352), (65, 300, 2080), (449, 700, 1024), (130, 136, 64), (1030, 256, 288)])
def test_products_in_pairs_of_every_tile(ctx, B, M, K, tile):
    """Tiles that start on half a scale tile, a last tile of any length, one K tile in the last stage, more tiles than pairs below."""
    x, w = rand(B, K, B + K), rand(M, K, M + K + 1)
    xv, wv = mx_values(x.double().numpy())[0], mx_values(w.double().numpy())[0]
    W, X = ctx.quantize_mx4(w.cuda()), ctx.quantize_mx4(x.cuda())
    try:
        ctx.debug_set_mx4_pairs(tile)
        for kind, left, wide in (("f32", 2, M + 5), ("bf16", 2, M + 5), ("f32", 4, (M + 15) // 8 * 8), ("bf16", 8, (M + 23) // 8 * 8)):   # plain stores, TMA stores
            whole = torch.full((B + 2, wide), 3.0, dtype=DTYPES[kind], device="cuda")
            out = whole[1:B + 1, left:M + left]
            ctx.gemm_mx4(W, X, out=out)
            ctx.check()
            check_product(out, xv, wv, K, kind)
            keep = out.clone()
            ctx.gemm_mx4(W, X, out=out, accumulate=True)
            assert torch.equal(out, (keep.float() + ctx.gemm_mx4(W, X)).to(DTYPES[kind]))
            out.fill_(3.0)
            assert (whole == 3.0).all()
    finally:
        ctx.debug_set_mx4_pairs(0)


@pytest.mark.parametrize("tile", [64, 128, 192, 256])
def test_a_pair_walks_many_tiles(ctx, tile):
    B, M, K = 1500, 4000, 544                     # 16 x 6 .. 24 tiles for 74 pairs, whole-number sums
    g = np.random.default_rng(tile)
    x, w = (torch.from_numpy(g.choice([0.0, 1, -1, 2, -2, 4, -4], (n, K)).astype(np.float32)).cuda() for n in (B, M))
    x[:, ::32], w[:, ::32] = 4, -4
    W, X = ctx.quantize_mx4(w), ctx.quantize_mx4(x)
    try:
        ctx.debug_set_mx4_pairs(tile)
        y = ctx.gemm_mx4(W, X)
        ctx.check()
    finally:
        ctx.debug_set_mx4_pairs(0)
    assert torch.equal(y.double(), x.double() @ w.double().t())


@pytest.mark.parametrize("B,M,K", [(1, 200, 4096), (9, 130, 992), (300, 260, 512)])
def test_whole_number_products_are_exact(ctx, B, M, K):
    """Elements 0, +-1, +-2, +-4 (and one 4 a block, so that every scale is 1): sums are whole numbers below 2^24, which fp32 holds."""
    g = np.random.default_rng(B)
    x, w = (g.choice([0.0, 1, -1, 2, -2, 4, -4], (n, K)).astype(np.float32) for n in (B, M))
    x[:, ::32], w[:, ::32] = 4, -4
    y = ctx.gemm_mx4(ctx.quantize_mx4(torch.from_numpy(w).cuda()), torch.from_numpy(x).cuda())
    assert np.array_equal(y.double().cpu().numpy(), x.astype(np.float64) @ w.astype(np.float64).T)


def test_every_block_has_its_own_scale(ctx):
    """One block of one row apart from zero at a time: its scale reaches its own products only."""
    K, M, B = 512, 160, 40
    x, w = np.zeros((B, K), np.float32), np.zeros((M, K), np.float32)
    g = np.random.default_rng(3)
    for r in range(M):
        w[r, 32 * (r % 16):32 * (r % 16) + 32] = 2.0 ** (r % 23 - 11)
    for t in range(B):
        x[t] = np.repeat(2.0 ** g.integers(-9, 9, 16), 32)
    y = ctx.gemm_mx4(ctx.quantize_mx4(torch.from_numpy(w).cuda()), torch.from_numpy(x).cuda())
    assert np.array_equal(y.double().cpu().numpy(), x.astype(np.float64) @ w.astype(np.float64).T)


def test_product_adds_to_what_is_there_and_writes_no_more(ctx):
    B, M, K = 19, 150, 352
    x, w = rand(B, K, 1), rand(M, K, 2)
    W, X = ctx.quantize_mx4(w.cuda()), ctx.quantize_mx4(x.cuda())
    for kind in ("f32", "bf16"):
        whole = torch.full((B + 2, M + 9), 3.0, dtype=DTYPES[kind], device="cuda")
        out = whole[1:B + 1, 4:M + 4]
        ctx.gemm_mx4(W, X, out=out, accumulate=True)
        plain = ctx.gemm_mx4(W, X)
        assert torch.equal(out, (plain + 3.0).to(DTYPES[kind]))
        ctx.gemm_mx4(W, X, out=out)
        assert torch.equal(out, plain.to(DTYPES[kind]))
        whole[1:B + 1, 4:M + 4] = 3.0
        assert (whole == 3.0).all()


@pytest.mark.parametrize("B,M,K", [(1, 128, 256), (1, 200, 32), (3, 129, 96), (1, 300, 5120), (7, 640, 2080), (1, 1000, 8192), (1, 128, 8224), (1, 18000, 8224), (1, 256, 17408), (1, 70, 992)])
@pytest.mark.parametrize("dtype,pad", [("f32", 0), ("bf16", 0), ("f16", 3)])
def test_few_tokens_are_quantized_by_the_product(ctx, B, M, K, dtype, pad):
    """One launch or two, with blocks of NaN and zeros, any row stride: the same bits."""
    x = torch.randn((B, K + pad), generator=torch.Generator().manual_seed(K + B)).to(DTYPES[dtype]).cuda()[:, :K]
    x[0, 0:32] = 0
    if B > 2:
        x[2, K - 1] = float("nan")
    W = ctx.quantize_mx4(rand(M, K, 7).cuda())
    one = ctx.gemm_mx4(W, x)
    try:
        ctx.lib.q38b_debug_set_mx4_two_launches(ctx.h, 1)
        scratch = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
        two = torch.empty_like(one)
        assert ctx.lib.q38b_gemm_mx4_x(ctx.h, W.codes.data_ptr(), W.ld, W.scales.data_ptr(), K, M, x.data_ptr(), KIND[dtype], K + pad, B, two.data_ptr(), 0, M, 0,
                                       scratch.data_ptr(), scratch.numel(), ctx._stream()) == 0
    finally:
        ctx.lib.q38b_debug_set_mx4_two_launches(ctx.h, 0)
    ctx.check()
    assert torch.equal(one.view(torch.int32), two.view(torch.int32)) and torch.equal(torch.isnan(one).all(1).cpu(), torch.arange(B) == 2)
    assert torch.equal(one.nan_to_num(), ctx.gemm_mx4(W, ctx.quantize_mx4(x)).nan_to_num())


@pytest.mark.parametrize("B,M,K", [
    (1, 19100, 1280), (1, 30000, 96), (2, 19100, 1280), (16, 25000, 1056), (32, 19100, 2080),   # two CTAs to an SM, one part
    (1, 9700, 2560), (9, 9700, 2304), (7, 5120, 6144), (32, 5000, 6176),                        # ... two and six parts
    (129, 1024, 5120), (300, 1000, 5152), (513, 1024, 2304), (256, 640, 4000),                  # tiles of 128 tokens in parts
    (3, 70000, 512), (32, 70001, 288)])                                                         # many rows
def test_whole_number_products_in_every_cut(ctx, B, M, K):
    """Sums of whole numbers below 2^24: exact whatever the parts, tiles and kernels; the quantizer inside gives the same, and what lies around stays."""
    gen = torch.Generator("cuda").manual_seed(B + M + K)
    x, w = (torch.randint(-4, 5, (n, K), generator=gen, device="cuda").float() for n in (B, M))
    x[:, ::32], w[:, ::32] = 4, -4                # every block scaled by one: whole numbers up to 4 are E2M1 values
    whole = torch.full((B + 2, M + 6), 3.0, device="cuda")
    y = whole[1:B + 1, 3:M + 3]
    W = ctx.quantize_mx4(w)
    ctx.gemm_mx4(W, ctx.quantize_mx4(x), out=y)
    ctx.check()
    assert torch.equal(y, (x.double() @ w.double().t()).float())
    assert torch.equal(y, ctx.gemm_mx4(W, x))
    ctx.check()
    y.fill_(3.0)
    assert (whole == 3.0).all()


def test_products_on_two_streams_at_once(ctx):
    """CTAs that share SMs, of one stream's few tokens and the other's many."""
    w, v = rand(5120, 6144, 1, "bf16").cuda(), rand(19100, 1280, 2, "bf16").cuda()
    W, V = ctx.quantize_mx4(w), ctx.quantize_mx4(v)
    a, b, c = rand(7, 6144, 3).cuda(), rand(1, 1280, 4).cuda(), rand(400, 1280, 5).cuda()
    want = [ctx.gemm_mx4(W, a), ctx.gemm_mx4(V, b), ctx.gemm_mx4(V, c)]
    torch.cuda.synchronize()
    sides, got = [torch.cuda.Stream() for _ in range(3)], [[], [], []]
    for _ in range(10):
        for i, (m, t) in enumerate(((W, a), (V, b), (V, c))):
            with torch.cuda.stream(sides[i]):
                got[i].append(ctx.gemm_mx4(m, t))
    torch.cuda.synchronize()
    ctx.check()
    for i in range(3):
        for y in got[i]:
            assert torch.equal(y, want[i])


def test_nan_block_reaches_its_row_and_column_only(ctx):
    B, M, K = 20, 140, 256
    x, w = rand(B, K, 1), rand(M, K, 2)
    x[3, 70], w[131, 5] = float("nan"), float("inf")
    y = ctx.gemm_mx4(ctx.quantize_mx4(w.cuda()), x.cuda()).cpu()
    bad = torch.isnan(y)
    assert bad[3].all() and bad[:, 131].all()
    bad[3], bad[:, 131] = False, False
    assert not bad.any()


def test_product_on_a_side_stream_in_a_graph(ctx):
    B, M, K = 5, 300, 2048
    W = ctx.quantize_mx4(rand(M, K, 1).cuda())
    x = rand(B, K, 2).cuda()
    out = torch.empty((B, M), device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ctx.gemm_mx4(W, x, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ctx.gemm_mx4(W, x, out=out)
    for seed in (3, 4):
        x.copy_(rand(B, K, seed))
        graph.replay()
        assert torch.equal(out, ctx.gemm_mx4(W, ctx.quantize_mx4(x)))
    ctx.check()


def test_refusals(ctx):
    W = ctx.quantize_mx4(rand(64, 256, 1).cuda())
    x = rand(3, 256, 2).cuda()
    for bad in (lambda: ctx.quantize_mx4(x.double()), lambda: ctx.quantize_mx4(x.t()), lambda: ctx.quantize_mx4(x.cpu()),
                lambda: ctx.gemm_mx4(W, x[:, :224]), lambda: ctx.gemm_mx4(W, x, out=torch.empty((3, 63), device="cuda")),
                lambda: ctx.gemm_mx4(W, x.int()), lambda: q.Mx4(W.codes, W.scales[:-1]), lambda: q.Mx4(W.codes[:, :40], W.scales)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(api.Q38BError):
        ctx.quantize_mx4(x[:, :250])          # K no multiple of 32
    with pytest.raises(api.Q38BError):
        ctx.gemm_mx4(q.Mx4(W.codes.flatten()[8:8 + 63 * 128].view(63, 128), W.scales), x)   # codes off their 16 bytes
    ctx.check()
