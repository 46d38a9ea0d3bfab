"""Norms and rotation of query and key heads (qk_norm_rope) against the formula in 64 bits.

Bound, in units u = 2^-24, for z_a c - z_b n and its partner: the sum of D squares, in chains of D / 32 and a tree of five, is off by at most
(D / 32 + 6) u, half of which reaches its root; mean, eps, rsqrtf (two steps) and two products: 8 u; cos and sin: the angle rounds to 24 bits of
half a turn, pi u / 2, and sincospif to two steps, 4 u together 6 u; products and difference 2 u.  So |y - exact| <=
(D / 64 + 19) u (|z_a| + |z_b|), and half a step of the output's type (its smallest step where it is subnormal)."""
import numpy as np
import pytest
import torch

import qwengine_b200 as q
from qwengine_b200 import api

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
KIND = {"f32": 0, "f16": 1, "bf16": 2}


def definition(x, w, pos, inv_freq, adjacent, eps, scale):
    """x float64 [rows, heads, D] -> y and |z_a| + |z_b| per element."""
    D, rot = x.shape[2], 2 * len(inv_freq)
    z = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (1.0 if w is None else w)
    y, mag = z.copy(), np.abs(z)
    if rot:
        a = (np.arange(0, rot, 2), np.arange(1, rot, 2)) if adjacent else (np.arange(rot // 2), np.arange(rot // 2, rot))
        angle = pos.astype(np.float64)[:, None, None] * inv_freq
        c, s = scale * np.cos(angle), scale * np.sin(angle)
        za, zb = z[..., a[0]], z[..., a[1]]
        y[..., a[0]], y[..., a[1]] = za * c - zb * s, zb * c + za * s
        mag[..., a[0]] = mag[..., a[1]] = scale * (np.abs(za) + np.abs(zb))
    return y, mag


def check(got, x, w, pos, inv_freq, adjacent=False, eps=1e-6, scale=1.0):
    want, mag = definition(x.double().cpu().numpy(), None if w is None else w.double().cpu().numpy(), pos.cpu().numpy(), inv_freq.cpu().numpy(), adjacent, eps, scale)
    tol = (x.shape[2] / 64 + 19) * 2.0 ** -24 * mag
    if got.dtype != torch.float32:
        info = torch.finfo(got.dtype)
        tol = tol + info.eps / 2 * np.maximum(np.abs(want) + tol, info.smallest_normal)
    bad = np.abs(got.double().cpu().numpy() - want) > tol
    assert not bad.any(), (np.argwhere(bad)[:4], np.abs(got.double().cpu().numpy() - want).max())


def inputs(rows, heads, D, seed, dtype="f32", src_head=None, pad=0):
    g = torch.Generator().manual_seed(seed)
    step = src_head or D
    x = torch.randn((rows, heads * step + pad), generator=g).mul_(torch.exp(0.5 * torch.randn((rows, 1), generator=g))).to(DTYPES[dtype]).cuda()
    return x[:, :heads * step].unflatten(1, (heads, step))[:, :, :D]


def freqs(rot, theta=1e7):
    return (theta ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)).cuda() if rot else torch.empty(0, dtype=torch.float64, device="cuda")


def places(rows, start):
    return torch.arange(start, start + rows, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("D,rot", [(256, 64), (256, 256), (128, 128), (64, 32), (96, 48), (80, 80), (192, 64), (2, 2), (1, 0), (33, 6), (66, 66), (510, 30), (1024, 1024)])
@pytest.mark.parametrize("adjacent", [False, True])
def test_head_sizes(ctx, D, rot, adjacent):
    x, y = inputs(5, 6, D, D + rot), inputs(5, 2, D, D + rot + 1)
    g = torch.Generator().manual_seed(1)
    wq, wk = (1 + 0.3 * torch.randn(D, generator=g)).cuda(), (1 + 0.3 * torch.randn(D, generator=g)).cuda()
    pos, f = places(5, 4097), freqs(rot)
    a, b = ctx.qk_norm_rope(x, y, pos, f, wq, wk, adjacent=adjacent)
    check(a, x, wq, pos, f, adjacent)
    check(b, y, wk, pos, f, adjacent)


@pytest.mark.parametrize("src,dst", [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "bf16"), ("f16", "f32"), ("bf16", "f16")])
@pytest.mark.parametrize("rows,D,rot", [(1, 256, 64), (7, 128, 128), (333, 96, 48)])
def test_types_and_rows(ctx, rows, D, rot, src, dst):
    x, y = inputs(rows, 8, D, rows, src, src_head=2 * D), inputs(rows, 2, D, rows + 1, src, pad=8)
    pos, f = places(rows, 100), freqs(rot)
    a, b = ctx.qk_norm_rope(x, y, pos, f, kind=KIND[dst])
    check(a, x, None, pos, f)
    check(b, y, None, pos, f)


@pytest.mark.parametrize("start", [0, 131071, 10 ** 6, 2 ** 31 - 5, -3, -2 ** 31])
def test_far_positions_keep_their_angle(ctx, start):
    """The first pair turns by a radian a position: 32-bit products lose the angle altogether far out."""
    x = inputs(4, 3, 64, 9)
    pos, f = places(4, start), freqs(64, 1e4)
    check(ctx.qk_norm_rope(x, None, pos, f)[0], x, None, pos, f)


def test_any_frequencies_scale_and_eps(ctx):
    x = inputs(6, 2, 128, 10)
    pos = torch.tensor([0, 5, 5, 1, 99999, 7], dtype=torch.int32, device="cuda")       # any order, the same one twice
    f = torch.tensor([0.0, -0.5, 3.75, 1e-12, 6.283185307179586, 100.0, -1e-300, 2.0 ** -60], dtype=torch.float64, device="cuda")
    check(ctx.qk_norm_rope(x, None, pos, f, scale=1.25, eps=0.5)[0], x, None, pos, f, scale=1.25, eps=0.5)


@pytest.mark.parametrize("off,pad,src_head", [(0, 0, 96), (1, 0, 97), (2, 6, 98), (4, 4, 100), (3, 1, 192)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides_and_offsets(ctx, off, pad, src_head, dtype):
    rows, heads, D = 9, 5, 96
    flat = inputs(1, 1, rows * (heads * src_head + pad) + off, 12, dtype).flatten()
    x = flat.as_strided((rows, heads, D), (heads * src_head + pad, src_head, 1), off)
    keep = torch.full((rows * (heads * src_head + pad) + off + 7,), 5.0, dtype=DTYPES[dtype], device="cuda")
    out = keep.as_strided((rows, heads, D), (heads * src_head + pad, src_head, 1), off)
    pos, f = places(rows, 77), freqs(48)
    ctx.qk_norm_rope(x, None, pos, f, adjacent=off % 2 == 1, q_out=out, kind=KIND[dtype])
    check(out, x, None, pos, f, adjacent=off % 2 == 1)
    out.fill_(5.0)
    assert (keep == 5.0).all()


def test_heads_outside_rows_inside(ctx):
    """[heads][rows][D] outputs, as a cache keeps them, from a source whose rows all are the same one."""
    x = inputs(1, 4, 128, 13).expand(6, 4, 128)
    cache = torch.zeros((4, 50, 128), dtype=torch.bfloat16, device="cuda")
    out = cache[:, 20:26].transpose(0, 1)
    pos, f = places(6, 20), freqs(128)
    ctx.qk_norm_rope(x, None, pos, f, q_out=out, kind=2)
    check(out, x, None, pos, f)
    assert not cache[:, :20].any() and not cache[:, 26:].any()


@pytest.mark.parametrize("dtype,D,rot,adjacent", [("f32", 256, 64, False), ("bf16", 128, 128, False), ("f16", 96, 96, True), ("f32", 66, 34, False)])
def test_in_place_gives_the_same(ctx, dtype, D, rot, adjacent):
    x, y = inputs(70, 6, D, 14, dtype, src_head=2 * D), inputs(70, 2, D, 15, dtype)
    pos, f = places(70, 3), freqs(rot)
    want = ctx.qk_norm_rope(x, y, pos, f, adjacent=adjacent)
    got = ctx.qk_norm_rope(x, y, pos, f, adjacent=adjacent, q_out=x, k_out=y)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and got[0] is x


def test_a_rows_results_do_not_depend_on_its_neighbours(ctx):
    x, y = inputs(300, 24, 256, 16, src_head=512), inputs(300, 4, 256, 17)
    pos, f = places(300, 1000), freqs(64)
    a, b = ctx.qk_norm_rope(x, y, pos, f, kind=2)
    for r in (0, 1, 150, 299):
        c, d = ctx.qk_norm_rope(x[r:r + 1], y[r:r + 1], pos[r:r + 1], f, kind=2)
        assert torch.equal(a[r:r + 1], c) and torch.equal(b[r:r + 1], d)


def test_zeros_infinities_and_nan_stay_in_their_head(ctx):
    x = inputs(3, 4, 64, 18).clone()
    x[0, 1] = 0.0
    x[1, 2, 5] = float("inf")
    x[2, 3, 63] = float("nan")
    out = ctx.qk_norm_rope(x, None, places(3, 9), freqs(64))[0].cpu()
    assert (out[0, 1] == 0).all()
    assert torch.isnan(out[1, 2, 5]) and torch.isnan(out[2, 3]).all()
    clean = torch.ones(3, 4, dtype=torch.bool)
    clean[1, 2] = clean[2, 3] = False
    assert torch.isfinite(out[clean]).all()


def test_on_a_side_stream_and_replayed(ctx):
    x, y = inputs(2, 24, 256, 19, src_head=512), inputs(2, 4, 256, 20)
    pos, f = places(2, 0), freqs(64)
    qo, ko = torch.empty((2, 24, 256), device="cuda"), torch.empty((2, 4, 256), device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ctx.qk_norm_rope(x, y, pos, f, q_out=qo, k_out=ko, kind=0)
    for start in (5, 70000):
        pos.copy_(places(2, start))
        graph.replay()
        check(qo, x, None, pos, f)
        check(ko, y, None, pos, f)


def test_refusals(ctx):
    x, pos, f = inputs(4, 2, 64, 21), places(4, 0), freqs(64)
    for bad in (lambda: ctx.qk_norm_rope(x.double(), None, pos, f), lambda: ctx.qk_norm_rope(x.transpose(1, 2), None, pos, f[:1]), lambda: ctx.qk_norm_rope(x, None, pos.long(), f),
                lambda: ctx.qk_norm_rope(x, None, pos[:3], f), lambda: ctx.qk_norm_rope(x, None, pos, f.float()), lambda: ctx.qk_norm_rope(x, None, pos, freqs(66)),
                lambda: ctx.qk_norm_rope(x, x[:3], pos, f), lambda: ctx.qk_norm_rope(x, x.half(), pos, f), lambda: ctx.qk_norm_rope(x, None, pos, f, q_weight=pos),
                lambda: ctx.qk_norm_rope(x, None, pos.cpu(), f), lambda: ctx.qk_norm_rope(x, None, pos, f, q_out=x, kind=2)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(api.Q38BError):      # rows of the destination that share elements
        ctx.qk_norm_rope(x, None, pos, f, q_out=torch.empty(128, device="cuda").as_strided((4, 2, 64), (0, 64, 1)))
    ctx.check()
