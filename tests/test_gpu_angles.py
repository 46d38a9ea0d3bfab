"""The cosines and sines that rotate the heads, read out bit for bit: elements that are all one have a norm of exactly one, weights of one and zero make
every pair (1, 0), and its rotation is (cos, sin) without another rounding.

Bound: the angle is cut off at 2^-32 turns; less its quadrant it is a whole number of them up to 2^29 in magnitude, which is rounded to a float and goes through
two Taylor polynomials.  That is a function of a number of 30 bits; over all of them, computed with the same roundings on the CPU, it is within 7.74e-8 of cosine
and sine (the second test looks at the ends of each quarter).  The frequency in turns and its fraction round in 64 bits, |position| 2^-53 (1 + f / 2 pi)
turns at most.  So 7.74e-8 + 2 pi 2^-32 + the 64-bit part."""
import numpy as np
import pytest
import torch

from test_gpu_heads import freqs

pytestmark = pytest.mark.gpu


def exact(pos, f):
    """cos and sin of pos * f for int64 pos and float64 f, the angle in extended precision (pos and f are taken as they are)."""
    angle = pos.astype(np.longdouble)[:, None] * f.astype(np.longdouble)[None, :]
    return np.cos(angle).astype(np.float64), np.sin(angle).astype(np.float64)


@pytest.mark.parametrize("D,rot", [(64, 64), (128, 128), (256, 64), (256, 256), (96, 48), (510, 30), (1024, 1024)])   # (both kernels)
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("start", [0, 40000, 1000003, -3000])
def test_cosines_and_sines(ctx, D, rot, adjacent, start):
    rows, half = 500, rot // 2
    f = freqs(rot, 1e4)
    pos = torch.arange(start, start + rows, dtype=torch.int32, device="cuda")
    w = torch.ones(D, device="cuda")
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if adjacent else (slice(0, half), slice(half, rot))
    w[b] = 0.0
    y = ctx.qk_norm_rope(torch.ones((rows, 1, D), device="cuda"), None, pos, f, w, eps=0.0, adjacent=adjacent)[0][:, 0].double().cpu().numpy()
    if rot < D:
        assert (y[:, rot:] == 1.0).all()      # the norm of ones is exactly one, so the elements below are the cosines and sines themselves
    c, s = exact(pos.cpu().numpy().astype(np.int64), f.cpu().numpy())
    far = 2 * np.pi * (abs(start) + rows) * 2.0 ** -53 * (1 + 1 / (2 * np.pi))
    tol = 7.74e-8 + 2 * np.pi * 2.0 ** -32 + far
    assert max(np.abs(y[:, a] - c).max(), np.abs(y[:, b] - s).max()) <= tol


@pytest.mark.parametrize("D", [128, 512])
def test_every_quarter_and_its_ends(ctx, D):
    """A frequency of one 2^-32 turn a position: the borders between quarters, the quarters, the half turn, and many others between them."""
    turns = np.concatenate([(np.arange(-4, 5)[:, None] * 2 ** 29 + np.arange(-20, 21)).reshape(-1), np.random.default_rng(D).integers(-2 ** 31, 2 ** 31, 30000)])
    turns = turns[(turns >= -2 ** 31) & (turns < 2 ** 31)]
    w = torch.ones(D, device="cuda")
    w[D // 2:] = 0.0
    f = torch.full((D // 2,), 2 * np.pi * 2.0 ** -32, dtype=torch.float64, device="cuda")
    y = ctx.qk_norm_rope(torch.ones((len(turns), 1, D), device="cuda"), None, torch.from_numpy(turns.astype(np.int32)).cuda(), f, w, eps=0.0)[0][:, 0]
    assert torch.equal(y, torch.cat([y[:, :1].expand(-1, D // 2), y[:, D // 2:D // 2 + 1].expand(-1, D // 2)], 1))      # the same pair everywhere
    y = y.double().cpu().numpy()
    c, s = exact(turns, np.array([2 * np.pi * 2.0 ** -32]))
    tol = 7.74e-8 + 2 * np.pi * 2.0 ** -32 + 2 * np.pi * 2.0 ** 31 * 2.0 ** -53
    assert max(np.abs(y[:, 0] - c[:, 0]).max(), np.abs(y[:, D // 2] - s[:, 0]).max()) <= tol
