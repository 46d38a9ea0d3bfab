"""One head (or one row) has no second one at a stride: that stride, whatever it is, does not make a call in place another one, and what a
pass records it also runs."""
import pytest
import torch

import qwengine_b200 as q
from qwengine_b200 import api

from test_gpu_heads import check, freqs, inputs, places

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,rot,off", [(128, 64, 0), (96, 48, 3), (66, 34, 1)])
@pytest.mark.parametrize("src_head,dst_head", [(None, 0), (0, None), (512, 128), (7, 300)])
@pytest.mark.parametrize("nb", [1, 3])
def test_a_pass_runs_what_it_records(ctx, nb, D, rot, off, src_head, dst_head):
    pos, f = places(nb, 40), freqs(rot)
    ps = q.Pass(ctx, max_nb=nb)
    a = ps.buffer_f32(D + off + 5)
    h = dict(buf=a, n_heads=1, off=off)
    if src_head is not None:
        h.update(head=src_head)
    h.update(dst_head=D if dst_head is None else dst_head)
    ps.qk_norm_rope(h, None, D, pos, f)
    x = inputs(nb, 1, D, D + nb)
    buf = ps.buffer_tensor(a)
    buf.fill_(7.0)
    buf[:, off:off + D] = x[:, 0]
    ps.run(nb)
    ctx.check()
    check(buf[:, off:off + D].unsqueeze(1), x, None, pos, f)
    assert (buf[:, :off] == 7.0).all() and (buf[:, off + D:] == 7.0).all()
    ps.close()


def test_a_pass_refuses_what_its_run_would(ctx):
    ps = q.Pass(ctx, max_nb=2)
    a, b = ps.buffer_f32(256), ps.buffer_f32(256)
    pos, f = places(2, 0), freqs(64)
    for h in (dict(buf=a, n_heads=1, dst_head=-128), dict(buf=a, n_heads=1, dst=b, dst_head=-1), dict(buf=a, n_heads=1, head=-1)):
        with pytest.raises(api.Q38BError):
            ps.qk_norm_rope(h, None, 128, pos, f)
    ps.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_direct_calls(ctx, dtype):
    """Views of one head, and of one row, whose strides differ although their elements are the same."""
    pos, f = places(5, 9), freqs(64)
    x = inputs(5, 1, 128, 3, dtype)
    want = ctx.qk_norm_rope(x, None, pos, f)[0]
    y = x.clone()
    got = ctx.qk_norm_rope(y.as_strided((5, 1, 128), (128, 256, 1)), None, pos, f, q_out=y.as_strided((5, 1, 128), (128, 128, 1)))[0]
    assert torch.equal(got, want) and torch.equal(y, want)
    x = inputs(1, 4, 128, 4, dtype)
    want = ctx.qk_norm_rope(x, None, pos[:1], f)[0]
    y = x.clone()
    ctx.qk_norm_rope(y.as_strided((1, 4, 128), (999, 128, 1)), None, pos[:1], f, q_out=y)
    assert torch.equal(y, want)
    for strides in ((512, 256, 1), (512, 0, 1)):            # several heads, several rows: element over element, or refused
        z = torch.zeros(4096, dtype=y.dtype, device="cuda")
        with pytest.raises(api.Q38BError):
            ctx.qk_norm_rope(z.as_strided((2, 2, 128), strides), None, pos[:2], f, q_out=z.as_strided((2, 2, 128), (512, 128, 1)))
    with pytest.raises(api.Q38BError):
        z = torch.zeros(4096, dtype=y.dtype, device="cuda")
        ctx.qk_norm_rope(z.as_strided((2, 2, 128), (256, 128, 1)), None, pos[:2], f, q_out=z.as_strided((2, 2, 128), (512, 128, 1)))
    ctx.check()
