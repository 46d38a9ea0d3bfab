"""The new operators one behind the other, as a host uses them: a prompt chunk through 4-bit projections to rotated heads and from the
last token to its candidates; and a recorded token step over GGUF matrices with the same two steps in it."""
import numpy as np
import pytest
import torch

import oracle
import qwengine_b200 as q
from qwengine_b200 import api, decode_pass, synth

from test_gpu_heads import check as check_heads, freqs, places
from test_gpu_logits import check as check_logits, definition as logits_definition
from test_gpu_mx4 import check_product, mx_values

pytestmark = pytest.mark.gpu

HID, NQ, NK, D, ROT, V = 1024, 6, 2, 128, 64, 5003


@pytest.mark.parametrize("tokens", [1, 7, 150])
def test_prompt_chunk_to_candidates(ctx, tokens):
    g = torch.Generator().manual_seed(tokens)
    x = torch.randn((tokens, HID), generator=g).bfloat16()
    wq, wk = torch.randn((NQ * 2 * D, HID), generator=g) / 32, torch.randn((NK * D, HID), generator=g) / 32
    head = torch.randn((V, HID), generator=g) / 32
    nq, nk = (1 + 0.2 * torch.randn(D, generator=g)).cuda(), (1 + 0.2 * torch.randn(D, generator=g)).cuda()
    Wq, Wk, H = (ctx.quantize_mx4(w.cuda()) for w in (wq, wk, head))
    X = ctx.quantize_mx4(x.cuda())                       # once for both projections
    qg, k = ctx.gemm_mx4(Wq, X), ctx.gemm_mx4(Wk, X)
    xv = mx_values(x.double().numpy())[0]
    check_product(qg, xv, mx_values(wq.double().numpy())[0], HID, "f32")
    check_product(k, xv, mx_values(wk.double().numpy())[0], HID, "f32")
    pos, f = places(tokens, 5000), freqs(ROT)
    heads = qg.unflatten(1, (NQ, 2 * D))[:, :, :D]       # each head beside its gate
    qo, ko = ctx.qk_norm_rope(heads, k.unflatten(1, (NK, D)), pos, f, nq, nk, kind=q.api.OUT_BF16)
    check_heads(qo, heads, nq, pos, f)
    check_heads(ko, k.unflatten(1, (NK, D)), nk, pos, f)
    logits = ctx.gemm_mx4(H, x[-1:].cuda())
    rng = np.random.default_rng(tokens)
    history, prompt = [rng.integers(0, 200, 300).tolist()], [250]
    biases, mask = [[(7, 2.0), (9, -1.0), (7, -2.0)]], rng.integers(0, 2 ** 32, (1, (V + 31) // 32), dtype=np.uint32)
    dev = lambda v, dtype: torch.tensor(v, dtype=dtype, device="cuda")   # noqa: E731
    out = ctx.adjust_logits(logits, penalties=dev([[1.3, 0.2, 0.1]], torch.float32), history=dev(history[0], torch.int32), history_begin=dev([0, 300], torch.int64),
                            prompt_len=dev(prompt, torch.int32), bias_ids=dev([7, 9, 7], torch.int32), bias_values=dev([2.0, -1.0, -2.0], torch.float32),
                            bias_begin=dev([0, 3], torch.int64), masks=torch.from_numpy(mask.view(np.int32)).cuda())
    check_logits(out, *logits_definition(logits.cpu().numpy(), penalties=np.array([[1.3, 0.2, 0.1]], np.float32), history=history, prompt=prompt, biases=biases, masks=mask))
    vals, idx = ctx.topk(out, 20)
    ctx.check()
    want_v, want_i = oracle.topk(out.cpu().numpy(), 20)
    assert np.array_equal(idx.cpu().numpy(), want_i) and np.array_equal(vals.cpu().numpy(), want_v)


def record(ctx, nb, pos, f, nq, nk, rules, in_place=True, merge=True):
    """quantize -> q + gate, k -> heads -> quantize -> head -> rules -> top-k."""
    ps = q.Pass(ctx, max_nb=nb)
    ps.set_merge(merge)
    x, xq, big, kv = ps.buffer_f32(HID), ps.buffer_q8k(HID), ps.buffer_f32(NQ * 2 * D), ps.buffer_f32(NK * D + 8)
    qs, ks, iq, logits, shaped, best = ps.buffer_f32(NQ * D), ps.buffer_f32(NK * D), ps.buffer_q8k(NQ * D), ps.buffer_f32(V), ps.buffer_f32(V + 3), ps.buffer_f32(32)
    ps.quantize(x, 0, HID, xq)
    ps.gemv(ps.matrix_upload("Q4_K", synth.make_weights("Q4_K", NQ * 2 * D, HID, seed=1), HID), xq, big)
    ps.gemv(ps.matrix_upload("Q4_K", synth.make_weights("Q4_K", NK * D, HID, seed=2), HID), xq, kv, 8)
    a, b = dict(buf=big, n_heads=NQ, head=2 * D), dict(buf=kv, n_heads=NK, off=8)
    if not in_place:
        a.update(dst=qs), b.update(dst=ks)
    ps.qk_norm_rope(a, b, D, pos, f, nq, nk)
    if in_place:
        ps.quantize(big, 0, NQ * D, iq)                   # (half of the heads and gates: any input will do)
    else:
        ps.quantize(qs, 0, NQ * D, iq)
    ps.gemv(ps.matrix_upload("Q6_K", synth.make_weights("Q6_K", V, NQ * D, seed=3), NQ * D), iq, logits)
    to, off = (logits, 0) if in_place else (shaped, 3)
    ps.adjust_logits(logits, 0, V, dst=to, dst_off=off, **rules)
    ps.topk(to, off, V, 16, best)
    return ps, dict(x=x, big=big, kv=kv, qs=qs, ks=ks, logits=logits, shaped=shaped, best=best)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("nb", [1, 3])
def test_recorded_token_step(ctx, nb, in_place):
    g = torch.Generator().manual_seed(5)
    nq, nk, f = (1 + 0.2 * torch.randn(D, generator=g)).cuda(), (1 + 0.2 * torch.randn(D, generator=g)).cuda(), freqs(ROT)
    pos = torch.zeros(nb, dtype=torch.int32, device="cuda")
    room = 40
    history = torch.full((nb, room), -1, dtype=torch.int32, device="cuda")
    masks = torch.from_numpy(np.random.default_rng(6).integers(-2 ** 31, 2 ** 31, (2, (V + 31) // 32)).astype(np.int32)).cuda()
    mask_of_row = torch.full((nb,), -1, dtype=torch.int32, device="cuda")
    rules = dict(penalties=torch.tensor([[1.2, 0.3, 0.1]] * nb, device="cuda"), history=history.view(-1), history_begin=torch.arange(nb + 1, device="cuda") * room,
                 prompt_len=torch.full((nb,), 2, dtype=torch.int32, device="cuda"), masks=masks, mask_of_row=mask_of_row,
                 bias_ids=torch.tensor([5] * nb, dtype=torch.int32, device="cuda"), bias_values=torch.ones(nb, device="cuda"), bias_begin=torch.arange(nb + 1, device="cuda"))
    ps, b = record(ctx, nb, pos, f, nq, nk, rules, in_place)
    plain, c = record(ctx, nb, pos, f, nq, nk, rules, in_place, merge=False)
    for step in range(3):
        pos.copy_(places(nb, 1000 * step))
        history[:, step] = step + 3
        if step == 2:
            mask_of_row[0] = 1
        x = synth.make_activations(nb, HID, seed=20 + step)
        y = np.empty((nb, 32), np.float32)
        ps.run_host(nb, b["x"], x, b["best"], 0, y)
        again = np.empty_like(y)
        plain.run_host(nb, c["x"], x, c["best"], 0, again)
        ctx.check()
        assert np.array_equal(y.view(np.int32), again.view(np.int32)), "merged and one kernel a step"
        # the same by direct calls
        from qwengine_b200 import formats as F
        wq, wk, wh = (torch.from_numpy(synth.make_weights(fmt, M, K, seed=s)).cuda() for fmt, M, K, s in (("Q4_K", NQ * 2 * D, HID, 1), ("Q4_K", NK * D, HID, 2), ("Q6_K", V, NQ * D, 3)))
        xq = ctx.quantize_q8k(torch.from_numpy(x).cuda())
        big, k = ctx.gemv("Q4_K", wq, xq, HID), ctx.gemv("Q4_K", wk, xq, HID)
        heads = big.unflatten(1, (NQ, 2 * D))[:, :, :D]
        qo, ko = ctx.qk_norm_rope(heads, k.unflatten(1, (NK, D)), pos, f, nq, nk, q_out=heads if in_place else None)
        check_heads(ko, k.unflatten(1, (NK, D)), nk, pos, f)
        got_k = ps.buffer_tensor(b["kv"])[:nb, 8:] if in_place else ps.buffer_tensor(b["ks"])[:nb]
        assert torch.equal(got_k, ko.flatten(1))
        hidden = big[:, :NQ * D].contiguous() if in_place else qo.flatten(1)
        logits = ctx.gemv("Q6_K", wh, ctx.quantize_q8k(hidden), NQ * D)
        shaped = ctx.adjust_logits(logits, **rules)
        lists = [[v for v in r if v >= 0] for r in history.cpu().tolist()]
        m = mask_of_row.cpu().tolist()
        check_logits(shaped, *logits_definition(logits.cpu().numpy(), penalties=rules["penalties"].cpu().numpy(), history=lists, prompt=[2] * nb, biases=[[(5, 1.0)]] * nb,
                                                masks=masks.cpu().numpy().view(np.uint32), mask_of_row=m))
        got = ps.buffer_tensor(b["logits"])[:nb] if in_place else ps.buffer_tensor(b["shaped"])[:nb, 3:]
        assert torch.equal(got, shaped)
        want_v, want_i = oracle.topk(shaped.cpu().numpy(), 16)
        assert np.array_equal(y[:, 16:].view(np.int32), want_i) and np.array_equal(y[:, :16], want_v)
    ps.close()
    plain.close()


def test_pass_refusals(ctx):
    ps = q.Pass(ctx, max_nb=2)
    a, b, col = ps.buffer_f32(1024), ps.buffer_f32(1024), ps.buffer_q8k(1024)
    pos, f = places(2, 0), freqs(64)
    head = lambda **kw: {**dict(buf=a, n_heads=4), **kw}   # noqa: E731
    for bad in (dict(q=head(n_heads=9)), dict(q=head(off=600)), dict(q=head(head=300, n_heads=4)), dict(q=head(buf=col)), dict(q=head(dst=b, dst_off=700)),
                dict(q=head(dst=b, dst_head=100)), dict(q=head(), k=head(off=256)), dict(q=head(), k=head(off=500, n_heads=2)), dict(q=head(dst=a, dst_off=4)),
                dict(q=head(dst=b), k=head(off=512, dst=b, dst_off=500)), dict(q=head(n_heads=0)), dict(q=head(buf=17))):
        with pytest.raises(api.Q38BError):
            ps.qk_norm_rope(bad["q"], bad.get("k"), 128, pos, f)
    with pytest.raises(ValueError):
        ps.qk_norm_rope(head(), None, 128, pos[:1], f)     # a position for every column
    for bad in (dict(src=a, off=1, n=1024), dict(src=col, off=0, n=10), dict(src=a, off=0, n=100, dst=a, dst_off=50), dict(src=a, off=0, n=100, dst=b, dst_off=1000), dict(src=a, off=0, n=0)):
        with pytest.raises(api.Q38BError):
            ps.adjust_logits(bad.pop("src"), bad.pop("off"), bad.pop("n"), **bad)
    with pytest.raises(api.Q38BError):
        ps.adjust_logits(a, 0, 100, penalties=torch.ones((2, 3), device="cuda"))
    ps.close()


def test_27b_shaped_layers_with_heads(ctx):
    """Four layers of the 27B-shaped pass with the attention layer's heads normed and rotated in place: one kernel more, the key heads as by a direct call."""
    g = torch.Generator().manual_seed(7)
    w = dict(q_weight=(1 + 0.2 * torch.randn(256, generator=g)).cuda(), k_weight=(1 + 0.2 * torch.randn(256, generator=g)).cuda())
    pos, f = places(1, 777), freqs(64)
    out = []
    for heads in (None, dict(positions=pos, inv_freq=f, **w)):
        ps = q.Pass(ctx, max_nb=1)
        made = decode_pass.build(ps, lambda spec, rows: ps.matrix_device(spec.fmt, weights(spec), spec.K), n_layers=4, head=False, heads=heads)
        ps.buffer_tensor(made["in_buf"]).copy_(torch.from_numpy(synth.make_activations(1, decode_pass.HIDDEN, seed=8)))
        ps.run(1)
        ctx.check()
        # buffers in the order decode_pass makes them: 3 is the projections' output, 4 keys and values
        out.append((ps.kernel_count, ps.buffer_tensor(4).clone(), ps.buffer_tensor(made["out_buf"]).clone()))
        ps.close()
    (n0, kv0, x0), (n1, kv1, x1) = out
    assert n1 == n0 + 1 and torch.equal(kv0[:, 1024:], kv1[:, 1024:]) and not torch.equal(x0, x1)
    k = kv0[:, :1024].unflatten(1, (4, 256))
    want = ctx.qk_norm_rope(k, None, pos, f, w["k_weight"])[0]
    check_heads(want, k, w["k_weight"], pos, f)
    assert torch.equal(kv1[:, :1024], want.flatten(1))


_made = {}


def weights(spec):
    if spec.name not in _made:
        _made[spec.name] = torch.from_numpy(synth.make_weights(spec.fmt, spec.M, spec.K, seed=len(_made), scale=decode_pass.UNIT_GAIN_SCALE[spec.fmt])).cuda()
    return _made[spec.name]
