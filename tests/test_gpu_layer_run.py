"""An attention layer's operators one behind the other, as a host uses them: 8-bit projections, rotated heads, the cache and the attention over it, the 8-bit output
projection, for prompts stepped together and then token by token; and the same steps recorded in a pass over GGUF matrices."""
import numpy as np
import pytest
import torch

import qwengine_b200 as q
from qwengine_b200 import api, decode_pass, formats as F, synth

from test_gpu_cache import Text, check as check_attention
from test_gpu_heads import check as check_heads, freqs, places
from test_gpu_i8 import check_product, definition as codes_of

pytestmark = pytest.mark.gpu

HID, NQ, NK, D, ROT, PAGE = 512, 12, 2, 64, 32, 16


class Batch:
    """Sequences that grow: pages handed out as they are needed, plan and tensors for the next chunk, and the keys and values they hold."""

    def __init__(self, n, room, nk=NK, D=D, dtype=torch.bfloat16):
        self.n, self.per, self.nk, self.D, self.page, self.dtype = n, -(-room // PAGE), nk, D, PAGE, {torch.bfloat16: "bf16", torch.float16: "f16"}[dtype]
        pages = n * self.per + 2
        g = torch.Generator().manual_seed(n)
        self.table = torch.randperm(pages, generator=g)[:n * self.per].view(n, self.per).to(torch.int32).cuda()
        self.k, self.v = (torch.full((pages, PAGE, nk, D), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
        self.cache = q.PagedCache(self.k, self.v)
        self.lengths, self.begin = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(n + 1, dtype=torch.int32, device="cuda")

    def chunk(self, new):
        totals = [int(t) + k for t, k in zip(self.lengths.tolist(), new)]
        self.plan = list(zip(new, totals))
        self.lengths.copy_(torch.tensor(totals, dtype=torch.int32))
        self.begin.copy_(torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32))
        return torch.cat([torch.arange(t - k, t, dtype=torch.int32) for k, t in self.plan]).cuda()

    def held(self):
        """keys, values: what the pages hold for each sequence"""
        out = []
        for c in (self.k, self.v):
            out.append([c[self.table[s].long()].flatten(0, 1)[:t].cpu() for s, (_, t) in enumerate(self.plan)])
        self.keys, self.values = out


def test_prompts_and_tokens_through_a_layer(ctx):
    g = torch.Generator().manual_seed(1)
    make = lambda rows, K: ctx.quantize_i8((torch.randn((rows, K), generator=g) / K ** 0.5).cuda())   # noqa: E731
    Wq, Wkv, Wo = make(NQ * D, HID), make(2 * NK * D, HID), make(HID, NQ * D)
    nq, nk, f = (1 + 0.2 * torch.randn(D, generator=g)).cuda(), (1 + 0.2 * torch.randn(D, generator=g)).cuda(), freqs(ROT)
    b = Batch(3, 120)
    for new in ([40, 7, 61], [1, 1, 1], [3, 1, 5], [0, 1, 1]):
        pos = b.chunk(new)
        rows = sum(new)
        x = torch.randn((rows, HID), generator=g).bfloat16()
        X = ctx.quantize_i8(x.cuda())                      # once for both projections
        qs, kv = ctx.gemm_i8(Wq, X), ctx.gemm_i8(Wkv, X)
        xc = codes_of(x.double().numpy())
        for y, W in ((qs, Wq), (kv, Wkv)):
            check_product(y, *xc, W.codes.cpu().numpy().astype(np.int64), W.scales.cpu().numpy(), "f32")
        k, v = kv.unflatten(1, (2, NK, D)).unbind(1)
        qo, ko = ctx.qk_norm_rope(qs.unflatten(1, (NQ, D)), k, pos, f, nq, nk)
        check_heads(ko, k, nk, pos, f)
        ctx.cache_append(b.cache, ko, v, b.table, b.lengths, b.begin)
        b.held()
        row = 0
        for s, (n, t) in enumerate(b.plan):                # what was written is the rows rounded once
            assert torch.equal(b.keys[s][t - n:], ko[row:row + n].bfloat16().cpu()) and torch.equal(b.values[s][t - n:], v[row:row + n].bfloat16().cpu())
            row += n
        mixed = ctx.attention(b.cache, qo, b.table, b.lengths, b.begin, kind=api.OUT_BF16)
        check_attention(b, qo, mixed, D ** -0.5)
        y = ctx.gemm_i8(Wo, mixed.flatten(1), kind=api.OUT_BF16)
        ctx.check()
        check_product(y, *codes_of(mixed.flatten(1).double().cpu().numpy()), Wo.codes.cpu().numpy().astype(np.int64), Wo.scales.cpu().numpy(), "bf16")


def test_chunks_and_single_tokens_agree(ctx):
    """A text in one chunk and token by token: the same keys, values and (within the bound) outputs."""
    g = torch.Generator().manual_seed(2)
    n = 37
    k, v, x = (torch.randn((n, h, D), generator=g).bfloat16().cuda() for h in (NK, NK, NQ))
    whole, single = Batch(1, 64), Batch(1, 64)
    whole.chunk([n])
    ctx.cache_append(whole.cache, k, v, whole.table, whole.lengths, whole.begin)
    whole.held()
    a = ctx.attention(whole.cache, x, whole.table, whole.lengths, whole.begin)
    check_attention(whole, x, a, D ** -0.5)
    for i in range(n):
        single.chunk([1])
        ctx.cache_append(single.cache, k[i:i + 1], v[i:i + 1], single.table, single.lengths, single.begin)
        single.held()
        check_attention(single, x[i:i + 1], ctx.attention(single.cache, x[i:i + 1], single.table, single.lengths, single.begin), D ** -0.5)
    ctx.check()
    assert torch.equal(whole.keys[0], single.keys[0]) and torch.equal(whole.values[0], single.values[0])


def test_recorded_step(ctx):
    """quantize -> q + gate, k and v -> heads -> cache -> attention -> quantize -> output projection, replayed while the text grows."""
    nb, inner = 3, NQ * D
    g = torch.Generator().manual_seed(5)
    nq, nk, f = (1 + 0.2 * torch.randn(D, generator=g)).cuda(), (1 + 0.2 * torch.randn(D, generator=g)).cuda(), freqs(ROT)
    pos = torch.zeros(nb, dtype=torch.int32, device="cuda")
    a, b = Batch(nb, 64), Batch(nb, 64)
    ps = q.Pass(ctx, max_nb=nb)
    x, xq, big, kv = ps.buffer_f32(HID), ps.buffer_q8k(HID), ps.buffer_f32(2 * inner), ps.buffer_f32(2 * NK * D + 4)
    mixed, iq, y = ps.buffer_f32(inner + 8), ps.buffer_q8k(inner), ps.buffer_f32(HID)
    wq, wkv, wo = (synth.make_weights("Q4_K", M, K, seed=s) for M, K, s in ((2 * inner, HID, 1), (2 * NK * D, HID, 2), (HID, inner, 3)))
    ps.quantize(x, 0, HID, xq)
    ps.gemv(ps.matrix_upload("Q4_K", wq, HID), xq, big)
    ps.gemv(ps.matrix_upload("Q4_K", wkv, HID), xq, kv, 4)
    ps.qk_norm_rope(dict(buf=big, n_heads=NQ, head=2 * D), dict(buf=kv, n_heads=NK, off=4), D, pos, f, nq, nk)
    ps.cache_append(a.cache, dict(buf=kv, off=4), dict(buf=kv, off=4 + NK * D), a.table, a.lengths, a.begin)
    ps.attention(a.cache, dict(buf=big, n_heads=NQ, head=2 * D), dict(buf=mixed, off=8), a.table, a.lengths, a.begin)
    ps.quantize(mixed, 8, inner, iq)
    ps.gemv(ps.matrix_upload("Q4_K", wo, inner), iq, y)
    dev = lambda w: torch.from_numpy(w).cuda()   # noqa: E731
    for step, new in enumerate(([1, 1, 1], [3, 0, 0], [0, 2, 1], [1, 1, 1])):
        pos.copy_(a.chunk(new))
        b.chunk(new)
        xs = synth.make_activations(nb, HID, seed=30 + step)
        ps.buffer_tensor(x).copy_(torch.from_numpy(xs))
        ps.run(nb)
        ctx.check()
        cols = ctx.quantize_q8k(dev(xs))
        bigd, kvd = ctx.gemv("Q4_K", dev(wq), cols, HID), ctx.gemv("Q4_K", dev(wkv), cols, HID)
        heads, keys = bigd.unflatten(1, (NQ, 2 * D))[:, :, :D], kvd[:, :NK * D].unflatten(1, (NK, D))
        ctx.qk_norm_rope(heads, keys, pos, f, nq, nk, q_out=heads, k_out=keys)
        ctx.cache_append(b.cache, keys, kvd[:, NK * D:].unflatten(1, (NK, D)), b.table, b.lengths, b.begin)
        out = ctx.attention(b.cache, heads, b.table, b.lengths, b.begin)
        b.held(), a.held()
        assert all(torch.equal(s, t) for s, t in zip(a.keys + a.values, b.keys + b.values))
        check_attention(b, heads, out, D ** -0.5)
        assert torch.equal(ps.buffer_tensor(mixed)[:, 8:], out.flatten(1))
        want = ctx.gemv("Q4_K", dev(wo), ctx.quantize_q8k(out.flatten(1).contiguous()), inner)
        assert torch.equal(ps.buffer_tensor(y), want)
    # a run for fewer columns ends the batch there
    a.chunk([1, 1, 1])
    keep = ps.buffer_tensor(mixed)[1:].clone()
    kept = a.k.clone()
    ps.run(1)
    ctx.check()
    assert torch.equal(ps.buffer_tensor(mixed)[1:], keep)
    s1 = a.table[1].long()
    assert torch.equal(torch.nan_to_num(a.k[s1]), torch.nan_to_num(kept[s1])), "the second sequence's keys"
    ps.close()


def test_pass_refusals(ctx):
    b = Batch(2, 40)
    ps = q.Pass(ctx, max_nb=2)
    buf, out, col = ps.buffer_f32(1024), ps.buffer_f32(NQ * D), ps.buffer_q8k(1024)
    batch = (b.table, b.lengths, b.begin)
    for k, v in ((dict(buf=col), dict(buf=buf)), (dict(buf=buf, off=1000), dict(buf=buf)), (dict(buf=buf), dict(buf=buf, off=-1)), (dict(buf=buf), dict(buf=buf, head=1000)), (dict(buf=9), dict(buf=buf))):
        with pytest.raises(api.Q38BError):
            ps.cache_append(b.cache, k, v, *batch)
    for heads, to, kw in ((dict(buf=buf, n_heads=NQ + 1), dict(buf=out), {}), (dict(buf=buf, n_heads=17 * NK), dict(buf=out), {}), (dict(buf=buf, n_heads=NQ), dict(buf=out, off=1), {}),
                          (dict(buf=buf, n_heads=4), dict(buf=buf, off=255), {}), (dict(buf=buf, n_heads=NQ), dict(buf=out, head=32), {}), (dict(buf=col, n_heads=4), dict(buf=out), {}),
                          (dict(buf=buf, n_heads=NQ), dict(buf=out), dict(scale=-1.0))):
        with pytest.raises(api.Q38BError):
            ps.attention(b.cache, heads, to, *batch, **kw)
    with pytest.raises(ValueError):
        ps.attention(b.cache, dict(buf=buf, n_heads=NQ), dict(buf=out), b.table.long(), b.lengths, b.begin)
    ps.close()


def test_27b_shaped_layers_with_a_cache(ctx):
    """Four layers of the 27B-shaped pass, the attention layer over a cache of its own: token by token as by direct calls on what the pass computed."""
    g = torch.Generator().manual_seed(7)
    w = dict(q_weight=(1 + 0.2 * torch.randn(256, generator=g)).cuda(), k_weight=(1 + 0.2 * torch.randn(256, generator=g)).cuda())
    pos, f = places(1, 0), freqs(64)
    b, mirror = Batch(1, 40, nk=4, D=256), Batch(1, 40, nk=4, D=256)
    ps = q.Pass(ctx, max_nb=1)
    made = decode_pass.build(ps, lambda spec, rows: ps.matrix_device(spec.fmt, weights(spec), spec.K), n_layers=4, head=False, heads=dict(positions=pos, inv_freq=f, **w),
                             cache=dict(caches=[b.cache], table=b.table, lengths=b.lengths, begin=b.begin))
    outs = []
    for step in range(3):
        pos.copy_(b.chunk([1]))
        mirror.chunk([1])
        ps.buffer_tensor(made["in_buf"]).copy_(torch.from_numpy(synth.make_activations(1, decode_pass.HIDDEN, seed=8 + step)))
        ps.run(1)
        ctx.check()
        # buffers in the order decode_pass makes them: 3 the projections' output, 4 keys and values, 9 the attention's outputs
        heads, kv = ps.buffer_tensor(3)[:, :12288].unflatten(1, (24, 512))[:, :, :256], ps.buffer_tensor(4).unflatten(1, (2, 4, 256))
        ctx.cache_append(mirror.cache, kv[:, 0], kv[:, 1], mirror.table, mirror.lengths, mirror.begin)
        b.held(), mirror.held()
        assert torch.equal(b.keys[0], mirror.keys[0]) and torch.equal(b.values[0], mirror.values[0])
        want = ctx.attention(mirror.cache, heads, mirror.table, mirror.lengths, mirror.begin)
        check_attention(mirror, heads, want, 256 ** -0.5)
        assert torch.equal(ps.buffer_tensor(9), want.flatten(1))
        outs.append(ps.buffer_tensor(made["out_buf"]).clone())
    assert bool(torch.stack(outs).isfinite().all()) and not torch.equal(outs[0], outs[1])
    ps.close()


_made = {}


def weights(spec):
    if spec.name not in _made:
        _made[spec.name] = torch.from_numpy(synth.make_weights(spec.fmt, spec.M, spec.K, seed=len(_made), scale=decode_pass.UNIT_GAIN_SCALE[spec.fmt])).cuda()
    return _made[spec.name]
