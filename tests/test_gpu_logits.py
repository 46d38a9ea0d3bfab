"""Penalties, biases and masks on logits (adjust_logits) against the formula in 64 bits, token by token.

Bound, u = 2^-24: the quotient or product rounds once, u |l'|; frequency * count once, both differences and the bias's sum once each, every one of them
at most u of the sum of magnitudes met so far: 5 u (|l'| + |freq count| + |pres| + |bias|).  What no rule touches comes back bit for bit."""
import numpy as np
import pytest
import torch

import qwengine_b200 as q   # noqa: F401
from qwengine_b200 import api

pytestmark = pytest.mark.gpu


def definition(x, off=0, penalties=None, history=None, prompt=None, biases=None, masks=None, mask_of_row=None):
    """Python lists per row; returns float64 values and their bounds."""
    y, tol = x.astype(np.float64), np.zeros(x.shape)
    n = x.shape[1]
    for r in range(x.shape[0]):
        mag = np.abs(y[r])
        touched = np.zeros(n, bool)
        if history is not None:
            rep, freq, pres = (float(v) for v in penalties[r])
            made = history[r][prompt[r]:]
            for v in set(history[r]):
                i = v - off
                if v < 0 or not 0 <= i < n:
                    continue
                c = made.count(v)
                y[r, i] = y[r, i] / rep if y[r, i] > 0 else y[r, i] * rep
                mag[i] = abs(y[r, i]) + abs(freq * c) + (abs(pres) if c else 0)
                y[r, i] -= freq * c + (pres if c else 0)
                touched[i] = True
        if biases is not None:
            for v, b in dict(biases[r]).items():
                if v >= 0 and 0 <= v - off < n:
                    y[r, v - off] += b
                    mag[v - off] += abs(b)
                    touched[v - off] = True
        tol[r][touched] = 5 * 2.0 ** -24 * mag[touched]
        m = -1 if masks is None else r if mask_of_row is None else mask_of_row[r]
        if m >= 0:
            bits = np.unpackbits(masks[m].view(np.uint8), bitorder="little")[off:off + n]
            y[r][bits == 0] = -np.inf
    return y, tol


def run(ctx, x, off=0, penalties=None, history=None, prompt=None, biases=None, masks=None, mask_of_row=None, **kw):
    dev = lambda v, dtype: torch.tensor(v, dtype=dtype, device="cuda")   # noqa: E731
    begin = lambda rows: dev(np.concatenate([[0], np.cumsum([len(r) for r in rows])]).tolist(), torch.int64)   # noqa: E731
    a = {}
    if history is not None:
        a.update(penalties=dev(penalties, torch.float32), history=dev([v for r in history for v in r], torch.int32), history_begin=begin(history), prompt_len=dev(prompt, torch.int32))
    if biases is not None:
        a.update(bias_ids=dev([v for r in biases for v, _ in r], torch.int32), bias_values=dev([b for r in biases for _, b in r], torch.float32), bias_begin=begin(biases))
    if masks is not None:
        a.update(masks=torch.from_numpy(masks.view(np.int32)).cuda(), mask_of_row=None if mask_of_row is None else dev(mask_of_row, torch.int32))
    x = torch.from_numpy(x).cuda() if isinstance(x, np.ndarray) else x
    y = ctx.adjust_logits(x, index_offset=off, **a, **kw)
    ctx.check()
    return y


def check(y, want, tol):
    y = y.double().cpu().numpy()
    assert np.array_equal(np.isneginf(y), np.isneginf(want)) and np.array_equal(np.isnan(y), np.isnan(want))
    fine = np.isfinite(want)
    assert np.array_equal(np.isfinite(y), fine)
    bad = np.abs(y[fine] - want[fine]) > tol[fine]
    assert not bad.any(), (bad.sum(), np.abs(y[fine] - want[fine]).max())


def case(rows, n, hist, nbias, seed, off=0, n_masks=0):
    g = np.random.default_rng(seed)
    x = (4 * g.standard_normal((rows, n))).astype(np.float32)
    top = off + n + 5                                              # some ids lie outside the logits
    history = [[int(v) for v in np.minimum(top, np.exp(g.random(int(g.integers(0, hist + 1))) * np.log(top + 1)).astype(int)) - 3] for _ in range(rows)]
    prompt = [int(g.integers(0, len(h) + 1)) for h in history]
    pen = np.stack([0.8 + g.random(rows), g.random(rows) - 0.2, g.random(rows) - 0.2], 1).astype(np.float32).tolist()
    biases = [[(int(g.integers(-2, top)), float(np.float32(3 * g.standard_normal()))) for _ in range(nbias)] for _ in range(rows)]
    out = dict(off=off, penalties=pen, history=history, prompt=prompt, biases=biases if nbias else None)
    if n_masks:
        out["masks"] = g.integers(0, 2 ** 32, (n_masks, (off + n + 31) // 32), dtype=np.uint32)
        out["mask_of_row"] = [int(v) for v in g.integers(-1, n_masks, rows)]
    return x, out


@pytest.mark.parametrize("rows,n,hist,nbias,n_masks", [(1, 1, 3, 1, 1), (1, 248320, 600, 0, 0), (3, 1000, 50, 7, 2), (8, 100001, 4000, 300, 4), (2, 4096, 0, 5, 1),
                                                       (2, 4097, 200, 0, 2), (5, 31, 40, 3, 5), (33, 2500, 900, 32, 9)])
def test_all_rules(ctx, rows, n, hist, nbias, n_masks):
    x, rules = case(rows, n, hist, nbias, rows + n, n_masks=n_masks)
    check(run(ctx, x, **rules), *definition(x, **rules))


@pytest.mark.parametrize("off", [1, 31, 32, 1000, 124160])
def test_a_shard_of_the_head(ctx, off):
    """Columns of a row-sharded head: token ids are offset, the mask is the whole vocabulary's."""
    x, rules = case(4, 3001, 500, 40, off, off=off, n_masks=3)
    rules["history"] = [[v + off if i % 2 else v for i, v in enumerate(r)] for r in rules["history"]]
    check(run(ctx, x, **rules), *definition(x, **rules))


def test_each_rule_alone(ctx):
    x, rules = case(4, 5000, 800, 20, 1, n_masks=4)
    for keep in (("penalties", "history", "prompt"), ("biases",), ("masks", "mask_of_row"), ("masks",), ()):
        only = {k: rules[k] for k in keep}
        y = run(ctx, x, **only)
        want, tol = definition(x, **only)
        check(y, want, tol)
        same = (tol == 0) & np.isfinite(want)
        assert np.array_equal(y.cpu().numpy()[same].view(np.uint32), x[same].view(np.uint32))


def test_repeats_count_and_prompt_tokens_only_are_not_generated(ctx):
    x = np.array([[2.0, -2.0, 1.0, 0.0, 3.0]], np.float32)
    y = run(ctx, x, penalties=[[2.0, 0.5, 0.25]], history=[[0, 1, 1, 4, 4, 4]], prompt=[3]).cpu().numpy()
    assert y.tolist() == [[1.0, -4.0, 1.0, 0.0, 1.5 - 1.5 - 0.25]]
    assert run(ctx, x, penalties=[[2.0, 0.5, 0.25]], history=[[3] * 100000], prompt=[0]).cpu().numpy()[0, 3] == -50000.25


def test_the_last_bias_of_a_token_counts(ctx):
    x = np.zeros((2, 10), np.float32)
    for _ in range(5):
        y = run(ctx, x, biases=[[(3, float(i)) for i in range(500)] + [(4, 1.0), (3, 7.0)], [(9, -1.0), (9, 2.0)]])
        assert y[0, 3] == 7.0 and y[0, 4] == 1.0 and y[1, 9] == 2.0 and y.abs().sum() == 10.0


def test_masks_that_leave_nothing_and_what_lies_under_them(ctx):
    n = 70
    x = np.zeros((3, n), np.float32)
    x[0, 5], x[1, 6], x[2, 7] = np.nan, np.inf, -np.inf
    masks = np.array([[0, 0, 0], [0xFFFFFFFF] * 3], np.uint32)
    y = run(ctx, x, masks=masks, mask_of_row=[0, 1, -1], biases=[[(5, 1.0)], [(6, 1.0)], [(7, 1.0)]]).cpu().numpy()
    assert np.isneginf(y[0]).all()                       # NaN goes under the mask too
    assert y[1, 6] == np.inf and (np.delete(y[1], 6) == 0).all() and y[2, 7] == -np.inf
    vals, idx = ctx.topk(run(ctx, x, masks=masks, mask_of_row=[0, 1, -1]), 3)
    assert idx[0].tolist() == [0, 1, 2] and torch.isneginf(vals[0]).all()


@pytest.mark.parametrize("pad,start", [(0, 0), (1, 0), (2, 1), (3, 2), (4, 3), (7, 5)])
def test_row_strides_offsets_and_in_place(ctx, pad, start):
    x, rules = case(5, 4099, 300, 10, pad, n_masks=2)
    want = run(ctx, x, **rules)
    flat = torch.full((start + 5 * (4099 + pad) + 9,), 123.0, device="cuda")
    v = flat.as_strided((5, 4099), (4099 + pad, 1), start)
    v.copy_(torch.from_numpy(x))
    out = torch.full_like(flat, 55.0)
    o = out.as_strided((5, 4099), (4099 + pad, 1), start)
    run(ctx, v, **rules, out=o)
    assert torch.equal(o, want)
    o.fill_(55.0)
    assert (out == 55.0).all()
    plain = torch.empty((5, 4099), device="cuda")        # source and destination aligned differently
    assert torch.equal(run(ctx, v, **rules, out=plain), want)
    assert run(ctx, v, **rules, out=v) is v and torch.equal(v, want)
    v.fill_(123.0)
    assert (flat == 123.0).all()


@pytest.mark.parametrize("rows,n,hist,nbias,n_masks,off", [(40, 248320, 3000, 40, 7, 0), (300, 20011, 900, 5, 300, 0), (41, 130000, 30000, 700, 3, 77), (640, 8192, 50, 0, 0, 31),
                                                           (641, 8193, 0, 3, 2, 0), (1200, 4099, 300, 20, 1200, 0)])
def test_four_at_a_time_give_the_bits_of_one(ctx, rows, n, hist, nbias, n_masks, off):
    """Rows that are aligned (contiguous ones) or not (an odd distance), every size of a CTA's piece."""
    g = np.random.default_rng(rows)
    x = torch.randn((rows, n + 3), generator=torch.Generator(device="cuda").manual_seed(rows), device="cuda")[:, 1:n + 1]
    length = g.integers(0, hist + 1, rows)
    begin = np.concatenate([[0], np.cumsum(length)])
    dev = lambda v, dtype: torch.from_numpy(np.ascontiguousarray(v)).to(dtype).cuda()   # noqa: E731
    rules = dict(masks=dev(g.integers(-2 ** 31, 2 ** 31, (max(n_masks, 1), (off + n + 31) // 32)), torch.int32), mask_of_row=dev(g.integers(-1, n_masks, rows), torch.int32)) if n_masks else {}
    if hist:
        rules.update(penalties=dev(np.stack([0.8 + g.random(rows), g.random(rows) - 0.2, g.random(rows)], 1), torch.float32), history_begin=dev(begin, torch.int64),
                     history=dev(np.exp(g.random(begin[-1]) * np.log(off + n + 9)).astype(np.int64) - 2, torch.int32), prompt_len=dev(g.integers(-3, hist + 9, rows), torch.int32))
    if nbias:
        rules.update(bias_ids=dev(g.integers(-2, off + n + 2, rows * nbias), torch.int32), bias_values=dev(g.standard_normal(rows * nbias), torch.float32), bias_begin=dev(np.arange(rows + 1) * nbias, torch.int64))
    got = ctx.adjust_logits(x, index_offset=off, **rules)
    wide = torch.empty((rows, (n + 7) // 4 * 4), device="cuda")
    aligned = torch.empty_like(wide)[:, :n]
    wide[:, :n] = x
    want = ctx.adjust_logits(wide[:, :n], index_offset=off, out=aligned, **rules)
    assert torch.equal(got.view(torch.int32), want.contiguous().view(torch.int32))
    want = want.contiguous()
    assert torch.equal(ctx.adjust_logits(wide[:, :n], index_offset=off, out=wide[:, :n], **rules).contiguous().view(torch.int32), want.view(torch.int32))
    here = ctx.adjust_logits(x, index_offset=off, out=x, **rules)
    assert torch.equal(here.contiguous().view(torch.int32), want.view(torch.int32))
    ctx.check()


def test_long_histories_give_the_same_bits_each_time(ctx):
    x, rules = case(6, 50000, 60000, 100, 2)
    a = run(ctx, x, **rules)
    check(a, *definition_counts(x, rules))
    for _ in range(3):
        assert torch.equal(run(ctx, x, **rules), a)


def definition_counts(x, rules):
    """definition() with the counting done once per row (list.count is quadratic)."""
    from collections import Counter
    y, tol = x.astype(np.float64), np.zeros(x.shape)
    for r in range(x.shape[0]):
        rep, freq, pres = (float(v) for v in rules["penalties"][r])
        made = Counter(rules["history"][r][rules["prompt"][r]:])
        for v in set(rules["history"][r]):
            if 0 <= v < x.shape[1]:
                l = y[r, v] / rep if y[r, v] > 0 else y[r, v] * rep
                c = made[v]
                tol[r, v] = 5 * 2.0 ** -24 * (abs(l) + abs(freq * c) + (abs(pres) if c else 0))
                y[r, v] = l - freq * c - (pres if c else 0)
        for v, b in dict(rules["biases"][r]).items():
            if 0 <= v < x.shape[1]:
                tol[r, v] += 5 * 2.0 ** -24 * (abs(y[r, v]) + abs(b))
                y[r, v] += b
    return y, tol


def test_replayed_with_new_lists(ctx):
    """A captured call reads the lists as they are at each replay: tokens are appended in place."""
    n, room = 3000, 64
    x = torch.randn((2, n), generator=torch.Generator().manual_seed(4)).cuda()
    history = torch.zeros(2 * room, dtype=torch.int32, device="cuda")
    begin = torch.tensor([0, 0, 0], dtype=torch.int64, device="cuda")
    pen, prompt = torch.tensor([[1.5, 0.1, 0.2]] * 2, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    out = torch.empty_like(x)
    call = lambda: ctx.adjust_logits(x, out=out, penalties=pen, history=history, history_begin=begin, prompt_len=prompt)   # noqa: E731
    call()
    assert torch.equal(out, x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for lists in ([[5], [7, 7]], [[5, 6, 5], [7, 7, 2999]]):
        history[:len(lists[0]) + len(lists[1])] = torch.tensor(lists[0] + lists[1], dtype=torch.int32)
        begin.copy_(torch.tensor([0, len(lists[0]), len(lists[0]) + len(lists[1])]))
        graph.replay()
        check(out, *definition(x.cpu().numpy(), penalties=pen.cpu().tolist(), history=lists, prompt=[0, 0]))


def test_refusals(ctx):
    x = torch.zeros((2, 100), device="cuda")
    i32, i64 = (lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")), (lambda *v: torch.tensor(v, dtype=torch.int64, device="cuda"))
    pen = torch.ones((2, 3), device="cuda")
    for bad in (dict(penalties=pen[:1], history=i32(1), history_begin=i64(0, 1, 1)), dict(penalties=pen, history=i64(1), history_begin=i64(0, 1, 1)),
                dict(penalties=pen, history=i32(1), history_begin=i64(0, 1)), dict(bias_ids=i32(1), bias_values=pen[0, :2], bias_begin=i64(0, 1, 1)),
                dict(masks=torch.zeros((2, 3), dtype=torch.int32, device="cuda")), dict(masks=torch.zeros((1, 4), dtype=torch.int32, device="cuda")),
                dict(out=torch.zeros((2, 99), device="cuda")), dict(mask_of_row=i64(0, 1)), dict(penalties=pen.cpu(), history=i32(1), history_begin=i64(0, 1, 1))):
        with pytest.raises(ValueError):
            ctx.adjust_logits(x, **bad)
    for bad in (dict(penalties=pen), dict(history=i32(1), history_begin=i64(0, 1, 1)), dict(mask_of_row=i32(0, 1)), dict(penalties=pen, history=i32(1))):
        with pytest.raises(api.Q38BError):
            ctx.adjust_logits(x, **bad)
    with pytest.raises(ValueError):
        ctx.adjust_logits(x.half())
    ctx.check()


def test_short_texts_at_every_alignment(ctx):
    """Texts of 0 to 10 tokens one behind the other, prompts of every length: their 16-byte pieces begin and end anywhere."""
    g = np.random.default_rng(8)
    rows, n = 600, 37
    history = [g.integers(-2, n + 2, int(g.integers(0, 11))).tolist() for _ in range(rows)]
    prompt = [int(g.integers(0, len(h) + 1)) for h in history]
    x = (3 * g.standard_normal((rows, n))).astype(np.float32)
    rules = dict(penalties=np.stack([g.uniform(1, 2, rows), g.uniform(-1, 1, rows), g.uniform(-1, 1, rows)], 1).astype(np.float32).tolist(), history=history, prompt=prompt)
    check(run(ctx, x, **rules), *definition(x, **rules))
    check(run(ctx, np.ascontiguousarray(x[:, :36]), **rules), *definition(x[:, :36], **rules))   # four at a time


@pytest.mark.parametrize("rows,n,hist,nbias,n_masks,off", [(300, 4000, 200, 9, 4, 0), (3, 70000, 4000, 50, 2, 5), (5, 248320, 0, 4, 2, 0), (9, 248320, 2000, 0, 0, 3), (64, 60001, 300, 3, 0, 0),
                                                           (100, 32768, 900, 40, 6, 0)])
def test_pieces_of_every_size(ctx, rows, n, hist, nbias, n_masks, off):
    """Whole and broken pieces of 2048, 4096, 8192 and 16384 logits, one wave of them and several."""
    test_four_at_a_time_give_the_bits_of_one(ctx, rows, n, hist, nbias, n_masks, off)


def test_pieces_against_the_formula(ctx):
    for rows, n, hist in ((300, 4000, 20), (40, 16400, 30), (2, 20000, 300)):
        x, rules = case(rows, n, hist, 6, n, n_masks=3)
        check(run(ctx, x, **rules), *definition(x, **rules))
