"""Operators of an attention layer between and in its products, as cases that can be timed and compared.

A case is a dict of plain values; `kind` names one of four uses:

  append     a chunk's new keys and values into the pages of a cache
  attention  the chunk's queries over the paged keys and values of their sequences, each query up to its own token
  rows8      rows of values to 8-bit integers with one scale a row
  product8   activations quantized so (a scale for each token), times weights held so (a scale for each output channel)

Sizes are those of the 27B-shaped decode pass (hidden 5120, FFN 17408, input projection 16384, 24 query and 4 key heads of 256) and ragged
ones round them.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
OUT_KIND = {"f32": 0, "f16": 1, "bf16": 2}
HIDDEN, FF, PROJ = 5120, 17408, 16384
LEAST_SCALE = 2.0 ** -126


def listed():
    b27 = dict(nq=24, nk=4, d=256)
    return [
        # one decoded token behind a short text
        dict(name="attention_token", kind="attention", seqs=1, new=1, past=699, ragged=False, page=16, dtype="bf16", **b27),
        # a batch of decoding sequences of very different lengths
        dict(name="attention_batch", kind="attention", seqs=32, new=1, past=32000, ragged=True, page=16, dtype="bf16", **b27),
        # seven drafted tokens verified at the end of one very long text
        dict(name="attention_verify", kind="attention", seqs=1, new=7, past=131065, ragged=False, page=64, dtype="bf16", **b27),
        # chunks of several prompts stepped together, 96-wide heads in groups of three
        dict(name="attention_ragged", kind="attention", seqs=5, new=333, past=1500, ragged=True, page=32, dtype="f16", nq=15, nk=5, d=96),
        # a long prompt's last chunk
        dict(name="attention_chunk", kind="attention", seqs=1, new=4096, past=28672, ragged=False, page=128, dtype="bf16", **b27),
        # one token's keys and values as the projections leave them
        dict(name="append_token", kind="append", seqs=1, new=1, past=699, ragged=False, page=16, dtype="bf16", src="f32", **b27),
        # a long prompt chunk's
        dict(name="append_chunk", kind="append", seqs=1, new=8192, past=0, ragged=False, page=16, dtype="bf16", src="f32", **b27),
        # a few activation rows
        dict(name="rows8_few", kind="rows8", rows=77, k=HIDDEN, src="f32"),
        # a weight matrix brought to the format when a model is loaded
        dict(name="rows8_weights", kind="rows8", rows=FF, k=HIDDEN, src="bf16"),
        # one token through an up projection
        dict(name="product8_token", kind="product8", tokens=1, m=FF, k=HIDDEN, src="f32", dst="f32"),
        # a short ragged prompt through the input projection
        dict(name="product8_ragged", kind="product8", tokens=333, m=PROJ, k=HIDDEN, src="f32", dst="f32"),
        # a long prompt chunk
        dict(name="product8_chunk", kind="product8", tokens=2048, m=FF, k=HIDDEN, src="bf16", dst="bf16"),
    ]


def draw(rng):
    log = lambda lo, hi: min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))  # noqa: E731
    kind = rng.choice(("attention", "attention", "attention", "append", "rows8", "product8", "product8"))
    src, dst = rng.choice((("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16")))
    while kind in ("attention", "append"):
        nk = rng.choice((1, 2, 4, 5, 8))
        c = dict(kind=kind, nq=nk * rng.choice((1, 3, 4, 6)), nk=nk, d=rng.choice((64, 80, 96, 128, 192, 256)), page=rng.choice((16, 32, 64, 128)),
                 dtype=rng.choice(("bf16", "f16")), ragged=rng.random() < 0.5)
        if rng.random() < 0.5:   # decoding, with up to seven drafted tokens
            c.update(seqs=log(1, 64), new=rng.choice((1, 1, 2, 4, 8)), past=log(1, 131072))
        else:
            c.update(seqs=log(1, 6), new=log(9, 4096), past=log(1, 32768) if rng.random() < 0.5 else 0)
        longest = c["new"] + c["past"]
        if c["seqs"] * longest * nk * c["d"] > 32 * 32001 * 1024 or c["seqs"] * c["new"] * c["nq"] * longest > 4096 * 24 * 32768:
            continue
        if c["seqs"] * c["new"] * c["nq"] * longest * c["d"] > 4096 * 24 * 32768 * 256:
            continue
        if kind == "append":
            c["src"] = rng.choice(("f32", c["dtype"]))
        return c
    if kind == "rows8":
        return dict(kind=kind, rows=log(1, FF), k=log(8, HIDDEN), src=src)
    while True:
        tokens, m, k = log(1, 2048), log(96, FF), log(256, FF)
        if tokens * m * k <= 2048 * FF * HIDDEN and m * k <= FF * HIDDEN:
            return dict(kind=kind, tokens=tokens, m=m, k=k, src=src, dst=dst)


def _sequences(c):
    """(new tokens, tokens in all) of each sequence; ragged: from all down to a tenth, in no order."""
    out = []
    for s in range(c["seqs"]):
        f = 1 - 0.9 * (s * 0.6180339887 % 1) if c["ragged"] else 1.0
        g = 1 - 0.95 * (s * 0.7548776662 % 1) if c["ragged"] else 1.0
        new = max(1, int(c["new"] * f))
        out.append((new, new + int(c["past"] * g)))
    return out


# ---- inputs ----------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + 29)
    return {"attention": _prepare_cache, "append": _prepare_cache, "rows8": _prepare_rows8, "product8": _prepare_product8}[case["kind"]](case, g)


def _normal(shape, g, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _prepare_cache(c, g):
    plan, page, dtype = _sequences(c), c["page"], DTYPES[c["dtype"]]
    need = [(total + page - 1) // page for _, total in plan]
    # the sequences' pages lie in no order among each other and some pages are nobody's
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((c["seqs"], max(need)), dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    begin = [0]
    for new, _ in plan:
        begin.append(begin[-1] + new)
    rows = begin[-1]
    shape = (pages, page, c["nk"], c["d"])
    s = dict(case=c, k_cache=_normal(shape, g, dtype), v_cache=_normal(shape, g, dtype), table=table, rows=rows,
             lengths=torch.tensor([t for _, t in plan], dtype=torch.int32, device="cuda"), begin=torch.tensor(begin, dtype=torch.int32, device="cuda"),
             most=max(n for n, _ in plan))
    if c["kind"] == "attention":
        # some queries look at a few keys only, others at all
        s["q"] = (_normal((rows, c["nq"], c["d"]), g) * torch.exp(0.5 * _normal((rows, c["nq"], 1), g))).to(dtype)
    else:
        src = DTYPES[c["src"]]
        both = _normal((rows, 2 * c["nk"] * c["d"]), g).to(src)   # keys and values side by side, as one projection leaves them
        s["k"], s["v"] = both.unflatten(1, (2, c["nk"], c["d"])).unbind(1)
    return s


def _prepare_rows8(c, g):
    x = _normal((c["rows"], c["k"]), g) * torch.exp(_normal((c["rows"], 1), g))
    return dict(case=c, x=x.to(DTYPES[c["src"]]))


def _prepare_product8(c, g):
    m, k = c["m"], c["k"]
    w = _normal((m, k), g) * (k ** -0.5 * torch.exp(0.5 * _normal((m, 1), g)))
    codes, scales = _codes8(w)
    del w
    # rows of codes begin at multiples of 16 bytes
    room = torch.zeros((m, (k + 15) // 16 * 16), dtype=torch.int8, device="cuda")
    room[:, :k] = codes
    # activations: some channels are larger than the others
    x = _normal((c["tokens"], k), g) * torch.exp(0.5 * _normal((1, k), g))
    return dict(case=c, codes=room[:, :k], scales=scales, x=x.to(DTYPES[c["src"]]))


# ---- one pass --------------------------------------------------------------------------------------------------------

_contexts = {}


def _context():
    """One context per device and process, as the library wants it."""
    import qwengine_b200 as q
    at = torch.cuda.current_device()
    if at not in _contexts:
        _contexts[at] = q.Context(at)
    return _contexts[at]


def run(state):
    return {"attention": _attention, "append": _append, "rows8": _rows8, "product8": _product8}[state["case"]["kind"]](state)


def _append(s):
    c = s["case"]
    if own:
        import qwengine_b200 as q
        _context().cache_append(q.PagedCache(s["k_cache"], s["v_cache"]), s["k"], s["v"], s["table"], s["lengths"], s["begin"])
        return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    lengths, begin = s["lengths"].long(), s["begin"].long()
    new = begin[1:] - begin[:-1]
    row = torch.arange(s["rows"], device="cuda")
    seq = torch.repeat_interleave(torch.arange(c["seqs"], device="cuda"), new, output_size=s["rows"])
    at = (lengths - new)[seq] + row - begin[seq]
    page, slot = s["table"].long()[seq, at // c["page"]], at % c["page"]
    s["k_cache"][page, slot] = s["k"].to(s["k_cache"].dtype)
    s["v_cache"][page, slot] = s["v"].to(s["v_cache"].dtype)
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _attention(s):
    c = s["case"]
    if own:
        import qwengine_b200 as q
        return _context().attention(q.PagedCache(s["k_cache"], s["v_cache"]), s["q"], s["table"], s["lengths"], s["begin"])
    lengths, begin = s["lengths"].long(), s["begin"].long()
    new = begin[1:] - begin[:-1]
    seqs, nk, group, d = c["seqs"], c["nk"], c["nq"] // c["nk"], c["d"]
    table = s["table"].long()
    keys = s["k_cache"][table].flatten(1, 2).permute(0, 2, 3, 1).float()          # [sequence, key head, element, token]
    values = s["v_cache"][table].flatten(1, 2).transpose(1, 2).float()            # [sequence, key head, token, element]
    i, j = torch.arange(s["most"], device="cuda"), torch.arange(keys.shape[-1], device="cuda")
    rows = (begin[:-1, None] + i).clamp(max=s["rows"] - 1)
    queries = s["q"][rows].float().unflatten(2, (nk, group)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    seen = j[None, None, :] <= (lengths - new)[:, None, None] + i[None, :, None]   # [sequence, new token, token]
    seen = seen & (j < lengths[:, None])[:, None, :]
    seen = seen.repeat_interleave(group, 1).unsqueeze(1)
    scores = (queries @ keys).mul_(d ** -0.5).masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    weights = scores.sub_(top).exp_()
    out = (weights @ values.masked_fill_((j >= lengths[:, None])[:, None, :, None], 0.0)) / weights.sum(-1, keepdim=True)
    out = out.unflatten(2, (-1, group)).permute(0, 2, 1, 3, 4).flatten(2, 3)       # [sequence, new token, head, element]
    return out[i[None, :] < new[:, None]].to(s["q"].dtype)


def _codes8(x):
    """8-bit integers and a scale for each row.  The scale is the largest magnitude over 127, rounded to fp32; the quotients are taken in 64 bits,
    where none that lies beside a half becomes it."""
    x = x.double()
    scale = (x.abs().amax(-1) / 127).float().clamp(min=LEAST_SCALE)
    return torch.round(x / scale.double().unsqueeze(-1)).to(torch.int8), scale


def _rows8(s):
    if own:
        m = _context().quantize_i8(s["x"])
        return {"codes": m.codes, "scales": m.scales}
    codes, scales = _codes8(s["x"])
    return {"codes": codes, "scales": scales}


def _product8(s):
    kind = s["case"]["dst"]
    if own:
        import qwengine_b200 as q
        return _context().gemm_i8(q.I8(s["codes"], s["scales"]), s["x"], kind=OUT_KIND[kind])
    codes, scale = _codes8(s["x"])
    return ((codes.float() @ s["codes"].float().t()) * scale.unsqueeze(-1) * s["scales"]).to(DTYPES[kind])


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    c = case
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if c["kind"] == "append":
        n = 2 * sum(new for new, _ in _sequences(c)) * c["nk"] * c["d"]
        return {"bytes": n * (size[c["src"]] + size[c["dtype"]]), "flops": 0}
    if c["kind"] == "attention":
        plan = _sequences(c)
        pairs = sum(new * (total - new) + new * (new + 1) // 2 for new, total in plan)
        rows, tokens = sum(new for new, _ in plan), sum(total for _, total in plan)
        return {"bytes": 4 * rows * c["nq"] * c["d"] + 4 * tokens * c["nk"] * c["d"], "flops": 4 * pairs * c["nq"] * c["d"]}
    if c["kind"] == "rows8":
        n = c["rows"] * c["k"]
        return {"bytes": n * (size[c["src"]] + 1) + 4 * c["rows"], "flops": 3 * n}
    b, m, k = c["tokens"], c["m"], c["k"]
    return {"bytes": m * k + 4 * m + b * k * size[c["src"]] + b * m * size[c["dst"]], "flops": 2 * b * m * k}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "append": _exact_append, "rows8": _exact_rows8, "product8": _exact_product8}[case["kind"]](s)


def _texts(s):
    """(sequence, first row, new tokens, tokens in all) of each sequence."""
    begin, lengths = s["begin"].tolist(), s["lengths"].tolist()
    return [(i, begin[i], begin[i + 1] - begin[i], n) for i, n in enumerate(lengths)]


def _slots(s, i, n):
    """Where sequence i's first n tokens lie among all slots of the cache."""
    page = s["case"]["page"]
    t = torch.arange(n, device="cuda")
    return s["table"][i].long()[torch.div(t, page, rounding_mode="floor")] * page + t % page


def _exact_append(s):
    out = {}
    for name, new in (("k_cache", s["k"]), ("v_cache", s["v"])):
        cache = s[name].double()
        flat = cache.flatten(0, 1)
        for i, row, count, total in _texts(s):
            flat[_slots(s, i, total)[total - count:]] = new[row:row + count].double()
        out[name] = cache
    return out


def _exact_attention(s):
    c = s["case"]
    group, out = c["nq"] // c["nk"], torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    k_slots, v_slots = s["k_cache"].flatten(0, 1), s["v_cache"].flatten(0, 1)
    for i, row, count, total in _texts(s):
        at = _slots(s, i, total)
        hidden = torch.ones((count, total), dtype=torch.bool, device="cuda").triu(total - count + 1)
        for h in range(c["nq"]):
            logits = s["q"][row:row + count, h].double() @ k_slots[at, h // group].double().t() / math.sqrt(c["d"])
            logits[hidden] = -math.inf
            out[row:row + count, h] = torch.softmax(logits, -1) @ v_slots[at, h // group].double()
    return out


def _exact_rows8(s):
    x = s["x"].double()
    largest = torch.linalg.vector_norm(x, math.inf, dim=1)
    step = torch.clamp((largest / 127).float(), min=LEAST_SCALE).double()[:, None]
    below = torch.floor(x / step)
    rest = x / step - below
    up = (rest > 0.5) | ((rest == 0.5) & (below % 2 != 0))
    return {"codes": (below + up).to(torch.int8), "scales": largest / 127}


def _exact_product8(s):
    q = _exact_rows8(s)
    step = torch.clamp(q["scales"].float(), min=LEAST_SCALE).double()
    return torch.einsum("tk,mk->tm", q["codes"].double(), s["codes"].double()) * torch.outer(step, s["scales"].double())
