"""Operators round the products of a token step and of a prompt chunk, as cases that can be timed and compared.

A case is a dict of plain values; `kind` names one of four uses:

  heads    query and key heads behind their projections: RMSNorm of each head, rotation by position
  logits   what lies between the output head and the top-k: penalties for repeated tokens, biases, grammar masks
  rows4    rows of values to microscaled 4-bit floating point and back (blocks of 32 E2M1 elements, E8M0 scales)
  product  activations quantized to that format, times weights held in it

Sizes are those of the 27B-shaped decode pass (hidden 5120, FFN 17408, 24 query and 4 key heads of 256 of which 64 rotate,
248320 logits) and ragged ones round them.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
OUT_KIND = {"f32": 0, "f16": 1, "bf16": 2}
HIDDEN, FF, PROJ, VOCAB = 5120, 17408, 16384, 248320
EPS = 1e-6
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # one decoded token: q and gate lie side by side in the projection's output, k behind it
        dict(name="heads_token", kind="heads", rows=1, nq=24, nk=4, d=256, rot=64, gate=True, adjacent=False, pos=40000, src="f32", dst="f32"),
        # a ragged chunk of a model with 96-wide heads in three to one groups, rotated in adjacent pairs, far into a long text
        dict(name="heads_ragged", kind="heads", rows=333, nq=15, nk=5, d=96, rot=48, gate=False, adjacent=True, pos=1000003, src="bf16", dst="bf16"),
        # a long prompt chunk from the prefill's fp32 outputs to 16-bit queries and keys
        dict(name="heads_chunk", kind="heads", rows=8192, nq=24, nk=4, d=256, rot=64, gate=True, adjacent=False, pos=0, src="f32", dst="bf16"),
        # sampling one token: a prompt and a few generated tokens, no grammar
        dict(name="logits_token", kind="logits", rows=1, n=VOCAB, prompt=512, made=88, bias=0, masks=0, pad=0),
        # eight sequences with biases, half of them under a grammar, rows at an odd distance
        dict(name="logits_grammar", kind="logits", rows=8, n=100001, prompt=3000, made=1000, bias=300, masks=4, pad=2),
        # a full batch with long texts behind it
        dict(name="logits_batch", kind="logits", rows=128, n=VOCAB, prompt=16000, made=4000, bias=32, masks=64, pad=0),
        # a few activation rows
        dict(name="rows4_few", kind="rows4", rows=77, k=HIDDEN, src="f32", dst="f32"),
        # a weight matrix brought to the format when a model is loaded
        dict(name="rows4_weights", kind="rows4", rows=FF, k=HIDDEN, src="bf16", dst="bf16"),
        # one token through an up projection
        dict(name="product_token", kind="product", tokens=1, m=FF, k=HIDDEN, src="f32", dst="f32"),
        # seven columns of a speculative verify step through a down projection
        dict(name="product_verify", kind="product", tokens=7, m=HIDDEN, k=FF, src="f32", dst="f32"),
        # a short ragged prompt through the input projection
        dict(name="product_ragged", kind="product", tokens=333, m=PROJ, k=HIDDEN, src="f32", dst="f32"),
        # a long prompt chunk
        dict(name="product_chunk", kind="product", tokens=2048, m=FF, k=HIDDEN, src="bf16", dst="bf16"),
    ]


def draw(rng):
    log = lambda lo, hi: min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))  # noqa: E731
    kind = rng.choice(("heads", "logits", "rows4", "product", "product"))
    src, dst = rng.choice((("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16")))
    if kind == "heads":
        d = rng.choice((64, 80, 96, 128, 192, 256))
        nk = rng.choice((1, 2, 4, 5, 8))
        nq = nk * rng.choice((1, 3, 4, 6))
        rows = log(1, max(1, min(8192, 8192 * 28 * 256 // ((nq + nk) * d))))
        rot = rng.choice((d, d // 2, d // 4))
        return dict(kind=kind, rows=rows, nq=nq, nk=nk, d=d, rot=rot, gate=rng.random() < 0.5, adjacent=rng.random() < 0.5, pos=log(1, 1 << 20), src=src, dst=dst)
    if kind == "logits":
        rows = log(1, 128)
        return dict(kind=kind, rows=rows, n=log(1000, VOCAB), prompt=log(1, 16000), made=log(1, 4000), bias=rng.choice((0, 1, 32, 300)),
                    masks=rng.choice((0, 1, rows)), pad=rng.choice((0, 0, 1, 2, 3)))
    if kind == "rows4":
        return dict(kind=kind, rows=log(1, FF), k=32 * log(1, HIDDEN // 32), src=src, dst=dst)
    while True:
        tokens, m, k = log(1, 2048), log(96, FF), 32 * log(8, FF // 32)
        if tokens * m * k <= 2048 * FF * HIDDEN and m * k <= FF * HIDDEN:
            return dict(kind=kind, tokens=tokens, m=m, k=k, src=src, dst=dst)


# ---- inputs ----------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + 17)
    return {"heads": _prepare_heads, "logits": _prepare_logits, "rows4": _prepare_rows4, "product": _prepare_product}[case["kind"]](case, g)


def _normal(shape, g):
    return torch.randn(shape, generator=g, device="cuda")


def _prepare_heads(c, g):
    rows, d = c["rows"], c["d"]
    width = c["nq"] * d * (2 if c["gate"] else 1) + c["nk"] * d
    # projections' outputs: a scale of its own for each channel
    x = (_normal((rows, width), g) * torch.exp(0.5 * _normal((1, width), g))).to(DTYPES[c["src"]])
    q = x[:, :width - c["nk"] * d].unflatten(1, (c["nq"], -1))[:, :, :d]
    k = x[:, width - c["nk"] * d:].unflatten(1, (c["nk"], d))
    start = c["pos"] + int(torch.randint(0, 1000, (1,), generator=g, device="cuda"))
    positions = torch.arange(start, start + rows, device="cuda", dtype=torch.int32)
    inv_freq = 1e7 ** (-torch.arange(0, c["rot"], 2, device="cuda", dtype=torch.float64) / c["rot"])
    return dict(case=c, q=q, k=k, positions=positions, inv_freq=inv_freq, wq=1 + 0.3 * _normal((d,), g), wk=1 + 0.3 * _normal((d,), g))


def _prepare_logits(c, g):
    rows, n = c["rows"], c["n"]
    logits = (4 * _normal((rows, n + c["pad"]), g))[:, :n]
    uniform = lambda *s: torch.rand(s, generator=g, device="cuda")  # noqa: E731
    # histories of different lengths; token ids fall off like a text's, so that many occur again
    prompt = (c["prompt"] * (0.25 + 0.75 * uniform(rows))).long().clamp(min=1)
    made = (c["made"] * (0.25 + 0.75 * uniform(rows))).long()
    begin = torch.zeros(rows + 1, dtype=torch.int64, device="cuda")
    begin[1:] = torch.cumsum(prompt + made, 0)
    total = int(begin[-1])
    history = torch.exp(uniform(total) * math.log(n)).long().clamp(max=n) - 1
    penalties = torch.stack([1 + 0.3 * uniform(rows), 0.5 * uniform(rows), 0.5 * uniform(rows)], 1)
    s = dict(case=c, logits=logits, history=history.to(torch.int32), begin=begin, prompt=prompt.to(torch.int32), penalties=penalties.contiguous(),
             bias_ids=None, bias_values=None, bias_begin=None, masks=None, mask_of_row=None)
    if c["bias"]:
        s["bias_ids"] = torch.randint(0, n, (rows * c["bias"],), generator=g, device="cuda", dtype=torch.int32)
        s["bias_values"] = 3 * _normal((rows * c["bias"],), g)
        s["bias_begin"] = torch.arange(rows + 1, device="cuda", dtype=torch.int64) * c["bias"]
    if c["masks"]:
        # grammars that leave about one token in sixteen; rows behind the last mask run free
        words = (n + 31) // 32
        bits = lambda: torch.randint(-2 ** 31, 2 ** 31, (c["masks"], words), generator=g, device="cuda", dtype=torch.int64)  # noqa: E731
        s["masks"] = (bits() & bits() & bits() & bits()).to(torch.int32)
        r = torch.arange(rows, device="cuda", dtype=torch.int32)
        s["mask_of_row"] = torch.where(r < c["masks"], r, -1).to(torch.int32)
    return s


def _prepare_rows4(c, g):
    x = _normal((c["rows"], c["k"]), g) * torch.exp(_normal((c["rows"], 1), g))
    return dict(case=c, x=x.to(DTYPES[c["src"]]))


def _prepare_product(c, g):
    m, k = c["m"], c["k"]
    w = _normal((m, k), g) * (k ** -0.5 * torch.exp(0.5 * _normal((m, 1), g)))
    code, e = _codes(w)
    del w
    codes = (code[:, 0::2] | (code[:, 1::2] << 4)).contiguous()
    scales = (e + 127).to(torch.uint8)
    # activations: some channels are much larger than the others
    x = _normal((c["tokens"], k), g) * torch.exp(_normal((1, k), g))
    return dict(case=c, codes=codes, scales=scales, tiles=_tiles(scales), x=x.to(DTYPES[c["src"]]))


def _tiles(scales):
    """The library's order of a matrix's scale bytes: tiles of 128 rows x 4 blocks, zeros behind the last row and block."""
    rows, blocks = scales.shape
    full = torch.zeros(((rows + 127) // 128 * 128, (blocks + 3) // 4 * 4), dtype=torch.uint8, device=scales.device)
    full[:rows, :blocks] = scales
    return full.view(full.shape[0] // 128, 4, 32, full.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).contiguous()


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
    return {"heads": _heads, "logits": _logits, "rows4": _rows4, "product": _product}[state["case"]["kind"]](state)


def _heads(s):
    c = s["case"]
    if own:
        q, k = _context().qk_norm_rope(s["q"], s["k"], s["positions"], s["inv_freq"], s["wq"], s["wk"], eps=EPS, adjacent=c["adjacent"], kind=OUT_KIND[c["dst"]])
        return {"q": q, "k": k}
    angle = s["positions"].double()[:, None, None] * s["inv_freq"]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    return {"q": _norm_rotate(s["q"], s["wq"], cos, sin, c), "k": _norm_rotate(s["k"], s["wk"], cos, sin, c)}


def _norm_rotate(x, w, cos, sin, c):
    x = x.float()
    z = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    rot = c["rot"]
    y = z.clone()
    if c["adjacent"]:
        a, b = z[..., 0:rot:2], z[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = z[..., :rot // 2], z[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = a * cos - b * sin, b * cos + a * sin
    return y.to(DTYPES[c["dst"]])


def _logits(s):
    if own:
        return _context().adjust_logits(s["logits"], penalties=s["penalties"], history=s["history"], history_begin=s["begin"], prompt_len=s["prompt"],
                                        bias_ids=s["bias_ids"], bias_values=s["bias_values"], bias_begin=s["bias_begin"], masks=s["masks"],
                                        mask_of_row=s["mask_of_row"])
    x = s["logits"].float()
    rows, n = x.shape
    at, first = _places(s["begin"], s["history"], n)
    made = first >= torch.repeat_interleave(s["prompt"].long(), s["begin"][1:] - s["begin"][:-1])
    seen = torch.bincount(at, minlength=rows * n).view(rows, n) > 0
    count = torch.bincount(at[made], minlength=rows * n).view(rows, n).float()
    rep, freq, pres = (s["penalties"][:, i:i + 1] for i in range(3))
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x) - freq * count - pres * (count > 0)
    if s["bias_ids"] is not None:
        at, _ = _places(s["bias_begin"], s["bias_ids"], n)
        last = torch.full((rows * n,), -1, dtype=torch.int64, device=x.device)
        last.scatter_reduce_(0, at, torch.arange(at.numel(), device=x.device), "amax")
        last = last.view(rows, n)
        x = x + torch.where(last >= 0, s["bias_values"][last.clamp(min=0)], 0.0)
    if s["masks"] is not None:
        bit = (s["masks"].unsqueeze(-1) >> torch.arange(32, device=x.device, dtype=torch.int32)) & 1
        allowed = bit.flatten(1)[:, :n][s["mask_of_row"].long().clamp(min=0)] != 0
        x = torch.where(allowed | (s["mask_of_row"] < 0)[:, None], x, -math.inf)
    return x


def _places(begin, ids, n):
    """Where each entry of the rows' lists lies in [rows, n], and its number in its row's list."""
    lengths = begin[1:] - begin[:-1]
    row = torch.repeat_interleave(torch.arange(lengths.numel(), device=ids.device), lengths)
    return row * n + ids.long(), torch.arange(ids.numel(), device=ids.device) - begin[row]


def _codes(x):
    """E2M1 codes (sign in bit 3) of every element and the power of two of every block of 32."""
    b = x.float().unflatten(1, (-1, 32))
    e = (torch.frexp(b.abs().amax(-1)).exponent - 3).clamp(-127, 127)
    a = torch.ldexp(b, -e.unsqueeze(-1))
    m = a.abs()
    code = (m > 0.25).to(torch.uint8) + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (m > 5)
    return (code + 8 * (a < 0)).flatten(1).to(torch.uint8), e


def _values(code, e):
    level = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=code.device)
    return torch.ldexp(level[code.long()].unflatten(1, (-1, 32)), e.unsqueeze(-1)).flatten(1)


def _rows4(s):
    if own:
        ctx = _context()
        return ctx.dequant_mx4(ctx.quantize_mx4(s["x"]), kind=OUT_KIND[s["case"]["dst"]])
    return _values(*_codes(s["x"])).to(DTYPES[s["case"]["dst"]])


def _product(s):
    if own:
        import qwengine_b200 as q
        return _context().gemm_mx4(q.Mx4(s["codes"], s["tiles"]), s["x"], kind=OUT_KIND[s["case"]["dst"]])
    code = torch.stack([s["codes"] & 15, s["codes"] >> 4], -1).flatten(1)
    w = _values(code, s["scales"].int() - 127)
    return (_values(*_codes(s["x"])) @ w.t()).to(DTYPES[s["case"]["dst"]])


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    c = case
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if c["kind"] == "heads":
        n = c["rows"] * (c["nq"] + c["nk"]) * c["d"]
        return {"bytes": n * (size[c["src"]] + size[c["dst"]]) + 8 * c["d"] + 4 * c["rows"] + 4 * c["rot"], "flops": 8 * n}
    if c["kind"] == "logits":
        n = c["rows"] * c["n"]
        listed_bytes = c["rows"] * (0.625 * 4 * (c["prompt"] + c["made"]) + 8 * c["bias"] + 32)
        return {"bytes": 8 * n + listed_bytes + min(c["masks"], c["rows"]) * c["n"] / 8, "flops": 4 * n}
    if c["kind"] == "rows4":
        n = c["rows"] * c["k"]
        return {"bytes": n * (size[c["src"]] + size[c["dst"]]), "flops": 4 * n}
    b, m, k = c["tokens"], c["m"], c["k"]
    return {"bytes": m * k * 17 / 32 + b * k * size[c["src"]] + b * m * size[c["dst"]], "flops": 2 * b * m * k}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"heads": _exact_heads, "logits": _exact_logits, "rows4": _exact_rows4, "product": _exact_product}[case["kind"]](s)


def _exact_heads(s):
    c = s["case"]
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), torch.outer(s["positions"].double(), s["inv_freq"])).unsqueeze(1)
    out = {}
    for name, x, w in (("q", s["q"], s["wq"]), ("k", s["k"], s["wk"])):
        x = x.double()
        z = x / (x.square().sum(-1, keepdim=True) / c["d"] + EPS).sqrt() * w.double()
        head, rest = z[..., :c["rot"]], z[..., c["rot"]:]
        pairs = head.unflatten(-1, (-1, 2)) if c["adjacent"] else head.unflatten(-1, (2, -1)).transpose(-1, -2)
        turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        turned = turned if c["adjacent"] else turned.transpose(-1, -2)
        out[name] = torch.cat([turned.flatten(-2), rest], -1)
    return out


def _exact_logits(s):
    x = s["logits"].double().cpu()
    host = {k: v.cpu() for k, v in s.items() if isinstance(v, torch.Tensor)}
    begin, bias_begin = host["begin"].tolist(), host["bias_begin"].tolist() if "bias_begin" in host else None
    for r in range(x.shape[0]):
        tokens = host["history"][begin[r]:begin[r + 1]].long()
        rep, freq, pres = host["penalties"][r].double().tolist()
        known = torch.unique(tokens)
        v = x[r, known]
        x[r, known] = torch.where(v > 0, v / rep, v * rep)
        made, times = torch.unique(tokens[int(host["prompt"][r]):], return_counts=True)
        x[r, made] -= freq * times.double() + pres
        if bias_begin is not None:
            ids = host["bias_ids"][bias_begin[r]:bias_begin[r + 1]].tolist()
            last = dict(zip(ids, host["bias_values"][bias_begin[r]:bias_begin[r + 1]].tolist()))
            x[r, list(last)] += torch.tensor(list(last.values()), dtype=torch.float64)
        if "masks" in host and int(host["mask_of_row"][r]) >= 0:
            bits = np.unpackbits(host["masks"][int(host["mask_of_row"][r])].numpy().view(np.uint8), bitorder="little")
            x[r, torch.from_numpy(bits[:x.shape[1]] == 0)] = -math.inf
    return x


def _exact_rounded(x):
    """Nearest value of the format: steps of 1/2 below two, of one below four, of two from there on; halves to even; at most 6."""
    b = x.double().unflatten(1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    p = (((top.view(torch.int64) >> 52) - 2).clamp(min=1023 - 127) << 52).view(torch.float64)   # the power of two below, over four
    a = b / p
    step = torch.where(a.abs() < 2, 0.5, torch.where(a.abs() < 4, 1.0, 2.0))
    return ((torch.round(a / step) * step).clamp(-6, 6) * p).flatten(1)


def _exact_rows4(s):
    return _exact_rounded(s["x"])


def _exact_product(s):
    low, high = s["codes"] & 15, s["codes"] >> 4
    code = torch.stack([low, high], -1).flatten(1).long()
    exponent, mantissa = (code >> 1) & 3, code & 1
    magnitude = torch.where(exponent == 0, mantissa * 0.5, (1 + 0.5 * mantissa) * torch.exp2(exponent.double() - 1))
    w = torch.where(code >= 8, -magnitude, magnitude).unflatten(1, (-1, 32)) * torch.exp2(s["scales"].double() - 127).unsqueeze(-1)
    return _exact_rounded(s["x"]) @ w.flatten(1).t()
