"""Times one matvec (or prefill GEMM, or one of the steps between them) on cuda:0 and prints one JSON line; also the command ncu profiles.

    python -m qwengine_b200.single --fmt IQ3_XXS --M 17408 --K 5120 --nb 1 [--copies 8] [--reps 5] [--no-pdl]
    python -m qwengine_b200.single --op prefill --fmt Q4_K --M 17408 --K 5120 --tokens 1024
    python -m qwengine_b200.single --op mx4 --M 17408 --K 5120 --tokens 2048          # 4-bit weights and activations, the quantizer included
    python -m qwengine_b200.single --op heads --tokens 8192                           # 24 + 4 heads of 256: norm, rotation
    python -m qwengine_b200.single --op logits --tokens 128 --history 8000            # penalties and a mask on rows of 248320
    python -m qwengine_b200.single --op i8 --M 17408 --K 5120 --tokens 2048           # 8-bit integer weights and activations, the quantizer included
    python -m qwengine_b200.single --op attention --tokens 4096 --history 28672       # 24 + 4 heads of 256 over a paged cache; --seqs 32 --tokens 1: decoding

Matvec: `copies` distinct resident matrices (random valid blocks; by default enough to exceed 1.5 GB, far beyond L2)
are recorded as one pass and replayed as a CUDA graph, so host launch overhead does not count.
"""
import argparse
import json

import torch

from . import Context, PagedCache, Pass, formats as F


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--op", default="gemv", choices=["gemv", "prefill", "mx4", "heads", "logits", "i8", "attention"])
    ap.add_argument("--fmt", default="IQ3_XXS")
    ap.add_argument("--M", type=int, default=17408)
    ap.add_argument("--K", type=int, default=5120)
    ap.add_argument("--nb", type=int, default=1)
    ap.add_argument("--tokens", type=int, default=1024)
    ap.add_argument("--history", type=int, default=1000)
    ap.add_argument("--seqs", type=int, default=1)
    ap.add_argument("--copies", type=int, default=0)
    ap.add_argument("--reps", type=int, default=5)
    ap.add_argument("--no-pdl", action="store_true")
    a = ap.parse_args()
    ctx = Context(0)
    ctx.set_pdl(not a.no_pdl)
    f = F.get(a.fmt)
    rb = f.row_bytes(a.K)
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    if a.op == "gemv":
        copies = a.copies or max(4, int(1.5e9 // (a.M * rb)) + 1)
        ps = Pass(ctx, max_nb=a.nb)
        xin, xq, yb = ps.buffer_f32(a.K), ps.buffer_q8k(a.K), ps.buffer_f32(a.M)
        ps.quantize(xin, 0, a.K, xq)
        for _ in range(copies):
            w = torch.randint(0, 256, (a.M, rb), dtype=torch.uint8, device="cuda")
            ps.gemv(ps.matrix_device(f, w, a.K), xq, yb, 0)
        ps.buffer_tensor(xin).normal_()
        for _ in range(2):
            ps.run(a.nb)
        torch.cuda.synchronize()
        e0.record()
        for _ in range(a.reps):
            ps.run(a.nb)
        e1.record()
        torch.cuda.synchronize()
        ctx.check()
        us = e0.elapsed_time(e1) * 1e3 / (a.reps * copies)
        print(json.dumps({"op": "gemv", "fmt": f.name, "M": a.M, "K": a.K, "nb": a.nb, "copies": copies, "us_per_launch": round(us, 2),
                          "weight_GBps": round(a.M * rb / us / 1e3, 1)}))
    elif a.op == "prefill":
        w = torch.randint(0, 256, (a.M, rb), dtype=torch.uint8, device="cuda")
        x = torch.randn((a.tokens, a.K), device="cuda", dtype=torch.bfloat16)
        y = torch.empty((a.tokens, a.M), device="cuda")
        for _ in range(2):
            ctx.gemm_prefill(f, w, x, a.K, out=y)
        torch.cuda.synchronize()
        e0.record()
        for _ in range(a.reps):
            ctx.gemm_prefill(f, w, x, a.K, out=y)
        e1.record()
        torch.cuda.synchronize()
        ctx.check()
        ms = e0.elapsed_time(e1) / a.reps
        print(json.dumps({"op": "prefill", "fmt": f.name, "M": a.M, "K": a.K, "tokens": a.tokens, "ms": round(ms, 4),
                          "TFLOPs": round(2.0 * a.tokens * a.M * a.K / ms / 1e9, 1)}))
    else:
        STEPS[a.op](ctx, a)


def timed(calls, reps):
    """Microseconds a call, the calls captured in one graph so that their launches do not count."""
    calls[0]()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for c in calls:
            c()
    graph.replay()
    torch.cuda.synchronize()
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    e0.record()
    for _ in range(reps):
        graph.replay()
    e1.record()
    torch.cuda.synchronize()
    return e0.elapsed_time(e1) * 1e3 / (reps * len(calls))


def mx4(ctx, a):
    copies = a.copies or int(3e8 // (a.M * a.K * 17 // 32)) + 1
    Ws = [ctx.quantize_mx4(torch.randn((a.M, a.K), device="cuda", dtype=torch.bfloat16)) for _ in range(copies)]
    x = torch.randn((a.tokens, a.K), device="cuda", dtype=torch.bfloat16)
    y = torch.empty((a.tokens, a.M), device="cuda", dtype=torch.bfloat16)
    us = timed([lambda W=W: ctx.gemm_mx4(W, x, out=y) for W in Ws], a.reps)
    ctx.check()
    print(json.dumps({"op": "mx4", "M": a.M, "K": a.K, "tokens": a.tokens, "copies": copies, "us": round(us, 2), "weight_GBps": round(a.M * a.K * 17 / 32 / us / 1e3, 1),
                      "TFLOPs": round(2.0 * a.tokens * a.M * a.K / us / 1e6, 1)}))


def heads(ctx, a):
    copies = a.copies or int(3e8 // (a.tokens * 13312 * 4)) + 1
    xs = [torch.randn((a.tokens, 12288 + 1024), device="cuda") for _ in range(min(copies, 40))]
    pos = torch.arange(a.tokens, device="cuda", dtype=torch.int32)
    freq = 1e7 ** (-torch.arange(0, 64, 2, device="cuda", dtype=torch.float64) / 64)
    w = torch.ones(256, device="cuda")
    us = timed([lambda x=x: ctx.qk_norm_rope(x[:, :12288].unflatten(1, (24, 512))[:, :, :256], x[:, 12288:].unflatten(1, (4, 256)), pos, freq, w, w, kind=2) for x in xs], a.reps)
    print(json.dumps({"op": "heads", "tokens": a.tokens, "us": round(us, 2), "GBps": round(a.tokens * 28 * 256 * 6 / us / 1e3, 1)}))


def logits(ctx, a):
    n = 248320
    x = torch.randn((a.tokens, n), device="cuda")
    y = torch.empty_like(x)
    rules = dict(penalties=torch.tensor([[1.1, 0.1, 0.1]] * a.tokens, device="cuda"), history=torch.randint(0, n, (a.tokens * a.history,), device="cuda", dtype=torch.int32),
                 history_begin=torch.arange(a.tokens + 1, device="cuda") * a.history, prompt_len=torch.full((a.tokens,), a.history // 2, device="cuda", dtype=torch.int32),
                 masks=torch.randint(-2 ** 31, 2 ** 31, (a.tokens, n // 32), device="cuda").to(torch.int32))
    us = timed([lambda: ctx.adjust_logits(x, out=y, **rules)] * 4, a.reps)
    print(json.dumps({"op": "logits", "rows": a.tokens, "history": a.history, "us": round(us, 2), "GBps": round(a.tokens * (n * 8.125 + a.history * 4) / us / 1e3, 1)}))


def i8(ctx, a):
    copies = a.copies or int(3e8 // (a.M * a.K)) + 1
    Ws = [ctx.quantize_i8(torch.randn((a.M, a.K), device="cuda", dtype=torch.bfloat16)) for _ in range(copies)]
    x = torch.randn((a.tokens, a.K), device="cuda", dtype=torch.bfloat16)
    y = torch.empty((a.tokens, a.M), device="cuda", dtype=torch.bfloat16)
    us = timed([lambda W=W: ctx.gemm_i8(W, x, out=y) for W in Ws], a.reps)
    ctx.check()
    print(json.dumps({"op": "i8", "M": a.M, "K": a.K, "tokens": a.tokens, "copies": copies, "us": round(us, 2), "weight_GBps": round(a.M * a.K / us / 1e3, 1),
                      "TOPs": round(2.0 * a.tokens * a.M * a.K / us / 1e6, 1)}))


def attention(ctx, a):
    text, page = a.tokens + a.history, 64
    per = (text + page - 1) // page
    copies = a.copies or int(3e8 // (a.seqs * text * 4096)) + 1
    caches = [PagedCache(*(torch.randn((a.seqs * per, page, 4, 256), device="cuda", dtype=torch.bfloat16) for _ in range(2))) for _ in range(min(copies, 40))]
    table = torch.arange(a.seqs * per, device="cuda", dtype=torch.int32).view(a.seqs, per)
    lengths = torch.full((a.seqs,), text, device="cuda", dtype=torch.int32)
    begin = torch.arange(a.seqs + 1, device="cuda", dtype=torch.int32) * a.tokens
    x = torch.randn((a.seqs * a.tokens, 24, 256), device="cuda", dtype=torch.bfloat16)
    y = torch.empty_like(x)
    us = timed([lambda c=c: ctx.attention(c, x, table, lengths, begin, out=y) for c in caches], a.reps)
    ctx.check()
    pairs = a.seqs * (a.tokens * a.history + a.tokens * (a.tokens + 1) // 2)
    print(json.dumps({"op": "attention", "seqs": a.seqs, "tokens": a.tokens, "history": a.history, "copies": len(caches), "us": round(us, 2),
                      "GBps": round((a.seqs * text * 4096 + x.numel() * 4) / us / 1e3, 1), "TFLOPs": round(4 * pairs * 24 * 256 / us / 1e6, 1)}))


STEPS = {"mx4": mx4, "heads": heads, "logits": logits, "i8": i8, "attention": attention}


if __name__ == "__main__":
    main()
