"""What the entry points of the token's own steps and of the 4-bit products refuse: checked before a device is touched, so without one."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def lib():
    from qwengine_b200 import build, load_library
    build.build()
    return load_library()


CTX = C.create_string_buffer(8192)      # never looked into: every call below is refused first
P, ODD = 0x10000, 0x10002               # addresses that are only compared and checked for their alignment
ARG, UNSUPPORTED, ALIGN, NOMEM = -1, -2, -3, -6


class Heads(C.Structure):
    """q38b_heads"""
    _fields_ = [("src", C.c_void_p), ("dst", C.c_void_p), ("src_row", C.c_longlong), ("src_head", C.c_longlong), ("dst_row", C.c_longlong),
                ("dst_head", C.c_longlong), ("weight", C.c_void_p), ("n_heads", C.c_int)]


class Rules(C.Structure):
    """q38b_logit_rules"""
    _fields_ = [(n, C.c_void_p) for n in ("penalties", "history", "history_begin", "prompt_len", "bias_ids", "bias_values", "bias_begin", "masks")] + \
               [("mask_ld", C.c_longlong), ("mask_of_row", C.c_void_p)]


def heads(**kw):
    v = dict(src=P, dst=P + 4096, src_row=512, src_head=64, dst_row=512, dst_head=64, weight=P, n_heads=8)
    v.update(kw)
    return Heads(**v)


def test_the_wrappers_bytes_are_the_structures():
    from qwengine_b200 import api
    assert api._pack_heads(1, 2, 3, 4, 5, 6, 7, 8) == bytes(Heads(1, 2, 3, 4, 5, 6, 7, 8))
    assert api._pack_rules(*range(1, 11)) == bytes(Rules(*range(1, 11)))


@pytest.mark.parametrize("change,status", [
    (dict(D=0), ARG), (dict(D=1025), ARG), (dict(rot=66), ARG), (dict(rot=31), ARG), (dict(rot=-2), ARG), (dict(rows=0), ARG), (dict(in_kind=3), ARG),
    (dict(out_kind=-1), ARG), (dict(positions=None), ARG), (dict(inv_freq=None), ARG), (dict(positions=P + 2), ALIGN), (dict(inv_freq=P + 4), ALIGN),
    (dict(q=heads(src=None)), ARG), (dict(q=heads(dst=None)), ARG), (dict(q=heads(n_heads=0)), ARG), (dict(q=heads(src_head=-64)), ARG),
    (dict(q=heads(dst_head=63)), ARG), (dict(q=heads(dst_row=63)), ARG), (dict(q=heads(src=P + 2)), ALIGN), (dict(q=heads(weight=P + 1)), ALIGN),
    (dict(q=heads(dst_row=64)), ARG), (dict(q=heads(dst_row=511)), ARG), (dict(q=heads(dst_row=64, dst_head=191)), ARG),   # rows among heads
    (dict(k=heads(dst=None)), ARG), (dict(k=heads(dst_row=0)), ARG),
    (dict(q=heads(dst=P, dst_head=65)), ARG),                        # in place, but not element over element
    (dict(q=heads(dst=P), out_kind=2), ARG),
])
def test_heads(lib, change, status):
    a = dict(ctx=CTX, q=heads(), k=heads(), D=64, rot=32, positions=P, inv_freq=P, in_kind=0, out_kind=0, rows=3)
    a.update(change)
    rc = lib.q38b_qk_norm_rope(a["ctx"], C.byref(a["q"]), C.byref(a["k"]), a["D"], a["rot"], 0, 1e-6, 1.0, a["positions"], a["inv_freq"], a["in_kind"],
                               a["out_kind"], a["rows"], None)
    assert rc == status


def test_heads_null(lib):
    assert lib.q38b_qk_norm_rope(None, C.byref(heads()), None, 64, 0, 0, 1e-6, 1.0, None, None, 0, 0, 1, None) == ARG
    assert lib.q38b_qk_norm_rope(CTX, None, None, 64, 0, 0, 1e-6, 1.0, None, None, 0, 0, 1, None) == ARG


@pytest.mark.parametrize("change,rules,status", [
    (dict(x=None), {}, ARG), (dict(y=None), {}, ARG), (dict(n=0), {}, ARG), (dict(rows=0), {}, ARG), (dict(rows=65536), {}, ARG), (dict(x_ld=99), {}, ARG),
    (dict(y_ld=99), {}, ARG), (dict(off=-1), {}, ARG), (dict(off=0x7FFFFFFF), {}, ARG), (dict(n=(1 << 30) + 1, x_ld=1 << 31, y_ld=1 << 31), {}, UNSUPPORTED), (dict(y=P, y_ld=104), {}, ARG), (dict(x=P + 2), {}, ALIGN),
    ({}, dict(penalties=P), ARG), ({}, dict(history=P, history_begin=P), ARG), ({}, dict(penalties=P, history=P), ARG), ({}, dict(prompt_len=P), ARG),
    ({}, dict(bias_ids=P, bias_values=P), ARG), ({}, dict(bias_begin=P), ARG), ({}, dict(mask_of_row=P), ARG), ({}, dict(masks=P, mask_ld=3), ARG),
    (dict(off=29), dict(masks=P, mask_ld=4), ARG), ({}, dict(masks=ODD, mask_ld=4), ALIGN), ({}, dict(penalties=P, history=P, history_begin=P + 4), ALIGN),
    ({}, dict(bias_ids=P, bias_values=P, bias_begin=P + 4), ALIGN),
])
def test_logits(lib, change, rules, status):
    a = dict(x=P, x_ld=100, n=100, rows=2, off=0, y=P + 65536, y_ld=100)
    a.update(change)
    r = Rules(**rules)
    assert lib.q38b_adjust_logits(CTX, a["x"], a["x_ld"], a["n"], a["rows"], a["off"], C.byref(r), a["y"], a["y_ld"], None) == status
    assert lib.q38b_adjust_logits(CTX, P, 100, 100, 2, 0, None, P + 65536, 100, None) == ARG


def test_mx4(lib):
    q = lambda x=P, kind=0, ld=64, K=64, rows=3, c=P, cld=32, s=P: lib.q38b_quantize_mx4(CTX, x, kind, ld, K, rows, c, cld, s, None)   # noqa: E731
    assert [q(x=None), q(kind=3), q(ld=63), q(K=48, ld=64), q(K=0), q(rows=0), q(c=None), q(s=None), q(cld=16)] == [ARG] * 9
    assert [q(c=P + 8), q(cld=40), q(s=P + 4), q(x=P + 2), q(x=P + 1, kind=2)] == [ALIGN] * 5
    d = lambda K=64, rows=3, c=P, cld=32, s=P, out=P, kind=0, ld=64: lib.q38b_dequant_mx4(CTX, c, cld, s, K, rows, out, kind, ld, None)   # noqa: E731
    assert [d(K=33), d(rows=0), d(c=None), d(out=None), d(kind=9), d(ld=63)] == [ARG] * 6 and [d(s=P + 8), d(out=P + 2), d(out=P + 1, kind=1)] == [ALIGN] * 3
    t = lambda src=P, ld=2, K=64, rows=3, s=P: lib.q38b_mx4_tile_scales(CTX, src, ld, K, rows, s, None)   # noqa: E731
    assert [t(src=None), t(ld=1), t(K=40), t(rows=0), t(s=None)] == [ARG] * 5 and t(s=P + 1) == ALIGN


@pytest.mark.parametrize("change,status", [
    (dict(W=None), ARG), (dict(Ws=None), ARG), (dict(X=None), ARG), (dict(Xs=None), ARG), (dict(Y=None), ARG), (dict(K=100), ARG), (dict(M=0), ARG), (dict(M=(1 << 30) + 1, ldy=1 << 31), ARG), (dict(B=0), ARG),
    (dict(kind=3), ARG), (dict(ldy=199), ARG), (dict(W_ld=16), ARG), (dict(X_ld=16), ARG), (dict(W=P + 8), ALIGN), (dict(X_ld=56), ALIGN), (dict(Xs=P + 8), ALIGN),
    (dict(Y=P + 2), ALIGN)])
def test_mx4_product(lib, change, status):
    a = dict(W=P, W_ld=48, Ws=P, K=96, M=200, X=P, X_ld=48, Xs=P, B=3, Y=P, kind=0, ldy=200)
    a.update(change)
    assert lib.q38b_gemm_mx4(CTX, a["W"], a["W_ld"], a["Ws"], a["K"], a["M"], a["X"], a["X_ld"], a["Xs"], a["B"], a["Y"], a["kind"], a["ldy"], 0, None) == status


def test_mx4_sizes_and_scratch(lib):
    assert lib.q38b_mx4_scale_bytes(32, 1) == 512 and lib.q38b_mx4_scale_bytes(5120, 129) == 2 * 40 * 512 and lib.q38b_mx4_scale_bytes(160, 128) == 2 * 512
    assert lib.q38b_mx4_scale_bytes(48, 1) == 0 and lib.q38b_mx4_scale_bytes(64, 0) == 0
    assert lib.q38b_mx4_scale_bytes(1 << 20, 1 << 20) == (1 << 13) * (1 << 13) * 512      # past 32 bits
    assert lib.q38b_gemm_mx4_scratch_bytes(96, 1) == 0 == lib.q38b_gemm_mx4_scratch_bytes(8192, 1)      # quantized by the product's kernel
    need = lib.q38b_gemm_mx4_scratch_bytes(96, 9)
    assert need >= 9 * 48 + 512 and lib.q38b_gemm_mx4_scratch_bytes(8224, 1) >= 4112 + 65 * 512
    x = lambda **kw: lib.q38b_gemm_mx4_x(CTX, P, 48, P, 96, 200, *[{**dict(x=P, kind=0, ld=96, B=9, Y=P, yk=0, ldy=200, acc=0, s=P, n=need), **kw}[k]   # noqa: E731
                                                                  for k in ("x", "kind", "ld", "B", "Y", "yk", "ldy", "acc", "s", "n")], None)
    assert x(n=need - 1) == NOMEM and x(s=P + 8) == ALIGN and x(s=None) == ARG and x(x=P + 2) == ALIGN and x(Y=P + 2) == ALIGN and x(B=1, s=P + 4, n=0) == ALIGN
    assert [x(x=None), x(kind=5), x(ld=95), x(B=0), x(Y=None), x(yk=4), x(ldy=100)] == [ARG] * 7
