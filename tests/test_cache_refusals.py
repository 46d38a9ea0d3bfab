"""What the paged cache, the attention over it and the 8-bit products refuse: checked before a device is touched, so without one."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def lib():
    from qwengine_b200 import build, load_library
    build.build()
    return load_library()


CTX = C.create_string_buffer(8192)      # never looked into: every call below is refused first
P = 0x10000                             # an address that is only compared and checked for its alignment
ARG, UNSUPPORTED, ALIGN, NOMEM = -1, -2, -3, -6


class Paged(C.Structure):
    """q38b_paged_kv"""
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p)] + [(n, C.c_longlong) for n in ("k_page", "k_slot", "k_head", "v_page", "v_slot", "v_head")] + \
               [(n, C.c_int) for n in ("kind", "n_pages", "page_size", "n_heads", "D", "n_seqs")] + [("table", C.c_void_p), ("table_ld", C.c_longlong), ("table_n", C.c_int)] + \
               [("lengths", C.c_void_p), ("begin", C.c_void_p)]


def paged(**kw):
    v = dict(k=P, v=P, k_page=2048, k_slot=128, k_head=64, v_page=2048, v_slot=128, v_head=64, kind=2, n_pages=10, page_size=16, n_heads=2, D=64, n_seqs=3, table=P, table_ld=8,
             table_n=8, lengths=P, begin=P)
    v.update(kw)
    return Paged(**v)


def test_the_wrappers_bytes_are_the_structure():
    from qwengine_b200 import api
    assert api._pack_paged(*range(1, 20)) == bytes(Paged(*range(1, 20)))


BAD_CACHES = [
    (dict(k=None), ARG), (dict(v=None), ARG), (dict(table=None), ARG), (dict(lengths=None), ARG), (dict(begin=None), ARG), (dict(kind=0), ARG), (dict(kind=3), ARG),
    (dict(n_pages=0), ARG), (dict(page_size=4), ARG), (dict(page_size=24), ARG), (dict(page_size=0), ARG), (dict(n_pages=1 << 27), ARG), (dict(n_heads=0), ARG), (dict(D=0), ARG),
    (dict(D=60), ARG), (dict(D=264, k_head=264, v_head=264), ARG), (dict(n_seqs=0), ARG), (dict(n_seqs=65536), ARG), (dict(table_n=0), ARG), (dict(table_ld=7), ARG),
    (dict(table_n=1 << 27, table_ld=1 << 27), ARG), (dict(k_head=56), ARG), (dict(v_slot=0), ARG), (dict(k_page=-2048), ARG), (dict(v_page=2052), ALIGN), (dict(k_head=68), ALIGN),
    (dict(k=P + 8), ALIGN), (dict(v=P + 2), ALIGN), (dict(table=P + 2), ALIGN), (dict(lengths=P + 1), ALIGN), (dict(begin=P + 2), ALIGN)]


@pytest.mark.parametrize("change,status", BAD_CACHES)
def test_caches(lib, change, status):
    assert lib.q38b_cache_append(CTX, C.byref(paged(**change)), P, P, 2, 128, 64, 128, 64, 5, None) == status
    assert lib.q38b_attention(CTX, C.byref(paged(**change)), P + 4096, 2, 256, 64, 4, 0.125, P, 2, 256, 64, None, 5, P, 1 << 40, None) == status


@pytest.mark.parametrize("change,status", [
    (dict(k=None), ARG), (dict(v=None), ARG), (dict(cache=None), ARG), (dict(kind=7), ARG), (dict(kind=1), UNSUPPORTED), (dict(rows=0), ARG), (dict(row=-1), ARG), (dict(head=-64), ARG),
    (dict(k=P + 1), ALIGN), (dict(kind=0, v=P + 2), ALIGN)])
def test_append(lib, change, status):
    a = dict(cache=paged(), k=P, v=P, kind=2, row=128, head=64, rows=5)
    a.update(change)
    rc = lib.q38b_cache_append(CTX, C.byref(a["cache"]) if a["cache"] else None, a["k"], a["v"], a["kind"], a["row"], a["head"], 128, 64, a["rows"], None)
    assert rc == status
    assert lib.q38b_cache_append(None, C.byref(paged()), P, P, 2, 128, 64, 128, 64, 5, None) == ARG


@pytest.mark.parametrize("change,status", [
    (dict(q=None), ARG), (dict(out=None), ARG), (dict(q=P), ARG), (dict(cache=None), ARG), (dict(work=None), ARG), (dict(rows=0), ARG), (dict(n_heads=0), ARG), (dict(n_heads=3), ARG), (dict(q_kind=4), ARG),
    (dict(out_kind=-1), ARG), (dict(q_kind=1), UNSUPPORTED), (dict(scale=0.0), ARG), (dict(scale=-1.0), ARG), (dict(scale=float("nan")), ARG), (dict(scale=float("inf")), ARG),
    (dict(q_row=-1), ARG), (dict(q_head=-1), ARG), (dict(out_row=63), ARG), (dict(out_head=32), ARG), (dict(out_row=255), ARG), (dict(out_row=64), ARG), (dict(out_row=64, out_head=319), ARG), (dict(q=P + 1), ALIGN), (dict(out=P + 1), ALIGN), (dict(out_kind=0, out=P + 2), ALIGN),
    (dict(lse=P + 2), ALIGN), (dict(work=P + 8), ALIGN), (dict(work_bytes=15), NOMEM)])
def test_attention(lib, change, status):
    a = dict(cache=paged(), q=P + 4096, q_kind=2, q_row=256, q_head=64, n_heads=4, scale=0.125, out=P, out_kind=2, out_row=256, out_head=64, lse=None, rows=5, work=P, work_bytes=1 << 40)
    a.update(change)
    a["cache"] = C.byref(a["cache"]) if a["cache"] else None
    assert lib.q38b_attention(CTX, *a.values(), None) == status


def test_attention_of_more_work_than_is_counted(lib):
    call = lambda cache, rows, nq=4: lib.q38b_attention(CTX, C.byref(cache), P + 4096, 2, 256, 64, nq, 0.125, P, 2, 64 * nq, 64, None, rows, P, 15, None)   # noqa: E731
    assert call(paged(), (1 << 30) // 4) == UNSUPPORTED and call(paged(), (1 << 30) // 4 - 1) == NOMEM
    wide = dict(table_n=1 << 20, table_ld=1 << 20, page_size=1024, n_pages=1 << 20, k_page=1 << 17, v_page=1 << 17)      # 2^30 tokens: 2^23 tiles of keys
    assert call(paged(**wide), 64 * 32) == NOMEM and call(paged(**wide), 64 * 128) == UNSUPPORTED


def test_quantize_i8(lib):
    q = lambda x=P, kind=0, ld=64, K=64, rows=3, c=P, cld=64, s=P: lib.q38b_quantize_i8(CTX, x, kind, ld, K, rows, c, cld, s, None)   # noqa: E731
    assert [q(x=None), q(kind=3), q(ld=63), q(K=0), q(K=131072, ld=1 << 20, cld=1 << 20), q(rows=0), q(rows=(1 << 30) + 1), q(c=None), q(s=None), q(cld=48)] == [ARG] * 10
    assert [q(c=P + 8), q(cld=72), q(s=P + 2), q(x=P + 2), q(x=P + 1, kind=2)] == [ALIGN] * 5


@pytest.mark.parametrize("change,status", [
    (dict(W=None), ARG), (dict(Ws=None), ARG), (dict(X=None), ARG), (dict(Xs=None), ARG), (dict(Y=None), ARG), (dict(K=0), ARG), (dict(K=131072, W_ld=1 << 20, X_ld=1 << 20), ARG), (dict(M=0), ARG),
    (dict(M=(1 << 30) + 1, ldy=1 << 31), ARG), (dict(B=0), ARG), (dict(kind=3), ARG), (dict(ldy=199), ARG), (dict(W_ld=96), ARG), (dict(X_ld=96), ARG), (dict(W=P + 8), ALIGN),
    (dict(X_ld=120), ALIGN), (dict(X=P + 4), ALIGN), (dict(Xs=P + 2), ALIGN), (dict(Y=P + 2), ALIGN)])
def test_i8_product(lib, change, status):
    a = dict(W=P, W_ld=112, Ws=P, K=100, M=200, X=P, X_ld=112, Xs=P, B=3, Y=P, kind=0, ldy=200)
    a.update(change)
    assert lib.q38b_gemm_i8(CTX, a["W"], a["W_ld"], a["Ws"], a["K"], a["M"], a["X"], a["X_ld"], a["Xs"], a["B"], a["Y"], a["kind"], a["ldy"], 0, None) == status


def test_i8_scratch(lib):
    need = lib.q38b_gemm_i8_scratch_bytes(100, 9)
    assert need >= 9 * 112 + 36 and lib.q38b_gemm_i8_scratch_bytes(0, 1) == 0 == lib.q38b_gemm_i8_scratch_bytes(131072, 1) == lib.q38b_gemm_i8_scratch_bytes(64, 0)
    assert lib.q38b_gemm_i8_scratch_bytes(131071, 1 << 20) >= 131071 << 20      # past 32 bits
    x = lambda **kw: lib.q38b_gemm_i8_x(CTX, P, 112, P, 100, 200, *[{**dict(x=P, kind=0, ld=100, B=9, Y=P, yk=0, ldy=200, acc=0, s=P, n=need), **kw}[k]   # noqa: E731
                                                                   for k in ("x", "kind", "ld", "B", "Y", "yk", "ldy", "acc", "s", "n")], None)
    assert x(n=need - 1) == NOMEM and x(s=P + 8) == ALIGN and x(s=None) == ARG and x(x=P + 2) == ALIGN and x(Y=P + 2) == ALIGN
    assert [x(x=None), x(kind=5), x(ld=99), x(B=0), x(Y=None), x(yk=4), x(ldy=100)] == [ARG] * 7
