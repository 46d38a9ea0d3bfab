"""How the 4-bit product and the quantizer in front of it are launched: the product may start while the quantizer still runs (programmatic dependent
launch), unless the context's switch for that is off."""
import ctypes as C

import pytest
import torch

import qwengine_b200 as q

pytestmark = pytest.mark.gpu


class EdgeData(C.Structure):
    """CUgraphEdgeData; type 1: programmatic"""
    _fields_ = [("from_port", C.c_ubyte), ("to_port", C.c_ubyte), ("type", C.c_ubyte), ("reserved", C.c_ubyte * 5)]


def edges(call):
    """The kinds of the edges between what a call launches."""
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    raw, n = C.c_void_p(graph.raw_cuda_graph()), C.c_size_t(16)
    a, b, data = (C.c_void_p * 16)(), (C.c_void_p * 16)(), (EdgeData * 16)()
    assert C.CDLL("libcuda.so.1").cuGraphGetEdges_v2(raw, a, b, data, C.byref(n)) == 0
    return [data[i].type for i in range(n.value)]


@pytest.mark.parametrize("B,M,K,launches", [(7, 300, 1024, 2), (300, 512, 1024, 2), (1, 256, 8224, 1)])     # one CTA a tile, pairs, one token: its kernel quantizes it
def test_the_switch_for_programmatic_launches(B, M, K, launches):
    ctx = q.Context(0)
    try:
        g = torch.Generator().manual_seed(B)
        W = ctx.quantize_mx4(torch.randn((M, K), generator=g).cuda())
        x, y = torch.randn((B, K), generator=g).cuda(), torch.empty((B, M), device="cuda")
        assert edges(lambda: ctx.gemm_mx4(W, x, out=y)) == [1] * (launches - 1)
        want = y.clone()
        ctx.set_pdl(False)
        assert edges(lambda: ctx.gemm_mx4(W, x, out=y)) == [0] * (launches - 1)
        assert torch.equal(y, want)
        ctx.set_pdl(True)
        assert edges(lambda: ctx.gemm_mx4(W, x, out=y)) == [1] * (launches - 1)
        ctx.check()
    finally:
        ctx.close()
