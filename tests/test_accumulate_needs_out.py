"""Products that add to what is there refuse to be called without it: a fresh output holds whatever memory held."""
import pytest
import torch

import qwengine_b200 as q


def context():
    """Never comes as far as the library: every call below is refused first."""
    c = q.Context.__new__(q.Context)
    c.lib, c.h, c.device, c._index = None, None, torch.device("cpu"), -1
    return c


def refused(call):
    with pytest.raises(ValueError, match="accumulate"):
        call()


@pytest.mark.parametrize("x", [torch.zeros(3, 64), "quantized"])
def test_gemm_mx4(x):
    W = q.Mx4(torch.zeros(5, 32, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8))
    refused(lambda: context().gemm_mx4(W, W if isinstance(x, str) else x, accumulate=True))


def test_products_of_gguf_blocks():
    c, w = context(), torch.zeros(5, 144, dtype=torch.uint8)
    refused(lambda: c.gemv("Q4_K", w, torch.zeros(1, 292, dtype=torch.uint8), 256, accumulate=True))
    refused(lambda: c.gemv_act_q8("Q4_K", w, torch.zeros(1, 256, dtype=torch.int8), torch.zeros(1, 8), 256, accumulate=True))
    refused(lambda: c.gemv_f32("Q4_K", w, torch.zeros(1, 256), 256, accumulate=True))
    refused(lambda: c.gemm_prefill("Q4_K", w, torch.zeros(1, 256, dtype=torch.bfloat16), 256, accumulate=True))
