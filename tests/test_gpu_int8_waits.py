"""The bounded waits of the 8-bit kernels report nothing after products of every tile width, one tile a CTA and many, and after the integer MLP."""
import ctypes

import pytest
import torch

import rows8_reference as ref

pytestmark = pytest.mark.gpu


def _status():
    from npa_b200 import _native as n
    torch.cuda.synchronize()
    status = ctypes.c_uint32(0)
    n.check(n.lib.npa_linear_tcgen05_status(ctypes.byref(status), 1))
    return status.value


@pytest.mark.parametrize("M,K,N", [(17, 100, 8), (1000, 300, 200), (20000, 130, 40), (40000, 64, 300), (3000, 129, 5000)])
def test_products(M, K, N):
    from npa_b200.int8 import linear_int8, quantize_rows
    assert _status() == 0
    g = torch.Generator(device="cuda").manual_seed(M)
    x, w = torch.randn(M, K, device="cuda", generator=g), torch.randn(N, K, device="cuda", generator=g)
    codes, t = quantize_rows(w)
    b = torch.randn(N, device="cuda", generator=g)
    y = linear_int8(x, codes, t, bias=b)
    q, s = ref.quantized(x)
    assert torch.equal(y.cpu(), ref.linear(q, s, codes, t, b))
    unsigned, us = quantize_rows(x, unsigned=True)
    q, s = ref.quantized(x, True)
    assert torch.equal(linear_int8(unsigned, codes, t, x_scales=us).cpu(), ref.linear(q, s, codes, t))
    assert _status() == 0


@pytest.mark.parametrize("rows,k,n", [(1, 66, 18), (60001, 163, 35), (40000, 250, 64)])
def test_mlp(rows, k, n):
    from npa_b200.int8 import mlp_int8, quantize_rows
    assert _status() == 0
    g = torch.Generator(device="cuda").manual_seed(rows)
    z, w1, w2 = (torch.randn(*s, device="cuda", generator=g) for s in ((rows, k), (128, k), (n, 128)))
    mlp_int8(z, *quantize_rows(w1), torch.randn(128, device="cuda", generator=g), *quantize_rows(w2))
    assert _status() == 0
