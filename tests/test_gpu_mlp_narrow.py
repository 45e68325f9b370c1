"""The adaptation MLP with few inputs or outputs on more rows than two tiles for each SM: every accumulator is used again."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("k,o", [(16, 16), (1, 1), (9, 48), (17, 3)])
def test_narrow_products_on_many_rows(k, o):
    from npa_b200 import _native as n
    from npa_b200.mlp import apply_mlp
    torch.manual_seed(0)
    rows = 3 * 148 * 128 + 5
    module = torch.nn.Sequential(torch.nn.Linear(k, 128), torch.nn.ReLU(), torch.nn.Linear(128, o, bias=False)).cuda()
    w1, b1, w2 = (p.detach().double() for p in module.parameters())
    z = torch.randn(rows, k, device="cuda")
    near = (z.double() @ w1.t() + b1).abs() < 1e-5 * (z.double().abs() @ w1.abs().t() + b1.abs())
    z = z[~near.any(1)]
    up = torch.randn(len(z), o, device="cuda")
    assert len(z) > 2 * 148 * 128
    zr = z.clone().requires_grad_(True)
    y = apply_mlp(module, zr)
    gz, = torch.autograd.grad(y, zr, up)
    status = ctypes.c_uint32(0)
    n.check(n.lib.npa_linear_tcgen05_status(ctypes.byref(status), 1))
    assert status.value == 0
    before = z.double() @ w1.t() + b1
    alive = (before > 0).double()
    # 2^-21 of each product's magnitude in each of the two layers, and 2^-24 of the sum's in each of up to 48 additions: 4e-6
    size_h, size_dh = z.double().abs() @ w1.abs().t() + b1.abs(), up.double().abs() @ w2.abs()
    assert ((y.double() - (before * alive) @ w2.t()).abs() <= 4e-6 * (size_h @ w2.abs().t())).all()
    assert ((gz.double() - ((up.double() @ w2) * alive) @ w1).abs() <= 4e-6 * (size_dh @ w1.abs())).all()
