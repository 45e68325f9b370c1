"""The MLP with an 8-bit checkpoint where one of its parameters is not finite: that belongs to a hidden unit or to an output, and the others
keep theirs."""
import pytest
import torch

import rows8_reference as ref

pytestmark = pytest.mark.gpu


def _parameters(k, o, size, seed):
    torch.manual_seed(seed)
    module = torch.nn.Sequential(torch.nn.Linear(k, 128), torch.nn.ReLU(), torch.nn.Linear(128, o, bias=False)).cuda()
    return module, [p.detach().clone() * size for p in module.parameters()]


@pytest.mark.parametrize("size", [2.0**-18, 1.0, 2.0**20])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("where", ["w1", "b1", "w2"])
def test_a_parameter_that_is_not_finite(where, bad, size):
    """The share of its hidden unit in y is zero (the ReLU is fmaxf(NaN, 0)); its output and its unit's gradients are not finite.  What is
    held in units of the largest finite parameter keeps 5e-6 of the largest sum of magnitudes, as with finite ones."""
    from npa_b200.mlp import apply_mlp
    if where == "b1" and bad > 0:
        pytest.skip("an infinite bias makes its unit infinite, and every output with it")
    module, (w1, b1, w2) = _parameters(66, 18, size, 3)
    b1[9] = 2.0**24  # next to it the others are small: where it did not count, its unit of the hidden layer overflowed
    g = torch.Generator(device="cuda").manual_seed(1)
    z = ref.clear_of_the_corner(torch.randn(600, 66, device="cuda", generator=g), w1, b1)[:300]
    up = torch.randn(300, 18, device="cuda", generator=g)
    broken = [w1.clone(), b1.clone(), w2.clone()]
    broken[{"w1": 0, "b1": 1, "w2": 2}[where]][{"w1": (7, 5), "b1": (7,), "w2": (4, 7)}[where]] = bad
    if where != "w2":  # the unit as the ReLU leaves it
        w1[7], b1[7] = 0, 0
    with torch.no_grad():
        for p, v in zip(module.parameters(), broken):
            p.copy_(v)
    zr = z.clone().requires_grad_(True)
    y = apply_mlp(module, zr, checkpoint=True)
    got = dict(zip(("y", "dz", "dW1", "db1", "dW2"), [y.detach(), *torch.autograd.grad(y, [zr, *module.parameters()], up)]))
    truth = dict(zip(got, ref.mlp_with_checkpoint(z, w1, b1, w2, up)))
    alive = (z.double() @ w1.double().t() + b1.double() > 0).double()
    held, az, a1, ab, a2, au = (t.double().abs().to(z.device) for t in (ref.kept(z), z, w1, b1, w2, up))
    h, dh = (az @ a1.t() + ab) * alive, (au @ a2) * alive
    sizes = dict(zip(got, (h @ a2.t(), dh @ a1, dh.t() @ held, dh.sum(0), au.t() @ h)))
    units, outputs = torch.arange(128, device="cuda") != 7, torch.arange(18, device="cuda") != (4 if where == "w2" else -1)
    columns = torch.arange(66, device="cuda") != (5 if where == "w1" else -1)
    rows = alive[:, 7] == 0 if where == "w2" else torch.ones(300, dtype=torch.bool, device="cuda")
    assert 50 < rows.sum()
    good = {"y": lambda t: t[:, outputs], "dz": lambda t: t[rows][:, columns], "dW1": lambda t: t[units], "db1": lambda t: t[units], "dW2": lambda t: t[:, units]}
    for name, part in good.items():
        a, t, m = part(got[name]).double(), part(truth[name]), part(sizes[name])
        assert ((a - t).abs() <= 5e-6 * float(m.max())).all(), name
    if where == "w2":
        assert not torch.isfinite(got["y"][~rows][:, 4]).any() and not torch.isfinite(got["db1"][7]) and not torch.isfinite(got["dz"][~rows]).any()
