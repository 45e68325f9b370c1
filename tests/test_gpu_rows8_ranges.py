"""The MLP with an 8-bit checkpoint where channels differ in size: inputs, hidden units, outputs and their gradients up to 2^40 apart.
Every element of every output is held to the sum of the magnitudes behind it, as 32-bit sums of products would hold it."""
import ctypes

import pytest
import torch

import rows8_reference as ref

pytestmark = pytest.mark.gpu
NAMES = ["y", "dz", "dW1", "db1", "dW2"]

# A number held as two of float16 is off by 2^-22 of itself, and the product of two tails is left out: 3 * 2^-22 a product, in each of two
# layers.  A sum is cut off at 2^-24 of what it has come to: 33 times in z W1^T (11 steps of 16 columns, three products each), 24 times
# in a sum over 128 hidden units or rows, 14 times over a CTA's tiles, 26 times over the CTAs, and in 32 bits around them: below 100.
BAR = 6 * 2.0**-22 + 100 * 2.0**-24


@pytest.fixture(autouse=True)
def no_wait_gave_up():
    yield
    from npa_b200 import _native as n
    status = ctypes.c_uint32(0)
    n.check(n.lib.npa_linear_tcgen05_status(ctypes.byref(status), 1))
    assert status.value == 0


def _powers(n, how, seed):
    """n powers of two: half of them 2^-12, or all between 2^-20 and 2^20 in any order, or in rising order."""
    if how == "half":
        e = torch.where(torch.arange(n) % 2 == 1, -12.0, 0.0)
    elif how == "rising":
        e = torch.linspace(-20, 20, n).round()
    else:
        e = torch.linspace(-20, 20, n).round()[torch.randperm(n, generator=torch.Generator().manual_seed(seed))]
    return torch.exp2(e).cuda()


def _rand(*shape, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g) * torch.exp(0.5 * torch.randn(*shape[:-1], 1, device="cuda", generator=g))


def _module(w1, b1, w2):
    module = torch.nn.Sequential(torch.nn.Linear(w1.shape[1], 128), torch.nn.ReLU(), torch.nn.Linear(128, w2.shape[0], bias=False)).cuda()
    with torch.no_grad():
        for p, v in zip(module.parameters(), (w1, b1, w2)):
            p.copy_(v)
    return module


def _weights(k, o, seed):
    torch.manual_seed(seed)
    module = torch.nn.Sequential(torch.nn.Linear(k, 128), torch.nn.ReLU(), torch.nn.Linear(128, o, bias=False)).cuda()
    return [p.detach().clone() for p in module.parameters()]


def _run(module, z, up):
    from npa_b200.mlp import apply_mlp
    z = z.detach().clone().requires_grad_(True)
    y = apply_mlp(module, z, checkpoint=True)
    return [y.detach(), *torch.autograd.grad(y, [z, *module.parameters()], up)]


def _sizes(z, w1, b1, w2, up):
    """Sums of the magnitudes behind (y, dz, dW1, db1, dW2), element by element."""
    alive = (z.double() @ w1.double().t() + b1.double() > 0).double()
    held, z, w1, b1, w2, up = (t.detach().double().abs().to(z.device) for t in (ref.kept(z), z, w1, b1, w2, up))
    h, again, dh = (z @ w1.t() + b1) * alive, (held @ w1.t() + b1) * alive, (up @ w2) * alive
    return h @ w2.t(), dh @ w1, dh.t() @ held, dh.sum(0), up.t() @ again


def _check(w1, b1, w2, z, up, least, bar=BAR):
    from npa_b200.mlp import apply_mlp
    z = ref.clear_of_the_corner(z, w1, b1)
    up = up[: len(z)]
    assert len(z) >= least
    truth = ref.mlp_with_checkpoint(z, w1, b1, w2, up)
    theirs = ref.mlp_with_checkpoint(z, w1, b1, w2, up, torch.float32)
    size = _sizes(z, w1, b1, w2, up)
    worst = {}
    module = _module(w1, b1, w2)
    got = _run(module, z, up)
    alone = torch.autograd.grad(apply_mlp(module, z, checkpoint=True), list(module.parameters()), up)
    assert all(torch.equal(a, b) for a, b in zip(alone, got[2:]))  # where z asks for no gradient
    for name, a, b, t, m in zip(NAMES, got, theirs, truth, size):
        floor = m.clamp_min(2.0**-120)
        worst[name] = (float(((a.double() - t).abs() / floor).max()), float(((b.double() - t).abs() / floor).max()))
    print({n: f"{v[0]:.1e} (torch fp32 {v[1]:.1e})" for n, v in worst.items()})
    assert all(v[0] <= bar for v in worst.values()), worst


CASES = {
    "alike": {},
    "inputs": {"z": 1},
    "inputs against weights": {"z": 1, "w1_in": -1},
    "weights of inputs": {"w1_in": 1},
    "hidden units": {"w1_out": 1, "b1": 1},
    "hidden units, not their biases": {"w1_out": 1},
    "hidden units against outputs": {"w1_out": 1, "b1": 1, "w2_in": -1},
    "weights of hidden units": {"w2_in": 1},
    "outputs": {"w2_out": 1},
    "outputs against their gradients": {"w2_out": 1, "up": -1},
    "gradients": {"up": 1},
    "everything": {"z": 1, "w1_in": -1, "w1_out": 1, "b1": 1, "w2_in": -1, "w2_out": 1, "up": -1},
}


@pytest.mark.parametrize("rows,k,o", [(300, 66, 18), (1500, 163, 35)])
@pytest.mark.parametrize("how", ["half", "mixed", "rising"])
@pytest.mark.parametrize("case", list(CASES))
def test_channels_of_different_size(case, how, rows, k, o):
    w1, b1, w2 = _weights(k, o, 1)
    z, up = _rand(2 * rows, k, seed=2), _rand(2 * rows, o, seed=3)
    sign = CASES[case]
    inputs, hidden, outputs = _powers(k, how, 4), _powers(128, how, 5), _powers(o, how, 6)
    z = z * inputs ** sign.get("z", 0)
    w1 = w1 * inputs ** sign.get("w1_in", 0) * hidden[:, None] ** sign.get("w1_out", 0)
    b1 = b1 * hidden ** sign.get("b1", 0)
    w2 = w2 * hidden ** sign.get("w2_in", 0) * outputs[:, None] ** sign.get("w2_out", 0)
    up = up * outputs ** sign.get("up", 0)
    _check(w1, b1, w2, z, up, rows)


@pytest.mark.parametrize("rows,k,o", [(1, 66, 18), (129, 5, 3), (4103, 163, 35), (20001, 176, 48), (65536, 96, 33)])
def test_elements_to_their_own_size(rows, k, o):
    w1, b1, w2 = _weights(k, o, rows)
    _check(w1, b1, w2, _rand(rows + rows // 4 + 8, k, seed=2), _rand(rows + rows // 4 + 8, o, seed=3), rows)


@pytest.mark.parametrize("rows,k,o", [(300, 66, 18), (1500, 163, 35), (40000, 100, 7)])
def test_far_groups_of_inputs(rows, k, o):
    """Groups of 32 columns up to 2^90 apart: each has exponents of its own, and its columns of dW1 nothing to do with the others."""
    w1, b1, w2 = _weights(k, o, 7)
    far = torch.exp2(torch.linspace(-45, 45, (k + 31) // 32)).cuda().repeat_interleave(32)[:k]
    _check(w1, b1, w2, _rand(2 * rows, k, seed=2) * far, _rand(2 * rows, o, seed=3), rows)
    _check(w1 / far, b1, w2, _rand(2 * rows, k, seed=2) * far, _rand(2 * rows, o, seed=3), rows)


@pytest.mark.parametrize("rows,k,o", [(300, 66, 18), (30000, 163, 35)])
def test_channels_without_a_value(rows, k, o):
    """Columns of zeros in every operand have no size of their own."""
    w1, b1, w2 = _weights(k, o, 8)
    z, up = _rand(2 * rows, k, seed=2), _rand(2 * rows, o, seed=3)
    z[:, ::3] = 0
    z[:, 32:64] = 0
    up[:, 1::2] = 0
    up[:, 0] *= 2.0**-30
    w1[:, 2::5] *= 2.0**-25
    w1[5] = 0
    w1[:, 7] = 0
    w2[:, 9] = 0
    w2[2] = 0
    b1[5] = 0
    _check(w1, b1, w2, z, up, rows)


# exponents of z, W1, W2 and the gradients of y; the outputs stay numbers
@pytest.mark.parametrize("ez,e1,e2,eu", [(-90, 130, -5, -5), (100, -110, 0, 0), (-20, 0, 130, -100), (0, 0, -100, 110), (-60, -50, 60, 40), (60, 40, -80, -40),
                                         (-40, 130, -40, 0), (0, 0, 0, -90), (0, 0, 0, 110)])
def test_operands_of_any_size(ez, e1, e2, eu):
    """Largest weights next to the largest number, and small ones against large inputs: units cover the range of 32 bits."""
    w1, b1, w2 = _weights(66, 18, 9)
    z, up = _rand(600, 66, seed=2), _rand(600, 18, seed=3)
    times = lambda t, e: (t.double() * 2.0**e).float()  # (2^130 itself is no number of 32 bits)
    _check(times(w1, e1), times(b1, e1 + ez), times(w2, e2), times(z, ez), times(up, eu), 300)


def test_what_is_not_finite_among_channels_apart():
    """A NaN in one far group of z, an infinity in one column of the gradients: the other groups, columns and rows keep their own accuracy."""
    w1, b1, w2 = _weights(100, 18, 7)
    far = torch.exp2(torch.linspace(-30, 30, 4)).cuda().repeat_interleave(32)[:100]
    w1 = w1 / far
    z = ref.clear_of_the_corner(_rand(600, 100, seed=2) * far, w1, b1)[:300]
    up = _rand(300, 18, seed=3) * _powers(18, "mixed", 6)
    rows = torch.arange(300, device="cuda") != 5
    truth, size = ref.mlp_with_checkpoint(z[rows], w1, b1, w2, up[rows]), _sizes(z[rows], w1, b1, w2, up[rows])
    module = _module(w1, b1, w2)
    bad = z.clone()
    bad[5, 40] = float("nan")  # every hidden unit of the row is NaN, and dead (fmaxf)
    y, dz, dw1, db1, dw2 = _run(module, bad, up)
    columns = torch.arange(100, device="cuda") // 32 != 1
    for name, a, t, m in (("y", y[rows], truth[0], size[0]), ("dz", dz[rows], truth[1], size[1]), ("dW1", dw1[:, columns], truth[2][:, columns], size[2][:, columns]),
                          ("db1", db1, truth[3], size[3]), ("dW2", dw2, truth[4], size[4])):
        assert ((a.double() - t).abs() <= BAR * m).all(), name
    assert torch.isnan(dw1[:, ~columns]).all()
    wild = up.clone()
    wild[5, 2] = float("inf")
    y, dz, dw1, db1, dw2 = _run(module, z, wild)
    alive = (z.double() @ w1.double().t() + b1.double() > 0)[5]
    truth, size = ref.mlp_with_checkpoint(z, w1, b1, w2, up), _sizes(z, w1, b1, w2, up)
    others = torch.arange(18, device="cuda") != 2
    for name, a, t, m in (("dz", dz[rows], truth[1][rows], size[1][rows]), ("dW1", dw1[~alive], truth[2][~alive], size[2][~alive]), ("db1", db1[~alive], truth[3][~alive], size[3][~alive]),
                          ("dW2", dw2[others], truth[4][others], size[4][others])):
        assert ((a.double() - t).abs() <= BAR * m).all(), name
    assert not torch.isfinite(dw2[2]).all() and not torch.isfinite(db1[alive]).any()
