"""Training steps whose MLP keeps its input in 8 bits, on particles with no hidden unit near the ReLU's corner (there the derivative has two
values, and one unit that falls the other way hides every smaller fault): gradients as from the formula in 32-bit torch; what a rollout holds."""
import pytest
import torch

import rows8_reference as ref

pytestmark = pytest.mark.gpu


class _Model(torch.nn.Module):
    def __init__(self, dim, C):
        super().__init__()
        self.model = torch.nn.Sequential(torch.nn.Linear(2 * C + C * dim + dim, 128), torch.nn.ReLU(), torch.nn.Linear(128, dim + C, bias=False))
        self.eps0, self.alpha, self.spatial_dims = 0.1, 0.5, dim


class _Formula(torch.autograd.Function):
    nearest = []  # distances of hidden units from the corner, in shares of their sums of magnitudes

    @staticmethod
    def forward(ctx, z, w1, b1, w2):
        before = z @ w1.t() + b1
        _Formula.nearest.append(float((before.abs() / (z.abs() @ w1.abs().t() + b1.abs())).min()))
        ctx.save_for_backward(ref.kept(z).to(z), before > 0, w1, b1, w2)
        return before.clamp_min(0) @ w2.t()

    @staticmethod
    def backward(ctx, up):
        z, alive, w1, b1, w2 = ctx.saved_tensors
        z, alive, flat = z.flatten(0, 1), alive.flatten(0, 1), up.flatten(0, 1)
        dh = (flat @ w2) * alive
        h = (z @ w1.t() + b1) * alive
        return (dh @ w1).view(*up.shape[:2], -1), dh.t() @ z, dh.sum(0), flat.t() @ h


def _grid(dim, N, B):
    from npa_b200 import sphops as sph
    return sph.HashGrid(dim=dim, boundary="clamped", mode="grid", grid_size=(8,) * dim, eps=0.15, num_particles=N, batch_size=B)


def _inputs(dim, C, N, B, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.rand(B, N, dim, device="cuda", generator=g) - 0.5
    x = x if dim == 2 else torch.cat([x, torch.zeros_like(x[..., :1])], -1).contiguous()
    return x, torch.randn(B, N, C, device="cuda", generator=g)


# Of 300 x 2 particles with 128 hidden units, half a unit lies within 5e-7 of its corner; the two ways of z W1^T differ by 2e-7 at most.
FAR_FROM_THE_CORNER = 5e-7


@pytest.mark.parametrize("steps", [1, 2])
@pytest.mark.parametrize("dim,C", [(2, 16), (3, 12)])
def test_gradients_away_from_the_corner(dim, C, steps, monkeypatch):
    """A term of a gradient is off by 8e-6 of its magnitude at most (the bar of the MLP alone), and a sum of 600 of random sign is 1/24 of
    their magnitudes: 2e-4 in norm.  From the second step on z itself differs by 1e-7, which moves a few codes of 40,000 by one: 1/64 of one
    of 600 terms in one of 66 columns, 8e-5 each in norm; room for ten."""
    from npa_b200 import stepping
    N, B = 300, 2
    torch.manual_seed(1)
    model, grid = _Model(dim, C).cuda(), _grid(dim, N, B)

    def rollout(x, s, formula):
        torch.manual_seed(2)
        sr = s.clone().requires_grad_(True)
        xx, ss = x, sr
        _Formula.nearest.clear()
        with monkeypatch.context() as m:
            if formula:
                m.setattr(stepping, "apply_mlp", lambda module, z, checkpoint: _Formula.apply(z, module[0].weight, module[0].bias, module[2].weight))
            for _ in range(steps):
                xx, ss, _ = stepping.step_euler(model, xx, ss, grid, checkpoint=True)
            grads = torch.autograd.grad(ss.square().mean() + xx.square().mean(), [sr, *model.parameters()])
        return [xx.detach(), ss.detach(), *grads]

    for seed in range(60):  # inputs that the formula finds clear
        x, s = _inputs(dim, C, N, B, seed)
        want = rollout(x, s, True)
        if min(_Formula.nearest) > FAR_FROM_THE_CORNER:
            break
    else:
        raise AssertionError("no such inputs")
    got = rollout(x, s, False)
    bar = 2e-4 if steps == 1 else 1e-3
    for k, (a, b) in enumerate(zip(got, want)):
        assert float((a - b).norm()) <= (1e-5 if k < 2 else bar) * float(b.norm()), k


@pytest.mark.parametrize("dim,C", [(2, 16), (3, 32)])
def test_what_a_rollout_holds(dim, C):
    """The MLP holds its checkpoint instead of its input and hidden layer; what the other operators of a step hold is theirs with or without."""
    from npa_b200 import stepping
    N, B, steps = 4096, 4, 6
    torch.manual_seed(1)
    model, grid = _Model(dim, C).cuda(), _grid(dim, N, B)
    x, s = _inputs(dim, C, N, B, 0)

    def held(**how):
        stepping.step_euler(model, x, s.clone().requires_grad_(True), grid, **how)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        xx, ss = x, s.clone().requires_grad_(True)
        for _ in range(steps):
            xx, ss, _ = stepping.step_euler(model, xx, ss, grid, **how)
        torch.cuda.synchronize()
        return (torch.cuda.memory_allocated() - before) / steps / (N * B)

    kept, plain = held(checkpoint=True), held()
    k = 2 * C + C * dim + dim
    saved = 4 * (k + 128) - (k + k / 32 + 16)
    print(f"bytes a particle and step: {plain:.0f}, with checkpoint {kept:.0f}; the MLP's own difference {saved:.0f}")
    assert kept <= plain - 0.6 * saved  # (an image of the weights a step, rows rounded up to 16, and the MLP's output, which the one-node step does not keep)
