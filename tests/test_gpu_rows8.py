"""Activations in 8 bits (rows8) and the MLP that keeps its input so: values against the definition, gradients against 64 bits of
the formula, against differences, and inside training steps."""
import ctypes

import pytest
import torch
import torch.utils.checkpoint

import rows8_reference as ref

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(autouse=True)
def no_wait_gave_up():
    yield
    from npa_b200 import _native as n
    status = ctypes.c_uint32(0)
    n.check(n.lib.npa_linear_tcgen05_status(ctypes.byref(status), 1))
    assert status.value == 0


def _rand(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(*shape, device="cuda", generator=g) * torch.exp(torch.randn(*shape[:-1], 1, device="cuda", generator=g))
    return x.to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 17), (2, 3, 66), (5, 32), (33, 163), (7, 1025), (4, 4100), (70001, 5), (0, 8)])
def test_values(shape, dtype):
    from npa_b200.rows8 import compress_rows
    x = _rand(*shape, dtype=dtype)
    if x.numel():
        x.reshape(-1, shape[-1])[0] = 0
    rows = compress_rows(x)
    assert rows.codes.dtype == torch.int8 and rows.codes.shape == x.shape and rows.exponents.shape == (*shape[:-1], (shape[-1] + 31) // 32)
    want = ref.kept(x)
    value = rows.restore()
    assert value.dtype == dtype and torch.equal(value.cpu(), want.to(dtype))
    for out in TYPES:
        assert torch.equal(rows.restore(out).cpu(), want.to(out).clamp(-65504, 65504) if out == torch.float16 else want.to(out))
    if x.numel():
        step = torch.exp2(rows.exponents.cpu().double() - 133)
        worst = torch.repeat_interleave(step, 32, -1)[..., : shape[-1]] / 2
        assert ((want - x.cpu().double()).abs() <= worst).all()
        assert rows.nbytes <= x.numel() // shape[-1] * (shape[-1] + 15 + (shape[-1] + 31) // 32)


@pytest.mark.parametrize("cols", [1, 31, 33, 100])
def test_values_at_the_borders(cols):
    """Magnitudes next to the change of an exponent, ties, subnormals, the largest numbers, groups that are not finite."""
    from npa_b200.rows8 import compress_rows
    g = torch.Generator().manual_seed(cols)
    rows = []
    for top in (127.0, 127.4999, 127.5, 127.50001, 128.0, 64.0, 63.9999, 1.9921875, 1.9921874, 3.4e38, 3.3895e38, 1e-38, 1e-45, 2.0 ** -126, 2.0 ** -119, 0.0):
        v = (torch.randint(-127, 128, (cols,), generator=g).float() + 0.5) * (top / 127.5)
        v = v.clamp(-top, top)
        v[0] = top
        rows += [v, -v]
    for bad in (float("inf"), float("-inf"), float("nan")):
        v = torch.randn(cols, generator=g)
        v[-1] = bad
        rows.append(v)
    x = torch.stack(rows).cuda()
    want = ref.kept(x).float()
    got = compress_rows(x).restore().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))
    big = torch.tensor([[65504.0, -65504.0, 65400.0]], device="cuda", dtype=torch.float16)
    assert torch.isfinite(compress_rows(big).restore()).all()


def test_strides_and_refusals():
    from npa_b200.mlp import apply_mlp
    from npa_b200.rows8 import Rows8, compress_rows
    x = _rand(40, 200)
    for view in (x[:, 3:103], x.t(), x[::2], x[:1].expand(7, 200), x.view(4, 10, 200).transpose(0, 1), x[5]):
        assert torch.equal(compress_rows(view).restore().cpu(), ref.kept(view).float())
    kept = compress_rows(x)
    loose = torch.full((40, 211), 55, dtype=torch.int8, device="cuda")
    loose[:, 4:204] = kept.codes
    assert torch.equal(Rows8(loose[:, 4:204], kept.exponents, torch.float32).restore(), kept.restore())
    module = torch.nn.Sequential(torch.nn.Linear(200, 128), torch.nn.ReLU(), torch.nn.Linear(128, 18, bias=False)).cuda()
    small = torch.nn.Sequential(torch.nn.Linear(200, 64), torch.nn.ReLU(), torch.nn.Linear(64, 18, bias=False)).cuda()
    good = torch.nn.Sequential(torch.nn.Linear(66, 128), torch.nn.ReLU(), torch.nn.Linear(128, 18, bias=False)).cuda()
    bad = [(TypeError, "x: expected", lambda: compress_rows(x.double())), (TypeError, "CUDA", lambda: compress_rows(x.cpu())),
           (RuntimeError, "at least one column", lambda: compress_rows(x[:, :0])), (RuntimeError, "no backward", lambda: compress_rows(x.clone().requires_grad_(True))),
           (RuntimeError, "exponents must have shape", lambda: Rows8(kept.codes, kept.exponents[:3], torch.float32).restore()),
           (TypeError, "dtype", lambda: kept.restore(torch.int32)), (ValueError, "checkpoint=True", lambda: apply_mlp(module, x, checkpoint=True)),
           (ValueError, "checkpoint=True", lambda: apply_mlp(small, x, checkpoint=True)), (TypeError, "z: expected a float32", lambda: apply_mlp(good, x[:, :66].double(), checkpoint=True)),
           (RuntimeError, "66 columns", lambda: apply_mlp(good, x, checkpoint=True))]
    for error, text, call in bad:
        with pytest.raises(error, match=text):
            call()


def _mlp(k, o, seed=0):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Linear(k, 128), torch.nn.ReLU(), torch.nn.Linear(128, o, bias=False)).cuda()


def _run(module, z, up, checkpoint=True, wanted=None):
    from npa_b200.mlp import apply_mlp
    z = z.detach().clone().requires_grad_(True)
    y = apply_mlp(module, z, checkpoint=checkpoint)
    return [y.detach(), *torch.autograd.grad(y, [z, *module.parameters()], up)]


def _magnitudes(z, w1, b1, w2, up):
    """Sums of magnitudes behind (y, dz, dW1, db1, dW2)."""
    alive = (z.double() @ w1.double().t() + b1.double() > 0).double()
    held, z, w1, b1, w2, up = (t.detach().double().abs().to(z.device) for t in (ref.kept(z), z, w1, b1, w2, up))
    h, dh = (torch.maximum(z, held) @ w1.t() + b1) * alive, (up @ w2) * alive
    return h @ w2.t(), dh @ w1, dh.t() @ held, dh.sum(0), up.t() @ h


NAMES = ["y", "dz", "dW1", "db1", "dW2"]
SHAPES = [(1, 66, 18), (3, 1, 1), (31, 175, 48), (127, 43, 11), (128, 163, 35), (129, 66, 18), (1000, 34, 10), (2048, 5, 48), (4103, 163, 35), (20001, 83, 19), (5000, 176, 33), (777, 64, 16), (300, 96, 32),
          (50000, 130, 34), (65536, 16, 16), (262144, 163, 35)]


@pytest.mark.parametrize("rows,k,o", SHAPES)
def test_gradients_match_float64_truth(rows, k, o):
    """Held to 64 bits, with torch's own float32 run of the same formula beside.

    An output is a sum of products behind another one.  A product of numbers split into heads and tails of 11 bits is off by 2^-21 of
    its magnitude at most, in each of the two layers; the tensor cores add up to 22 steps of three products in a chain and cut off 2^-24
    of the sum's magnitude each time: 2 * 2^-21 + 66 * 2^-24 = 4.9e-6 of the sum of the magnitudes, which is what `size` is (of the
    output's own size it is more where terms cancel: a sum of 128 hidden units behind one input is a fortieth of its terms)."""
    module = _mlp(k, o)
    w1, b1, w2 = module.parameters()
    z = ref.clear_of_the_corner(_rand(rows + rows // 8 + 64, k, seed=1) * torch.exp(0.5 * _rand(1, k, seed=2).clamp(-2, 2)), w1, b1)[:rows]
    up = _rand(rows, o, seed=3)
    assert len(z) == rows
    truth = ref.mlp_with_checkpoint(z, w1, b1, w2, up)
    theirs = ref.mlp_with_checkpoint(z, w1, b1, w2, up, torch.float32)
    size = _magnitudes(z, w1, b1, w2, up)
    for name, a, b, t, m in zip(NAMES, _run(module, z, up), theirs, truth, size):
        scale = float(m.max())
        ours, torchs = float((a.double() - t).abs().max()), float((b.double() - t).abs().max())
        assert ours <= 4 * torchs + 5e-6 * scale, (name, ours, torchs, scale)
        norm = float((a.double() - t).norm() / t.norm())
        print(f"{name}: error {ours:.3e} (torch fp32 {torchs:.3e}) at scale {scale:.3e}; in norm {norm:.2e}")


def test_against_the_plain_backward():
    """y, dz and db1 those of the 32-bit pass to the rounding of both (twice the bar above); dW1 and dW2 within what half a unit of each
    code can move them."""
    from npa_b200.rows8 import compress_rows
    module = _mlp(66, 18)
    w1, b1, w2 = (p.detach().double() for p in module.parameters())
    z, up = ref.clear_of_the_corner(_rand(5000, 66, seed=1), w1, b1)[:4000], _rand(4000, 18, seed=2)
    kept, plain = _run(module, z, up), _run(module, z, up, checkpoint=False)
    size = _magnitudes(z, *module.parameters(), up)
    for k in (0, 1, 3):
        assert float((kept[k] - plain[k]).abs().max()) <= 1e-5 * float(size[k].max())
    half = torch.repeat_interleave(torch.exp2(compress_rows(z).exponents.double() - 134), 32, -1)[:, :66]
    alive = (z.double() @ w1.t() + b1 > 0).double()
    dh = (up.double() @ w2) * alive
    room1, room2 = dh.abs().t() @ half, up.double().abs().t() @ (half @ w1.abs().t() * alive)
    for k, room in ((2, room1), (4, room2)):
        off = (kept[k] - plain[k]).double().abs()
        assert (off <= 1.001 * room + 4e-6 * float(plain[k].abs().max())).all()
        assert float(off.max()) > 0  # it is the rounded input that was read


def test_against_differences():
    """On an input that 8 bits hold exactly the gradients are those of the function: central differences in 64 bits."""
    module = _mlp(40, 7)
    w1, b1, w2 = (p.detach() for p in module.parameters())
    g = torch.Generator(device="cuda").manual_seed(0)
    z = torch.randint(-127, 128, (400, 40), device="cuda", generator=g).float() / 64
    z[:, 0], z[:, 33] = 127 / 64, -100 / 64  # each group's largest: units of 1 / 64
    z = ref.clear_of_the_corner(z, w1, b1)[:300]
    assert torch.equal(ref.kept(z).float(), z.cpu())
    up = _rand(len(z), 7, seed=3)
    got = _run(module, z, up)
    args = [t.double() for t in (z, w1, b1, w2)]

    def loss(args):
        z, w1, b1, w2 = args
        return float((((z @ w1.t() + b1).clamp_min(0) @ w2.t()) * up.double()).sum())

    for which, grad in enumerate(got[1:]):
        direction = torch.randn(args[which].shape, device="cuda", dtype=torch.float64, generator=g)
        step = 1e-7  # far below the distance of any unit from the corner: the loss is linear in each argument alone
        ends = []
        for sign in (1, -1):
            moved = list(args)
            moved[which] = args[which] + sign * step * direction
            ends.append(loss(moved))
        slope = (ends[0] - ends[1]) / (2 * step)
        along = float((grad.double() * direction).sum())
        # rounding of the differences: 2^-53 of the sum of magnitudes over the step; of the gradient: the bar of 4e-6 of its largest, per element
        size = float((up.double().abs() @ w2.double().abs()).sum()) * 5
        room = size * 2.0 ** -50 / step + 4e-6 * float(grad.abs().max()) * float(direction.abs().sum())
        assert abs(slope - along) <= room, (which, slope, along, room)


def test_what_is_asked_for_and_what_is_kept():
    """Gradients of some inputs only, twice through one graph, an input of no rows, memory held, changes in place noticed."""
    from npa_b200.mlp import apply_mlp
    module = _mlp(66, 18)
    z, up = _rand(3, 500, 66, seed=1), _rand(3, 500, 18, seed=2)
    full = _run(module, z, up)
    y = apply_mlp(module, z, checkpoint=True)  # z needs none
    for a, b in zip(torch.autograd.grad(y, list(module.parameters()), up, retain_graph=True), full[2:]):
        assert torch.equal(a, b)
    for a, b in zip(torch.autograd.grad(y, list(module.parameters()), up), full[2:]):
        assert torch.equal(a, b)
    zr = z.clone().requires_grad_(True)
    y = apply_mlp(module, zr, checkpoint=True)
    assert torch.equal(torch.autograd.grad(y, zr, up.expand(3, 500, 18))[0], full[1])
    for p in module.parameters():
        p.requires_grad_(False)
    assert torch.equal(torch.autograd.grad(apply_mlp(module, zr, checkpoint=True), zr, up)[0], full[1])
    with torch.no_grad():
        assert torch.equal(apply_mlp(module, zr, checkpoint=True), apply_mlp(module, zr))
    for p in module.parameters():
        p.requires_grad_(True)
    y = apply_mlp(module, z[:, :0], checkpoint=True)
    assert y.shape == (3, 0, 18) and all(float(t.abs().sum()) == 0 for t in torch.autograd.grad(y.sum(), list(module.parameters())))
    y = apply_mlp(module, z, checkpoint=True)
    with torch.no_grad():
        module[2].weight.mul_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(up)
    big = torch.randn(100000, 66, device="cuda")
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = apply_mlp(module, big, checkpoint=True)
    held = torch.cuda.memory_allocated() - before - y.numel() * 4
    assert held <= 100000 * (80 + 3 + 16) + (1 << 21)
    big.zero_()  # nothing of the input itself is kept
    y.sum().backward()


def test_rows_that_are_not_finite():
    """They make the gradient of the first weights NaN, as in 32 bits, and leave the gradients of other rows alone; so do zero rows and
    rows of very different sizes.  (The hidden layer of such a row is zero: the MLP's ReLU is fmaxf(NaN, 0), with or without checkpoint.)"""
    module = _mlp(66, 18)
    w1, b1, w2 = module.parameters()
    z = ref.clear_of_the_corner(_rand(400, 66, seed=1), w1, b1)[:300]
    z = z * torch.exp2(torch.randint(-40, 20, (300, 1), device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)).float())
    z[7] = 0
    z = ref.clear_of_the_corner(z, w1, b1)
    up = _rand(len(z), 18, seed=2) * torch.exp2(torch.randint(-30, 30, (len(z), 1), device="cuda", generator=torch.Generator(device="cuda").manual_seed(6)).float())
    truth = ref.mlp_with_checkpoint(z, w1, b1, w2, up)
    got = _run(module, z, up)
    rows = (got[1].double() - truth[1]).abs().amax(1) / truth[1].abs().amax(1)
    assert float(rows.max()) <= 4e-6  # each row to its own size
    for a, t in zip(got[2:], truth[2:]):
        assert float((a.double() - t).abs().max()) <= 4e-6 * float(t.abs().max())
    z[5, 3] = float("nan")
    bad = _run(module, z, up)
    plain = _run(module, z, up, checkpoint=False)
    assert torch.isnan(plain[2]).any() and torch.isnan(bad[2])[torch.isnan(plain[2])].all() and not torch.isnan(plain[4]).any() and not torch.isnan(bad[4]).any()
    rest = torch.arange(len(z), device="cuda") != 5
    assert torch.equal(bad[1][rest], got[1][rest]) and torch.equal(bad[0][rest], got[0][rest])


def test_two_runs_are_bit_identical_on_any_stream():
    module = _mlp(163, 35)
    z, up = _rand(30000, 163, seed=1), _rand(30000, 35, seed=2)
    first = _run(module, z, up)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for r in range(4):
        with torch.cuda.stream(streams[r % 2]):
            got.append(_run(module, z, up))
    torch.cuda.synchronize()
    for out in got:
        for a, b in zip(first, out):
            assert torch.equal(a, b)


def test_a_captured_training_pass():
    """Forward and backward recorded in a graph and replayed on new inputs; two graphs at once."""
    from npa_b200.mlp import apply_mlp
    module = _mlp(66, 18)
    inputs = [(_rand(3000, 66, seed=k), _rand(3000, 18, seed=10 + k)) for k in range(3)]
    want = [_run(module, *i) for i in inputs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _run(module, *inputs[0])
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for k in range(2):
        z, up = inputs[k][0].clone().requires_grad_(True), inputs[k][1].clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = apply_mlp(module, z, checkpoint=True)
            outs = [y, *torch.autograd.grad(y, [z, *module.parameters()], up)]
        graphs.append((g, z, up, [o.detach() for o in outs]))
    for k, (g, z, up, _) in enumerate(graphs):
        with torch.no_grad():
            z.copy_(inputs[k + 1][0])
            up.copy_(inputs[k + 1][1])
    for g, *_ in graphs:
        g.replay()
    torch.cuda.synchronize()
    for k, (_, _, _, outs) in enumerate(graphs):
        for a, b in zip(outs, want[k + 1]):
            assert torch.equal(a, b)


class _Model(torch.nn.Module):
    def __init__(self, dim, C):
        super().__init__()
        self.model = torch.nn.Sequential(torch.nn.Linear(2 * C + C * dim + dim, 128), torch.nn.ReLU(), torch.nn.Linear(128, dim + C, bias=False))
        self.eps0, self.alpha, self.spatial_dims = 0.1, 0.5, dim


@pytest.mark.parametrize("dim,C,N", [(2, 16, 2500), (3, 12, 3001)])
def test_training_steps(dim, C, N):
    """A rollout of steps with checkpoints: states as without, gradients of the states as without, and those of the weights as from the
    same rollout with a plain torch MLP of the same formula."""
    from npa_b200 import sphops as sph, stepping
    torch.manual_seed(1)
    model = _Model(dim, C).cuda()
    grid = sph.HashGrid(dim=dim, boundary="clamped", mode="grid", grid_size=(8,) * dim, eps=0.15, num_particles=N, batch_size=2)
    x = torch.rand(2, N, dim, device="cuda") - 0.5
    x = x if dim == 2 else torch.cat([x, torch.zeros_like(x[..., :1])], -1).contiguous()
    s = torch.randn(2, N, C, device="cuda")

    class Plain(torch.autograd.Function):
        @staticmethod
        def forward(ctx, z, w1, b1, w2):
            before = z @ w1.t() + b1
            ctx.save_for_backward(ref.kept(z).to(z), before > 0, w1, b1, w2)
            return before.clamp_min(0) @ w2.t()

        @staticmethod
        def backward(ctx, up):
            z, alive, w1, b1, w2 = ctx.saved_tensors
            z, alive, flat = z.flatten(0, 1), alive.flatten(0, 1), up.flatten(0, 1)
            dh = (flat @ w2) * alive
            h = (z @ w1.t() + b1) * alive
            return (dh @ w1).view(*up.shape[:2], -1), dh.t() @ z, dh.sum(0), flat.t() @ h

    def rollout(**how):
        torch.manual_seed(2)
        sr = s.clone().requires_grad_(True)
        xx, ss = x, sr
        for _ in range(2):
            xx, ss, _ = stepping.step_euler(model, xx, ss, grid, **how)
        grads = torch.autograd.grad(ss.square().mean() + xx.square().mean(), [sr, *model.parameters()])
        return [xx.detach(), ss.detach(), *grads]

    kept, plain = rollout(checkpoint=True), rollout()
    real = stepping.apply_mlp
    stepping.apply_mlp = lambda module, z, checkpoint: Plain.apply(z, module[0].weight, module[0].bias, module[2].weight)
    try:
        formula = rollout(checkpoint=True)
    finally:
        stepping.apply_mlp = real
    # Between the paths lie roundings of 1e-7.  Of 640,000 to 770,000 hidden units a step about one lies so near its corner that it falls
    # the other way, which moves its row's gradient by an eighth (one of 64 units alive) and that of all of 5,000 rows by 2e-3 in norm;
    # thirty such units move it by 1e-2.  The states themselves are continuous.
    for k in range(2):
        assert float((kept[k] - plain[k]).norm()) <= 1e-5 * float(plain[k].norm()), k
    assert float((kept[2] - plain[2]).norm()) <= 1e-2 * float(plain[2].norm())
    for k in range(3, 6):
        assert float((kept[k] - formula[k]).norm()) <= 1e-2 * float(formula[k].norm()), k


def test_saved_on_the_host_and_recomputed():
    """Saved-tensor hooks see what the MLP keeps: moved to the host and back, dropped and recomputed, or refused when it comes back changed."""
    from npa_b200.mlp import apply_mlp
    module = _mlp(83, 19)
    z, up = _rand(700, 83, seed=1), _rand(700, 19, seed=2)
    want = _run(module, z, up)
    with torch.autograd.graph.save_on_cpu():
        zr = z.clone().requires_grad_(True)
        y = apply_mlp(module, zr, checkpoint=True)
    for a, b in zip(torch.autograd.grad(y, [zr, *module.parameters()], up), want[1:]):
        assert torch.equal(a, b)
    zr = z.clone().requires_grad_(True)
    y = torch.utils.checkpoint.checkpoint(lambda t: apply_mlp(module, t, checkpoint=True), zr, use_reentrant=False)
    for a, b in zip(torch.autograd.grad(y, [zr, *module.parameters()], up), want[1:]):
        assert torch.equal(a, b)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t[:-1] if t.dtype == torch.uint8 else t):
        y = apply_mlp(module, z, checkpoint=True)
    with pytest.raises(RuntimeError, match="saved-tensor hook"):
        torch.autograd.grad(y, list(module.parameters()), up)


@pytest.mark.parametrize("k,o", [(66, 18), (163, 35)])
def test_strided_parameters_and_upstream(k, o):
    """Transposed weights, a bias with gaps, upstream gradients that are broadcast or lie transposed or off 16 bytes."""
    from npa_b200 import _native as n
    module = _mlp(k, o)
    w1, b1, w2 = (p.detach() for p in module.parameters())
    z, up = _rand(1000, k, seed=1), _rand(1000, o, seed=2)
    want = _run(module, z, up)
    w1t, w2t = w1.t().contiguous().t(), w2.t().contiguous().t()
    gap = torch.zeros(256, device="cuda")[::2]
    gap.copy_(b1)
    odd = torch.empty(1000 * o + 1, device="cuda")[1:].view(1000, o)
    odd.copy_(up)
    leaves = [t.requires_grad_(True) for t in (z.clone(), w1t, gap, w2t)]
    y = n.ops.mlp_checkpoint(*leaves)
    for upstream in (up, up.t().contiguous().t(), odd):
        got = [y.detach(), *torch.autograd.grad(y, leaves, upstream, retain_graph=True)]
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    one = torch.autograd.grad(y, leaves, up[:1].expand(1000, o), retain_graph=True)
    for a, b in zip(one, _run(module, z, up[:1].expand(1000, o).contiguous())[1:]):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda t: n.ops.mlp_checkpoint(t, w1t, gap, w2t), (z,), (z,))


def test_upstream_that_is_not_finite():
    """An infinity in one row's upstream gradient stays in that row of dz and in the units alive there; masked units do not see it."""
    module = _mlp(66, 18)
    w1, b1, w2 = (p.detach() for p in module.parameters())
    z = ref.clear_of_the_corner(_rand(400, 66, seed=1), w1, b1)[:300]
    up = _rand(300, 18, seed=2) * 1e-6
    want = _run(module, z, up)
    alive = (z.double() @ w1.double().t() + b1.double() > 0)[5]
    up[5, 2] = float("inf")
    got = _run(module, z, up)
    rest = torch.arange(300, device="cuda") != 5
    assert torch.equal(got[1][rest], want[1][rest]) and not torch.isfinite(got[1][5]).all()
    assert not torch.isfinite(got[3][alive]).any() and torch.isfinite(got[3][~alive]).all()
    # the row's finite share of the dead units' gradient is zero, so what they had stays to the rounding of their sum
    assert float((got[2][~alive] - want[2][~alive]).abs().max()) <= 4e-6 * float(want[2].abs().max())
    others = torch.arange(18, device="cuda") != 2
    assert torch.isfinite(got[4][others]).all() and not torch.isfinite(got[4][2]).all()


@pytest.mark.parametrize("cols", [33, 66, 100, 163, 240])
@pytest.mark.parametrize("offset", [0, 1])
def test_what_follows_a_row_of_codes_stays_as_it_was(cols, offset):
    """Rows of codes inside wider ones: the columns behind them belong to the caller, whichever way the values are read."""
    from npa_b200 import _native as n
    rows, pitch = 77, 256
    x = _rand(rows * cols + offset, seed=5).cuda()[offset:]
    stream, at = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream), lambda t: ctypes.c_void_p(t.data_ptr())
    exps, scales = torch.zeros(rows * 8, dtype=torch.uint8, device="cuda"), torch.zeros(rows, device="cuda")
    packed = (cols + 15) // 16 * 16
    for call in (lambda c, p: n.lib.npa_rows8_compress(at(x), 0, cols, rows, cols, at(c), p, at(exps), stream),
                 lambda c, p: n.lib.npa_quantize_rows(at(x), 0, cols, rows, cols, at(c), 3, p, at(scales), stream)):
        wide, narrow = (torch.full((rows, p), 99, dtype=torch.int8, device="cuda") for p in (pitch, packed))
        assert call(wide, pitch) == 0 and call(narrow, packed) == 0
        assert (wide[:, cols:] == 99).all()
        assert torch.equal(wide[:, :cols], narrow[:, :cols])


@pytest.mark.parametrize("k, o", [(32, 32), (64, 16), (96, 48), (100, 20), (128, 32), (144, 40), (160, 48), (176, 44)])
def test_rows_whose_starts_share_banks(k, o):
    """Widths of a multiple of four leave in pieces of 16 bytes, in an order of their own for each row."""
    module = _mlp(k, o, seed=k)
    z, up = _rand(1000, k, seed=1), _rand(1000, o, seed=2)
    full = _run(module, z, up)
    w1, b1, w2 = (p.detach().double() for p in module.parameters())
    h = z.double() @ w1.T + b1
    y, dz = h.relu() @ w2.T, ((up.double() @ w2) * (h > 0)) @ w1
    # sums of k and 128 products at 32 bits, against the size of what is summed; the few units of the ReLU within rounding of
    # zero are left out with their rows
    sizes = (z.double().abs() @ w1.abs().T + b1.abs()) @ w2.abs().T, (up.double().abs() @ w2.abs()) @ w1.abs()
    clear = (h.abs() > 1e-5 * (z.double().abs() @ w1.abs().T + b1.abs())).all(1)
    assert clear.sum() > 900
    assert ((full[0] - y).abs() <= 5e-6 * sizes[0]).all()
    assert ((full[1] - dz).abs() <= 5e-6 * sizes[1])[clear].all()
    # what one backward asks for is what it makes, and the same
    from npa_b200.mlp import apply_mlp
    zr = z.clone().requires_grad_(True)
    part = torch.autograd.grad(apply_mlp(module, zr, checkpoint=True), list(module.parameters()), up)
    assert all(torch.equal(a, b) for a, b in zip(part, full[2:]))
    assert torch.equal(torch.autograd.grad(apply_mlp(module, zr, checkpoint=True), zr, up)[0], full[1])
