"""The 8-bit operators of the package as measurable cases.

A case is a dict of plain values.  ``kind`` says what a pass is:

* ``linear``  a product of rows and a weight matrix in 8-bit integers, with a scale for each row and each output
              channel (``int8.linear_int8``); the rows are given in floating point, or as codes with their scales;
* ``mlp``     the adaptation MLP of a particle model in 8-bit integers, both layers (``int8.mlp_int8``);
* ``rows``    activations into 8 bits and back, as a checkpoint holds them (``rows8.compress_rows``, ``restore``);
* ``train``   the adaptation MLP forward and backward, with nothing kept in between but 8-bit rows and the bits of the
              ReLU (``mlp.apply_mlp(..., checkpoint=True)``).

``own`` selects the package's operators; otherwise a pass computes the same values by elementary torch operations.
"""
from __future__ import annotations

import math

import torch

own = False

HIDDEN = 128  # width of the per-particle MLP
GROUP = 32    # columns that share an exponent in 8-bit rows
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
LARGEST = 8192 * 4096 * 4096  # products in one pass


def listed():
    return [
        # One token through a square layer: nothing but reading the weights, and latency.
        dict(name="linear_one_token", kind="linear", M=1, K=4096, N=4096, dtype="bfloat16", bias=False, relu=False, codes=False),
        # A handful of rows through an odd layer with everything on.
        dict(name="linear_few_odd", kind="linear", M=13, K=1000, N=1537, dtype="float32", bias=True, relu=True, codes=False),
        # Rows of a small batch that an earlier layer has left as codes.
        dict(name="linear_batch_codes", kind="linear", M=333, K=2048, N=5120, dtype="float16", bias=True, relu=False, codes=True),
        # A whole prompt, or the particles of a wide model: the tensor cores' case.
        dict(name="linear_prompt", kind="linear", M=8192, K=4096, N=4096, dtype="bfloat16", bias=True, relu=False, codes=False),
        # An interactive rollout of one small system in 2D with 16 features.
        dict(name="mlp_interactive", kind="mlp", M=2500, K=66, N=18),
        # The largest 3D systems with 32 features: 4 x 65,536 particles.
        dict(name="mlp_splat", kind="mlp", M=262144, K=163, N=35),
        # Perception rows of an everyday 2D step.
        dict(name="rows_growing", kind="rows", M=32768, K=66, dtype="float32"),
        # Activations of a wide model in half the bytes, odd sizes.
        dict(name="rows_wide_odd", kind="rows", M=8191, K=4100, dtype="bfloat16"),
        # Training of a single small system.
        dict(name="train_small", kind="train", M=2500, K=66, N=18),
        # The everyday training step in 2D: 8 systems of 4,096 particles.
        dict(name="train_growing", kind="train", M=32768, K=66, N=18),
        # An odd number of particles in 3D with 16 features.
        dict(name="train_odd_3d", kind="train", M=65537, K=83, N=19),
        # The largest 3D training step: 4 systems of 65,536 particles with 32 channels.
        dict(name="train_splat", kind="train", M=262144, K=163, N=35),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "mlp", "rows", "train", "train"])
    if kind == "linear":
        K, N = _log_uniform(rng, 16, 8192), _log_uniform(rng, 8, 8192)
        M = _log_uniform(rng, 1, max(1, min(65536, LARGEST // (K * N))))
        return dict(kind=kind, M=M, K=K, N=N, dtype=rng.choice(sorted(TYPES)), bias=rng.random() < 0.5, relu=rng.random() < 0.25,
                    codes=rng.random() < 0.25)
    if kind == "rows":
        K = _log_uniform(rng, 1, 8192)
        return dict(kind=kind, M=_log_uniform(rng, 1, max(1, min(262144, 262144 * 163 // K))), K=K, dtype=rng.choice(sorted(TYPES)))
    dim, C = rng.choice([2, 3]), rng.choice([8, 12, 13, 16, 16, 20, 24, 32])
    return dict(kind=kind, M=_log_uniform(rng, 1, 262144), K=2 * C + C * dim + dim, N=dim + C)


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _uniform(shape, bound, g):
    return torch.empty(shape, device="cuda").uniform_(-bound, bound, generator=g)


def _activations(M, K, g, spread=0.5):
    """Rows of different size with features of different size, one row in 32 close to nothing (particles that do not live)."""
    x = torch.randn(M, K, device="cuda", generator=g)
    x *= torch.exp(spread * torch.randn(K, device="cuda", generator=g))
    size = torch.exp(spread * torch.randn(M, 1, device="cuda", generator=g))
    dead = torch.rand(M, 1, device="cuda", generator=g) < 1 / 32
    return x * torch.where(dead, 1e-4 * size, size)


def _weight_codes(w):
    """A weight matrix as an 8-bit model keeps it: codes in rows whose pitch is a multiple of 16 bytes, and a scale for each row."""
    wide = w.double()
    scale = (wide.abs().amax(1) / 127).float()
    codes = torch.zeros(w.shape[0], -(-w.shape[1] // 16) * 16, dtype=torch.int8, device=w.device)
    codes[:, : w.shape[1]] = torch.round(wide / scale.double()[:, None]).to(torch.int8)
    return codes[:, : w.shape[1]], scale


def _clear_of_the_corner(M, K, w1, b1, g):
    """Rows none of whose hidden units lies at the ReLU's corner within the rounding of 32 bits: there the derivative has two values,
    and which one is taken is a matter of the order of a sum."""
    z = _activations(M + M // 8 + 64, K, g)
    wide, w, b = z.double(), w1.double(), b1.double()
    near = (wide @ w.t() + b).abs() < 1e-5 * (wide.abs() @ w.abs().t() + b.abs())
    return z[torch.nonzero(~near.any(1)).flatten()[:M]].contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c, kind = dict(case), case["kind"]
    M, K = c["M"], c["K"]
    if kind == "rows":
        c["x"] = _activations(M, K, g).to(TYPES[c["dtype"]])
        return c
    N = c["N"]
    if kind == "linear":
        dtype = TYPES[c["dtype"]]
        x = _activations(M, K, g)
        c["w"], c["w_scale"] = _weight_codes(_uniform((N, K), K ** -0.5, g) * torch.exp(0.3 * torch.randn(N, 1, device="cuda", generator=g)))
        c["b"] = _uniform((N,), 0.5, g).to(dtype) if c["bias"] else None
        if c["codes"]:
            c["x"], c["x_scale"] = _weight_codes(x)
        else:
            c["x"], c["x_scale"] = x.to(dtype), None
        return c
    w1, b1, w2 = _uniform((HIDDEN, K), K ** -0.5, g), _uniform((HIDDEN,), K ** -0.5, g), _uniform((N, HIDDEN), HIDDEN ** -0.5, g)
    if kind == "mlp":
        c["z"], c["b1"] = _activations(M, K, g), b1
        (c["w1"], c["w1_scale"]), (c["w2"], c["w2_scale"]) = _weight_codes(w1), _weight_codes(w2)
        return c
    module = torch.nn.Sequential(torch.nn.Linear(K, HIDDEN), torch.nn.ReLU(), torch.nn.Linear(HIDDEN, N, bias=False)).to("cuda")
    with torch.no_grad():
        module[0].weight.copy_(w1)
        module[0].bias.copy_(b1)
        module[2].weight.copy_(w2)
    c["module"] = module
    c["z"] = _clear_of_the_corner(M, K, w1, b1, g).requires_grad_(True)
    c["up"] = torch.randn(M, N, device="cuda", generator=g) * torch.exp(0.5 * torch.randn(M, 1, device="cuda", generator=g))
    return c


# ---- a pass ----------------------------------------------------------------------------------------------------------
def _codes(x, most):
    """Codes (as whole numbers in floating point) and scales of rows; the quotient is rounded from 64 bits, because in 32 it may come to
    lie on the border between two codes."""
    scale = (x.abs().amax(-1).double() / most).float().clamp_min(2.0 ** -126)
    return torch.round(x.double() / scale.double()[:, None]), scale


def _product(a, b):
    """a b^T of whole numbers below 256, exact: in 32 bits where every sum is below 2^24."""
    if a.shape[1] * 255 * 127 <= 1 << 24:
        return a.float() @ b.float().t()
    return (a.double() @ b.double().t()).float()


def _plain_linear(c):
    x, scale = (c["x"], c["x_scale"]) if c["codes"] else _codes(c["x"].float(), 127)
    out = _product(x, c["w"]) * (scale[:, None] * c["w_scale"])
    if c["b"] is not None:
        out = out + c["b"].float()
    if c["relu"]:
        out = out.clamp_min(0)
    return out.to(TYPES[c["dtype"]])


def _plain_mlp(c):
    q, scale = _codes(c["z"], 127)
    h = (_product(q, c["w1"]) * (scale[:, None] * c["w1_scale"]) + c["b1"]).clamp_min(0)
    p, scale = _codes(h, 255)
    return _product(p, c["w2"]) * (scale[:, None] * c["w2_scale"])


def _eight_bits(x):
    """What 8-bit rows hold of x, in 32 bits: groups of 32 columns with a common power of two."""
    M, K = x.shape
    groups = -(-K // GROUP)
    x = torch.nn.functional.pad(x.float(), (0, groups * GROUP - K)).reshape(M, groups, GROUP)
    most = x.abs().amax(2, keepdim=True)
    exponent = ((most.view(torch.int32) + 0x10000) >> 23).clamp(7, 254)
    step = ((exponent - 133 + 127) << 23).view(torch.float32)  # 2^(exponent - 133)
    return (torch.round(x / step).clamp(-127, 127) * step).reshape(M, groups * GROUP)[:, :K]


def _plain_train(c):
    w1, b1, w2 = (p.detach() for p in c["module"].parameters())
    z, up = c["z"].detach(), c["up"]
    h = (z @ w1.t() + b1).clamp_min(0)
    y, alive = h @ w2.t(), (h > 0).float()
    kept = _eight_bits(z)
    again = (kept @ w1.t() + b1) * alive
    dh = (up @ w2) * alive
    return [y, dh @ w1, dh.t() @ kept, dh.sum(0), up.t() @ again]


def run(state):
    c, kind = state, state["kind"]
    if not own:
        if kind == "linear":
            return _plain_linear(c)
        if kind == "mlp":
            return _plain_mlp(c)
        if kind == "rows":
            return _eight_bits(c["x"]).to(c["x"].dtype)
        return _plain_train(c)
    if kind == "linear":
        from npa_b200.int8 import linear_int8
        return linear_int8(c["x"], c["w"], c["w_scale"], bias=c["b"], relu=c["relu"], x_scales=c["x_scale"], out_dtype=TYPES[c["dtype"]])
    if kind == "mlp":
        from npa_b200.int8 import mlp_int8
        return mlp_int8(c["z"], c["w1"], c["w1_scale"], c["b1"], c["w2"], c["w2_scale"])
    if kind == "rows":
        from npa_b200.rows8 import compress_rows
        return compress_rows(c["x"]).restore()
    from npa_b200.mlp import apply_mlp
    y = apply_mlp(c["module"], c["z"], checkpoint=True)
    return [y.detach(), *torch.autograd.grad(y, [c["z"], *c["module"].parameters()], c["up"])]


def work(case):
    M, K, kind = case["M"], case["K"], case["kind"]
    size = 4 if case.get("dtype", "float32") == "float32" else 2
    if kind == "linear":
        N = case["N"]
        rows = M * K + 4 * M if case["codes"] else M * K * size
        return {"bytes": rows + N * K + 4 * N + (N * size if case["bias"] else 0) + M * N * size, "flops": 2 * M * N * K}
    kept = K + -(-K // GROUP)
    if kind == "rows":
        return {"bytes": M * (2 * K * size + 2 * kept), "flops": 4 * M * K}
    N = case["N"]
    if kind == "mlp":
        return {"bytes": 4 * M * (K + N) + HIDDEN * (K + N) + 4 * (2 * HIDDEN + N), "flops": 2 * M * HIDDEN * (K + N)}
    weights = 4 * (HIDDEN * (K + N) + HIDDEN)
    return {"bytes": M * (8 * K + 8 * N + 2 * (kept + HIDDEN // 8)) + 3 * weights, "flops": 2 * M * HIDDEN * (4 * K + 3 * N)}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------
def _exact_rows(x, most):
    """Quantised rows of 64-bit values: the scale is a number of 32 bits by definition."""
    largest = torch.maximum(x.max(dim=1).values, -x.min(dim=1).values)
    scale = torch.maximum((largest / most).float().double(), torch.tensor(2.0 ** -126, dtype=torch.float64, device=x.device))
    q = x / scale[:, None]
    low = torch.floor(q)
    up = (q - low > 0.5) | ((q - low == 0.5) & (torch.remainder(low, 2) == 1))
    return low + up, scale


def exact(case, seed):
    c, kind = prepare(case, seed), case["kind"]
    if kind == "linear":
        if c["codes"]:
            q, scale = c["x"].double(), c["x_scale"].double()
        else:
            q, scale = _exact_rows(c["x"].double(), 127)
        out = torch.einsum("mk,nk->mn", q, c["w"].double()) * scale[:, None] * c["w_scale"].double()
        if c["bias"]:
            out += c["b"].double()
        return torch.relu(out) if c["relu"] else out
    if kind == "mlp":
        q, scale = _exact_rows(c["z"].double(), 127)
        # the hidden row is held in 32 bits, each of its three operations rounded, because the codes of the second layer hang on it
        factor = (scale[:, None] * c["w1_scale"].double()).float().double()
        h = torch.relu(((torch.einsum("mk,nk->mn", q, c["w1"].double()) * factor).float().double() + c["b1"].double()).float().double())
        p, scale = _exact_rows(h, 255)
        return torch.einsum("mk,nk->mn", p, c["w2"].double()) * scale[:, None] * c["w2_scale"].double()
    x = (c["x"] if kind == "rows" else c["z"].detach()).double()
    kept = torch.empty_like(x)
    for k in range(0, x.shape[1], GROUP):
        part = x[:, k: k + GROUP]
        most = part.abs().amax(1, keepdim=True)
        # the smallest power of two in whose units the largest value rounds to at most 127
        exponent = torch.frexp(most)[1].double() - 7
        unit = torch.exp2(torch.where(torch.round(most / torch.exp2(exponent)) > 127, exponent + 1, exponent).clamp(-126, 121))
        kept[:, k: k + GROUP] = torch.round(part / unit).clamp(-127, 127) * unit
    if kind == "rows":
        return kept
    w1, b1, w2 = (p.detach().double() for p in c["module"].parameters())
    up = c["up"].double()
    before = torch.addmm(b1, x, w1.t())
    y = torch.relu(before) @ w2.t()
    dh = torch.where(before > 0, up @ w2, torch.zeros_like(before))
    again = torch.where(before > 0, torch.addmm(b1, kept, w1.t()), torch.zeros_like(before))
    return [y, dh @ w1, dh.t() @ kept, dh.sum(0), up.t() @ again]
