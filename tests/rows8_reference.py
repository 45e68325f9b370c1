"""The definitions of the 8-bit operators in 64 bits, on the CPU, for the tests of int8 and rows8."""
import torch

FLOOR = 2.0 ** -126


def quantized(x, unsigned=False):
    """Codes (int64) and scales (float32) of rows, from the exact quotient."""
    x = x.detach().cpu().double()
    finite = torch.isfinite(x).all(-1)
    x = torch.where(finite[..., None], x, torch.zeros_like(x))
    if unsigned:
        x = x.clamp_min(0)
    scale = (x.abs().amax(-1) / (255 if unsigned else 127)).float().clamp_min(FLOOR)
    codes = torch.round(x / scale.double()[..., None]).long()
    return codes, torch.where(finite, scale, torch.full_like(scale, float("nan")))


def linear(codes, scales, w, w_scales, bias=None, relu=False, dtype=torch.float32):
    """Each operation behind the exact sum rounded to float32, the result to ``dtype``: bit by bit what the operator gives."""
    total = codes.cpu().double() @ w.cpu().double().t()
    out = total.float() * (scales.cpu().float()[..., None] * w_scales.cpu().float())
    if bias is not None:
        out = out + bias.cpu().float()
    if relu:
        out = torch.where(out < 0, torch.zeros_like(out), out)
    return out.to(dtype)


def kept(x):
    """What 8-bit rows hold of x, in float64; NaN in a group that is not finite."""
    x = x.detach().cpu().double()
    out = torch.empty_like(x)
    for k in range(0, x.shape[-1], 32):
        part = x[..., k:k + 32]
        most = part.abs().amax(-1, keepdim=True)
        bad = ~torch.isfinite(part).all(-1, keepdim=True)
        part, most = torch.where(bad, torch.zeros_like(part), part), torch.where(bad, torch.zeros_like(most), most)
        e = torch.frexp(most)[1].double() - 7  # 64 to 128 units
        e = torch.where(torch.round(most / torch.exp2(e)) > 127, e + 1, e).clamp(-126, 121)
        value = torch.round(part / torch.exp2(e)).clamp(-127, 127) * torch.exp2(e)
        out[..., k:k + 32] = torch.where(bad, torch.full_like(value, float("nan")), value)
    return out


def mlp_with_checkpoint(z, w1, b1, w2, up, dtype=torch.float64):
    """(y, dz, dW1, db1, dW2) of the adaptation MLP whose backward sees ``kept(z)`` and the mask of the forward."""
    held = kept(z).to(dtype).to(z.device)
    z, w1, b1, w2, up = (t.detach().to(dtype) for t in (z, w1, b1, w2, up))
    z, held, up = z.reshape(-1, z.shape[-1]), held.reshape(-1, z.shape[-1]), up.reshape(-1, up.shape[-1])
    before = z @ w1.t() + b1
    alive = before > 0
    h = torch.where(alive, held @ w1.t() + b1, torch.zeros_like(before))
    dh = torch.where(alive, up @ w2, torch.zeros_like(before))
    return before.clamp_min(0) @ w2.t(), dh @ w1, dh.t() @ held, dh.sum(0), up.t() @ h


def clear_of_the_corner(z, w1, b1):
    """Rows of z with no hidden unit within the rounding of 32 bits of the ReLU's corner, where the derivative has two values."""
    wide, w, b = z.double(), w1.double(), b1.double()
    near = (wide @ w.t() + b).abs() < 1e-5 * (wide.abs() @ w.abs().t() + b.abs())
    return z[~near.any(1)]
