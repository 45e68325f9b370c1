"""Products in 8-bit integers, with a scale for each row (particle, token) and each output channel.

What a model computes in evaluation and in interactive rollouts are products of activations with fixed weights; in 8 bits
the weights are a quarter as large and the tensor cores four times as fast as with single TF32 products.

    q, s = quantize_rows(x)                       # codes int8, scale = max |x| / 127 for each row
    w, t = quantize_rows(linear.weight)           # the weights' channels are the rows of their matrix
    y = linear_int8(x, w, t, bias=linear.bias)    # rows quantised on the way in
    y = linear_int8(q, w, t, x_scales=s)          # or given as codes
    model.model = Int8MLP(model.model)            # both layers of an adaptation MLP; stepping.step_euler runs it

The sum over codes is exact and what surrounds it is rounded operation by operation as the docstrings say, so results do
not depend on the path a call takes, nor on the other rows of a batch.  There is no backward: calls on tensors that
require gradients are refused while gradients are recorded.
"""
from __future__ import annotations

import torch

from . import _native as N


def quantize_rows(x, unsigned=False):
    """``(codes, scales)`` of the rows of ``x`` ``[..., k]`` (float32, float16 or bfloat16, any strides).

    ``scales[...] = max(max |x| / 127, 2**-126)`` rounded to float32; ``codes = x / scales`` rounded to nearest, ties to
    even, int8.  ``unsigned=True`` divides by 255 instead, for rows without numbers below zero (those count as zero), and
    gives uint8.  A row with an infinity or a NaN has the scale NaN.  The rows of ``codes`` lie a multiple of 16 bytes apart."""
    return N.ops.quantize_rows(x, unsigned)


def dequantize_rows(codes, scales, dtype=torch.float32):
    """``codes * scales[..., None]`` in ``dtype``."""
    return N.ops.dequantize_rows(codes, scales, dtype)


def linear_int8(x, w, w_scales, bias=None, relu=False, x_scales=None, out_dtype=None):
    """``x w^T`` of rows ``x`` ``[..., k]`` and weight codes ``w`` ``[n, k]`` (int8, scales ``[n]``) -> ``[..., n]``.

    ``x`` holds numbers, which are quantised as by ``quantize_rows``, or int8 / uint8 codes with ``x_scales``.
    ``out = act(float32(sum) * (x_scales * w_scales) + bias)``, each operation rounded to float32 and the result to
    ``out_dtype`` (the type of ``x``; float32 for codes).  ``k`` is at most 65,536."""
    return N.ops.linear_int8(x, w, w_scales, bias, relu, x_scales, out_dtype)


def mlp_int8(z, w1, w1_scales, b1, w2, w2_scales):
    """Both layers of an adaptation MLP: ``h = relu(z w1^T + b1)`` as ``linear_int8``, ``y = h w2^T`` with ``h`` quantised to
    unsigned codes.  ``z`` ``[..., k]`` float32, ``w1`` ``[hidden, k]``, ``b1`` float32, ``w2`` ``[n, hidden]`` -> ``[..., n]`` float32."""
    return N.ops.mlp_int8(z, w1, w1_scales, b1, w2, w2_scales)


class Int8MLP(torch.nn.Module):
    """``Sequential(Linear, ReLU, Linear(bias=False))`` in float32, for evaluation in 8-bit integers (``mlp_int8``).

    Takes the place of ``model.model`` in an NPA model; the buffers travel with ``state_dict`` and ``to``.  The rows of the
    codes lie a multiple of 16 bytes apart, as the kernel for both layers reads them, whatever gave them other memory."""

    def __init__(self, module):
        super().__init__()
        try:
            first, act, last = module
            fits = (isinstance(first, torch.nn.Linear) and isinstance(act, torch.nn.ReLU) and isinstance(last, torch.nn.Linear)
                    and first.bias is not None and last.bias is None and first.out_features == last.in_features)
        except (TypeError, ValueError):
            fits = False
        if not fits:
            raise ValueError("Int8MLP takes Sequential(Linear, ReLU, Linear(bias=False))")
        with torch.no_grad():
            for name, layer in (("w1", first), ("w2", last)):
                codes, scales = quantize_rows(layer.weight.float())
                self.register_buffer(name, codes)
                self.register_buffer(name + "_scales", scales)
            self.register_buffer("b1", first.bias.detach().float().clone())
        self.in_features, self.out_features = first.in_features, last.out_features

    def _lay_out(self):
        """A copy that is moved has dense rows (66 bytes apart, say), and so has an assigned one: back to multiples of 16."""
        for name in ("w1", "w2"):
            codes = getattr(self, name)
            if codes.stride(1) != 1 or codes.stride(0) % 16 or (codes.is_cuda and codes.data_ptr() % 16):
                wide = codes.new_zeros(codes.shape[0], -(-codes.shape[1] // 16) * 16)
                wide[:, : codes.shape[1]] = codes
                setattr(self, name, wide[:, : codes.shape[1]])

    def _apply(self, fn, recurse=True):
        super()._apply(fn, recurse)
        self._lay_out()
        return self

    def _load_from_state_dict(self, *args, **kwargs):
        super()._load_from_state_dict(*args, **kwargs)
        self._lay_out()

    def forward(self, z):
        return mlp_int8(z, self.w1, self.w1_scales, self.b1, self.w2, self.w2_scales)

    def extra_repr(self):
        return f"in_features={self.in_features}, hidden={self.b1.numel()}, out_features={self.out_features}"
