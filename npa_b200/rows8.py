"""Activations in 8 bits, for what a backward pass has to keep.

Groups of 32 columns of a row share a power of two, one byte, so that an activation takes 1 + 1/32 bytes instead of 4 and
comes back within half a unit: ``|restored - x| <= max |group| / 127`` at most, and ``max |group| / 254`` at the group's best.

    kept = compress_rows(x)      # codes, exponents
    x8 = kept.restore()          # values, in the type of x

``mlp.apply_mlp(module, z, checkpoint=True)`` keeps the input of the adaptation MLP this way between forward and backward.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _native as N

GROUP = 32  # columns that share an exponent


@dataclass(frozen=True)
class Rows8:
    """8-bit rows: ``codes`` ``[..., k]`` int8, ``exponents`` ``[..., ceil(k / 32)]`` uint8; the value of a code is
    ``code * 2 ** (exponent - 133)``, and NaN where the exponent is 255.  ``dtype`` is the type that was compressed."""

    codes: torch.Tensor
    exponents: torch.Tensor
    dtype: torch.dtype

    def restore(self, dtype=None):
        """The values, contiguous, in ``dtype`` (that of the compressed tensor)."""
        return N.ops.restore_rows(self.codes, self.exponents, self.dtype if dtype is None else dtype)

    @property
    def nbytes(self) -> int:
        """Bytes held, padding of the rows to 16 bytes included."""
        return self.codes.untyped_storage().nbytes() + self.exponents.untyped_storage().nbytes()


def compress_rows(x) -> Rows8:
    """``x`` ``[..., k]`` (float32, float16 or bfloat16, any strides) in 8 bits.

    The exponent of a group is the smallest in whose units its largest magnitude rounds to at most 127; codes are rounded
    to nearest, ties to even.  A group with an infinity or a NaN comes back as NaN.  The call carries no gradient and is
    refused on tensors that require one while gradients are recorded."""
    return Rows8(*N.ops.compress_rows(x), x.dtype)
