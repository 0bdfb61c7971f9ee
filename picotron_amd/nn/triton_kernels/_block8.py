"""Activations held in 8 bits, in PyTorch: what the kernels of ``csrc/block8.hpp`` hold, to the bit in blocks of finite elements.

A block of 128 elements shares ``step = top / 127``, top its largest magnitude; an element's code is ``128 + round(x * (127 / top))``
and its value ``(code - 128) * step``, all in fp32.  A block whose top is below 2^-100 is held as zeros; one with an infinity or a
NaN comes back as NaN.
"""

from __future__ import annotations

import math

import torch
from torch import Tensor
from torch.nn import functional as F

from picotron_amd.ops import BLOCK8

_MOST_STEP = float.fromhex("0x1.020406p+121")  # the largest whose 127th multiple is finite in fp32

NO_SECOND_DERIVATIVE = (
    "the backward of an operator that keeps its inputs in 8 bits has no derivative of its own (create_graph=True); "
    "use it without checkpoint_8bit"
)


def encode(x: Tensor) -> tuple[Tensor, Tensor]:
    """(codes, steps) of the blocks along the last dimension, the last of them filled up with zeros: uint8 (..., blocks, 128)
    and fp32 (..., blocks, 1)."""

    x = F.pad(x.float(), (0, -x.size(-1) % BLOCK8)).unflatten(-1, (-1, BLOCK8))
    top = x.abs().amax(-1, keepdim=True)
    most = torch.full_like(top, 127.0)  # a tensor: by a number, torch multiplies with a rounded reciprocal on the GPU
    finite = top.isfinite()
    held = finite & (top >= 2.0**-100)
    steps = torch.where(held, (top / most).clamp_max(_MOST_STEP), torch.where(finite, 0.0, math.nan))
    codes = torch.where(held, (x * (most / top)).round(), 0.0)
    return (codes + 128).to(torch.uint8), steps


def decode(codes: Tensor, steps: Tensor, size: int) -> Tensor:
    """The ``size`` values of the last dimension that :func:`encode` took, fp32."""

    return ((codes.float() - 128) * steps).flatten(-2)[..., :size]
