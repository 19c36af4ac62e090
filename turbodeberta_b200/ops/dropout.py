"""Dropout from a counter-based generator: ``y = x / (1 - p)`` where an element stays, zero where it is dropped.

The mask is a function of ``(seed, offset, index of the element)`` alone and is made anew in the backward pass, so nothing of it is
kept between the two.  Elements are counted in row-major order; eight of them share the Philox4x32-10 block (Salmon, Moraes, Dror and
Shaw, 2011) with counter ``(index // 8, offset)`` and key ``seed``, whose words are taken as eight 16-bit numbers, low half first; an
element stays when its number is at least ``round(65536 * p)``.  A probability is therefore a multiple of 2**-16, and the scale is that of
the rounded one.  The reference has no dropout of its own (HF's ``nn.Dropout`` modules run around its kernels, ``model.py:112``).
"""
from __future__ import annotations

import torch

from .. import _cabi as cabi


def split_seed(seed) -> tuple:
    """(tensor or None, number): a seed as the native calls take it."""
    if isinstance(seed, torch.Tensor):
        return seed, 0
    return None, signed64(seed, "seed")


def signed64(value, name: str) -> int:
    """The 64 bits of a whole number, as a signed one."""
    value = int(value)
    if not -(1 << 63) <= value < 1 << 64:
        raise ValueError(f"{name} does not fit 64 bits")
    return value - (1 << 64) if value >= 1 << 63 else value


def dropout(x: torch.Tensor, p: float, seed, offset: int = 0) -> torch.Tensor:
    """Drop elements of ``x`` (float32 or bfloat16, any shape and strides) with probability ``p``; differentiable in ``x`` (once, and
    backward: a second derivative and forward-mode tangents are refused).

    ``seed`` is a number, or an int64 CUDA tensor of one element that the kernels read: in a CUDA graph a number is recorded with the
    launch, so every replay drops the same elements, while a tensor may be given new values between replays (a forward pass and its
    backward pass have to see the same one).  ``offset`` tells calls with one seed apart: layers of a pass, or steps.

    A dropped element and its gradient are zero whatever ``x`` holds there, NaN included."""
    tensor, value = split_seed(seed)
    return cabi.host.dropout(x, p, tensor, value, signed64(offset, "offset"))
