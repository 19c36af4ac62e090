"""LayerNorm over the last dimension, alone and as the end of a sublayer, with gradients of every input.

``layer_norm(x, weight, bias, eps)`` is ``(x - mean) / sqrt(var + eps) * weight + bias``; ``dropout_add_layer_norm(x, residual, ...)`` is
``layer_norm(dropout(x, p, seed, offset) + residual, ...)`` in one pass forward and one (and a short sum) backward: what
``DebertaV2SelfOutput`` and ``DebertaV2Output`` of the HF model end in.  Sums, means and deviations are taken in fp32 and the result is
rounded once; the backward pass makes the dropout mask and the sum again from ``x`` and ``residual``.  Gradients of the weights are added
up in a fixed order: two runs give the same bits.
Second derivatives and forward-mode tangents are refused.
"""
from __future__ import annotations

import torch

from .. import _cabi as cabi
from .dropout import signed64, split_seed


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, eps: float = 1e-7) -> torch.Tensor:
    """``x``: float32 or bfloat16, any strides, up to 16384 columns.  ``weight``, ``bias``: of ``x``'s dtype, or float32."""
    return cabi.host.norm(x, None, weight, bias, eps, 0.0, None, 0, 0)


def dropout_add_layer_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, eps: float = 1e-7,
                           p: float = 0.0, seed=None, offset: int = 0) -> torch.Tensor:
    """``layer_norm(dropout(x, p, seed, offset) + residual, weight, bias, eps)``; ``residual`` has the shape and dtype of ``x``.
    ``seed`` (see ``ops.dropout.dropout``) is needed where ``p`` is not zero."""
    if residual is None:
        raise ValueError("residual is missing: use layer_norm")
    if seed is None:
        if p != 0:
            raise ValueError("dropout needs a seed")
        seed = 0
    tensor, value = split_seed(seed)
    return cabi.host.norm(x, residual, weight, bias, eps, p, tensor, value, signed64(offset, "offset"))
