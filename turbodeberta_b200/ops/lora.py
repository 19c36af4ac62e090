"""A shared projection with low-rank adapters of many requests at once.

``y[t] = x[t] W^T + b + s_a (x[t] A_a^T) B_a^T`` with ``a`` the adapter of row ``t``: one model's projection serves fine-tunings of many
owners in one batch, each row with its own.  Rows may come in any order and an adapter may appear in any number of places.  Differentiable
in ``x``, ``lora_a`` and ``lora_b`` (once, and backward: a second derivative and forward-mode tangents are refused); the shared projection is frozen.
"""
from __future__ import annotations

import torch

from .. import _cabi as cabi


def lora_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, lora_a: torch.Tensor, lora_b: torch.Tensor,
                scaling=1.0, adapter_ids: torch.Tensor | None = None) -> torch.Tensor:
    """``x [..., in]``, ``weight [out, in]``, ``bias [out]`` or None, ``lora_a [adapters, rank, in]``, ``lora_b [adapters, out, rank]``, all
    float32 or all bfloat16; rank up to 256.

    ``scaling``: a number, or a float32 vector with one entry per adapter.  ``adapter_ids`` (int32 or int64): the adapter of every row, in the
    shape of ``x`` without its last dimension, or one for each entry of ``x``'s first dimension (the sequences of a padded batch); it may be
    left out when there is one adapter.  A row whose id is not that of an adapter (-1, say) gets the shared projection alone.  The ids are not
    checked on the host: that would wait for the device.

    What an adapter holds, NaN and infinities included, reaches its own rows only, and so do the gradients.  Where a row of ``x`` or of the result's
    gradient holds infinities, the gradients of its adapter's factors may be NaN where the formula has infinities.

    The bf16 kernels report a device-side wait that gave up through status words that ``check_pending_status()`` (``ops.flash_attention``)
    reads; the call itself does not wait for the device."""
    if isinstance(scaling, torch.Tensor):
        return cabi.host.lora_linear(x, weight, bias, lora_a, lora_b, scaling, 1.0, adapter_ids)
    return cabi.host.lora_linear(x, weight, bias, lora_a, lora_b, None, float(scaling), adapter_ids)
