"""The HF model's modules around its matrix products, for training.

``patch_model(model, train_kernels=True)`` gives the stock modules these classes (parameters and names stay): LayerNorms and dropouts run the
kernels of ``ops.layer_norm`` and ``ops.dropout``, and the ends of both halves of a layer (``DebertaV2SelfOutput``, ``DebertaV2Output``: dropout,
residual, LayerNorm) run as one.  Passes of modules in eval mode that record no gradients, other types than float32 and bfloat16, autocast,
forward-mode derivatives, ``torch.func``'s transforms and the CPU run as before.  In training mode the kernels run without gradients too: a
checkpoint's first pass may be one without, and the pass that is made again for its gradients has to drop the same elements.  A second derivative
(``create_graph=True``) is refused.

The attention has no backward pass (neither has the reference's), so a training loop reaches what lies behind the last attention whose
inputs are frozen: task heads, and the last layer's projections, norms and adapters.
"""
from __future__ import annotations

import torch
from torch import nn
from torch.autograd import forward_ad
from transformers.models.deberta_v2.modeling_deberta_v2 import DebertaV2Output, DebertaV2SelfOutput

from .ops.dropout import dropout
from .ops.layer_norm import dropout_add_layer_norm, layer_norm

_TYPES = (torch.float32, torch.bfloat16)


def _applies(module: nn.Module, x: torch.Tensor) -> bool:
    return ((module.training or torch.is_grad_enabled()) and x.is_cuda and x.dtype in _TYPES and not torch.is_autocast_enabled()
            and forward_ad._current_level < 0 and torch._C._functorch.peek_interpreter_stack() is None)


def _norm_applies(norm: nn.LayerNorm, x: torch.Tensor) -> bool:
    w, b = norm.weight, norm.bias
    return (_applies(norm, x) and w is not None and b is not None and w.dim() == 1 and w.dtype == b.dtype and w.dtype in (x.dtype, torch.float32)
            and x.shape[-1] == w.numel() and w.numel() <= 16384)


def _fresh_seed(x: torch.Tensor) -> torch.Tensor:
    """From torch's generator of the device, so that ``torch.manual_seed``, checkpointed recomputation and captured graphs (each replay draws
    anew) mean what they mean for torch's own dropout."""
    return torch.empty((1,), dtype=torch.int64, device=x.device).random_()


def _stock(module: nn.Module, types) -> bool:
    """Whether one kernel may do what calling the module does: exactly one of ``types``, no subclass, with no ``forward`` of its own and no hooks."""
    return (type(module) in types and "forward" not in module.__dict__
            and not (module._forward_hooks or module._forward_pre_hooks or module._backward_hooks or module._backward_pre_hooks))


class FlashLayerNorm(nn.LayerNorm):
    def forward(self, x):
        if _norm_applies(self, x):
            return layer_norm(x, self.weight, self.bias, self.eps)
        return super().forward(x)


class FlashDropout(nn.Dropout):
    def forward(self, x):
        if self.training and self.p > 0 and not self.inplace and _applies(self, x):
            return dropout(x, self.p, _fresh_seed(x))
        return super().forward(x)


class _JoinedEnd:
    """``LayerNorm(dropout(dense(hidden_states)) + input_tensor)``"""

    def forward(self, hidden_states, input_tensor):
        x = self.dense(hidden_states)
        norm, drop = self.LayerNorm, self.dropout
        if (_stock(norm, NORMS) and _stock(drop, (*DROPOUTS, nn.Identity)) and not nn.modules.module._has_any_global_hook()
                and x.shape == input_tensor.shape and x.dtype == input_tensor.dtype and _norm_applies(norm, x)):
            p = drop.p if type(drop) in DROPOUTS and drop.training else 0.0
            return dropout_add_layer_norm(x, input_tensor, norm.weight, norm.bias, norm.eps, p, _fresh_seed(x) if p > 0 else None)
        return norm(drop(x) + input_tensor)


class FlashDebertaV2SelfOutput(_JoinedEnd, DebertaV2SelfOutput):
    pass


class FlashDebertaV2Output(_JoinedEnd, DebertaV2Output):
    pass


#: what stands for what; the native inference loop takes either
NORMS = (nn.LayerNorm, FlashLayerNorm)
DROPOUTS = (nn.Dropout, FlashDropout)
SELF_OUTPUTS = (DebertaV2SelfOutput, FlashDebertaV2SelfOutput)
OUTPUTS = (DebertaV2Output, FlashDebertaV2Output)
_PAIRS = dict((NORMS, DROPOUTS, SELF_OUTPUTS, OUTPUTS))


def use_train_kernels(model: nn.Module) -> nn.Module:
    """Swap, in place, the classes of the stock modules (subclasses of them stay as they are)."""
    for module in model.modules():
        new = _PAIRS.get(type(module))
        if new is not None:
            module.__class__ = new
    return model
