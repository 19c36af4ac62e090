"""Many fine-tunings of one encoder at once: low-rank adapters beside its projections, chosen per request.

::

    model = patch_model(DebertaV2Model(config)).cuda().bfloat16().eval()
    layers = add_adapters(model, count=8, rank=16, scaling=2.0)        # {name of the projection: AdapterLinear}
    load_adapter(model, 3, {name: (A, B), ...})                        # one customer's fine-tuning
    with torch.inference_mode(), use_adapters([3, 3, -1, 5]):          # of the batch's sequences; -1: the plain model
        out = model(input_ids, attention_mask)

One batch mixes requests of any adapters (``ops.lora.lora_linear``), on the padded and the packed route alike.  The reference has nothing of
this kind; there every fine-tuning is a model of its own.

The ids are those of the thread and of the block, and neither need be the same when a checkpointed pass is made again: that happens within the backward
pass, in autograd's own thread.  ``checkpoint(keep_adapters(part), x, ...)``, or ``checkpoint(part, x, use_reentrant=False,
context_fn=recompute_contexts)``, gives the pass its ids again; without either it raises.
"""
from __future__ import annotations

import contextlib
import threading

import torch
from torch import nn

from .ops.lora import lora_linear

#: projections that take adapters where nothing else is said (by the ends of their names)
DEFAULT_TARGETS = ("self.value_proj", "attention.output.dense", "intermediate.dense", "output.dense")


class _Active(threading.local):
    ids = None                  # of the batch's sequences
    rows = None                 # of the packed stream's tokens
    task = -1                   # the backward pass within which both were chosen; -1: none
    before = None               # what was in use outside of the present block


_ACTIVE = _Active()
_backward_pass = torch._C._current_graph_task_id             # that this thread is running; -1: none


class _active:
    """A block in which ``ids`` and ``rows`` are in use; may be entered again, by several threads at once too (a checkpoint's pass is made again as often as
    its gradients are asked for)."""
    __slots__ = ("ids", "rows")

    def __init__(self, ids, rows):
        self.ids, self.rows = ids, rows

    def __enter__(self):
        _ACTIVE.before = (_ACTIVE.ids, _ACTIVE.rows, _ACTIVE.task, _ACTIVE.before)
        _ACTIVE.ids, _ACTIVE.rows, _ACTIVE.task = self.ids, self.rows, _backward_pass()

    def __exit__(self, *error):
        _ACTIVE.ids, _ACTIVE.rows, _ACTIVE.task, _ACTIVE.before = _ACTIVE.before


class AdapterLinear(nn.Module):
    """A frozen ``nn.Linear`` with ``count`` adapters of up to ``rank``: ``lora_a [count, rank, in]`` (small random numbers) and ``lora_b [count, out,
    rank]`` (zeros, so that a fresh adapter changes nothing).  Outside ``use_adapters`` it is the Linear alone."""

    _used = False               # with ids, ever

    def __init__(self, base: nn.Linear, count: int, rank: int, scaling: float = 1.0):
        super().__init__()
        if count < 1 or rank < 1:
            raise ValueError("count and rank must be positive")
        self.base = base.requires_grad_(False)
        self.in_features, self.out_features = base.in_features, base.out_features
        self.count, self.rank, self.scaling = count, rank, float(scaling)
        like = dict(dtype=base.weight.dtype, device=base.weight.device)
        self.lora_a = nn.Parameter(torch.randn(count, rank, base.in_features, **like) * base.in_features ** -0.5)
        self.lora_b = nn.Parameter(torch.zeros(count, base.out_features, rank, **like))

    def forward(self, x):
        ids = _ACTIVE.ids if _ACTIVE.rows is None else _ACTIVE.rows
        if self._used and _ACTIVE.task != _backward_pass():  # made again by a checkpoint: what is in use here, if anything, need not be the first pass's
            raise RuntimeError("a checkpointed pass is being made again and does not know its adapter ids: checkpoint keep_adapters(function), or give "
                               "checkpoint context_fn=recompute_contexts")
        if ids is None:
            return self.base(x)
        self._used = True
        if ids.device != x.device:
            ids = ids.to(x.device)
        inputs = [x, self.base.weight, self.base.bias, self.lora_a, self.lora_b]
        if not torch.is_autocast_enabled(x.device.type):
            return lora_linear(*inputs, self.scaling, ids)
        # as an nn.Linear: operands of any type but fp64, the result in autocast's.  The kernels have no fp16: its operands are computed in fp32.
        to = torch.get_autocast_dtype(x.device.type)
        inputs = [t if t is None or t.dtype == torch.float64 else t.to(to).to(torch.bfloat16 if to == torch.bfloat16 else torch.float32) for t in inputs]
        return lora_linear(*inputs, self.scaling, ids).to(to)

    def extra_repr(self):
        return f"count={self.count}, rank={self.rank}, scaling={self.scaling}"


def add_adapters(model: nn.Module, count: int, rank: int, scaling: float = 1.0, targets=DEFAULT_TARGETS) -> dict:
    """Put an ``AdapterLinear`` in the place of every ``nn.Linear`` whose name is, or ends in a dot and, one of ``targets``; the model's own parameters
    there are frozen.  Returns them by name.  Query and key projections whose weights also make the relative-position tables
    (``share_att_key``) are refused: the tables are the batch's, not a request's."""
    if any(isinstance(m, AdapterLinear) for m in model.modules()):
        raise ValueError("the model has adapters already")
    found = {}
    for name, module in list(model.named_modules()):
        if type(module) is not nn.Linear or not any(name == t or name.endswith("." + t) for t in targets):
            continue
        parent, _, child = name.rpartition(".")
        owner = model.get_submodule(parent)
        if child in ("query_proj", "key_proj") and getattr(owner, "share_att_key", False) and getattr(owner, "relative_attention", False):
            raise ValueError(f"{name} also makes the relative-position tables (share_att_key) and takes no adapters")
        if child in ("pos_key_proj", "pos_query_proj"):
            raise ValueError(f"{name} makes the relative-position tables and takes no adapters")
        found[name] = (owner, child, module)
    if not found:
        raise ValueError(f"no Linear of the model is named like {tuple(targets)}")
    out = {}
    for name, (owner, child, module) in found.items():
        out[name] = AdapterLinear(module, count, rank, scaling).train(module.training)
        setattr(owner, child, out[name])
    return out


@torch.no_grad()
def load_adapter(model: nn.Module, index: int, weights: dict, scaling: float | None = None) -> None:
    """Write adapter ``index``: ``weights`` maps names of projections to ``(A [rank, in], B [out, rank])``, of any rank up to the model's; projections that
    are not named get none.  ``scaling``: the adapter's own, where it is not the model's."""
    layers = {n: m for n, m in model.named_modules() if isinstance(m, AdapterLinear)}
    unknown = set(weights) - set(layers)
    if unknown:
        raise ValueError(f"no adapters at {sorted(unknown)}")
    for name, layer in layers.items():
        if not 0 <= index < layer.count:
            raise ValueError(f"adapter {index}: the model has {layer.count}")
        if name in weights:
            a, b = weights[name]
            if a.dim() != 2 or b.dim() != 2 or a.shape[0] != b.shape[1] or a.shape[0] > layer.rank or a.shape[1] != layer.in_features or b.shape[0] != layer.out_features:
                raise ValueError(f"{name}: A {tuple(a.shape)} and B {tuple(b.shape)} do not fit [rank, {layer.in_features}] and [{layer.out_features}, rank], "
                                 f"rank up to {layer.rank}")
    for name, layer in layers.items():
        layer.lora_a[index].zero_()
        layer.lora_b[index].zero_()
        if name in weights:
            a, b = weights[name]
            factor = 1.0 if scaling is None else scaling / layer.scaling
            layer.lora_a[index, :a.shape[0]].copy_(a)
            layer.lora_b[index, :, :a.shape[0]].copy_(b.float() * factor if factor != 1.0 else b)


@contextlib.contextmanager
def use_adapters(ids):
    """Within it, this thread's passes use adapter ``ids[i]`` for the batch's sequence ``i``; a negative id is the plain model's.  ``ids``: numbers, or an
    integer tensor (on the device, so that nothing is copied per pass; its values are not checked, and one that is no adapter's means none)."""
    if not isinstance(ids, torch.Tensor):
        ids = torch.tensor([int(i) for i in ids], dtype=torch.int32)
    if ids.dim() != 1 or ids.dtype not in (torch.int32, torch.int64):
        raise ValueError("ids must be one integer for each sequence of the batch")
    if not ids.is_cuda and torch.cuda.is_available():
        ids = ids.cuda()
    with _active(ids, None):
        yield


def keep_adapters(function):
    """``function``, called with the adapter ids (or none) that are in use now, whichever thread calls it and whenever: what a checkpoint is to be given."""
    ids, rows = _ACTIVE.ids, _ACTIVE.rows

    def kept(*args, **kwargs):
        with _active(ids, rows):
            return function(*args, **kwargs)

    return kept


def recompute_contexts():
    """The ``context_fn`` of a checkpoint without ``use_reentrant``: the pass that is made again has the ids of the first.  In a Hugging Face model:
    ``model.gradient_checkpointing_enable({"use_reentrant": False, "context_fn": recompute_contexts})``."""
    return contextlib.nullcontext(), _active(_ACTIVE.ids, _ACTIVE.rows)


@contextlib.contextmanager
def packed_rows(indices: torch.Tensor, batch: int, length: int):
    """Within it, the layers see the packed stream whose tokens lie at ``indices`` of the padded ``[batch, length]``."""
    ids, before = _ACTIVE.ids, _ACTIVE.rows
    if ids is not None:
        if ids.numel() != batch:
            raise ValueError(f"adapter ids of {ids.numel()} sequences, but the batch has {batch}")
        _ACTIVE.rows = ids.to(indices.device)[torch.div(indices, length, rounding_mode="floor")][None]
    try:
        yield
    finally:
        _ACTIVE.rows = before
