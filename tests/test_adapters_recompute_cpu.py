"""Adapters under checkpointing: a recomputed pass has the ids of the pass that it repeats, or says that it does not know them.  The operator is
replaced by its formula, so no GPU is needed; a recomputed pass then runs in the thread of the backward call, and a thread of its own is tried too."""
import threading

import pytest
import torch
from torch import nn
from torch.utils.checkpoint import checkpoint

from turbodeberta_b200 import adapters as A


@pytest.fixture(autouse=True)
def formula(monkeypatch):
    def lora_linear(x, weight, bias, a, b, scaling, ids):
        ids = ids.reshape(x.shape[:-1]) if ids.numel() * x.shape[-1] == x.numel() else ids[:, None].expand(x.shape[:-1])
        keep = (ids >= 0).to(x.dtype)[..., None]
        a, b = a[ids.clamp(min=0)], b[ids.clamp(min=0)]
        return nn.functional.linear(x, weight, bias) + keep * scaling * torch.einsum("...or,...rk,...k->...o", b, a, x)

    monkeypatch.setattr(A, "lora_linear", lora_linear)


class Block(nn.Module):
    def __init__(self):
        super().__init__()
        torch.manual_seed(0)
        self.one, self.two = nn.Linear(6, 5), nn.Linear(5, 4)

    def forward(self, x):
        return self.two(torch.tanh(self.one(x)))


def _model():
    model = nn.Sequential(Block(), nn.Linear(4, 3))
    A.add_adapters(model, 3, 2, targets=("one", "two"))
    with torch.no_grad():
        for m in model.modules():
            if isinstance(m, A.AdapterLinear):
                m.lora_b.normal_()
    return model


def _x():
    return torch.randn(4, 2, 6, generator=torch.Generator().manual_seed(1)).requires_grad_()


def _grads(model, x, y, thread=False):
    model.zero_grad()
    errors = []

    def backward():
        try:
            model[1](y).square().sum().backward()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    if thread:
        t = threading.Thread(target=backward)
        t.start()
        t.join()
    else:
        backward()
    if errors:
        raise errors[0]
    return [x.grad] + [p.grad for p in model.parameters() if p.requires_grad]


def _ways():
    return {"reentrant": lambda block, x: checkpoint(A.keep_adapters(block), x, use_reentrant=True),
            "other": lambda block, x: checkpoint(A.keep_adapters(block), x, use_reentrant=False),
            "contexts": lambda block, x: checkpoint(block, x, use_reentrant=False, context_fn=A.recompute_contexts)}


@pytest.mark.parametrize("thread", [False, True])
@pytest.mark.parametrize("where", ["inside", "outside", "inside another"])
@pytest.mark.parametrize("way", list(_ways()))
def test_a_recomputed_pass_has_the_ids_of_the_first(way, where, thread):
    model = _model()
    ids = [2, -1, 0, 2]
    x = _x()
    with A.use_adapters(ids):
        want = _grads(model, x, model[0](x))
    assert all(g is not None and g.abs().sum() > 0 for g in want)
    x = _x()
    with A.use_adapters(ids):
        y = _ways()[way](model[0], x)
        if where == "inside":
            got = _grads(model, x, y, thread)
    if where == "outside":
        got = _grads(model, x, y, thread)
    elif where == "inside another":
        with A.use_adapters([1, 1, 1, 1]):
            got = _grads(model, x, y, thread)
    assert all(torch.equal(g, w) for g, w in zip(got, want))


@pytest.mark.parametrize("trains", [True, False])
@pytest.mark.parametrize("where", ["inside", "outside", "inside another"])
def test_a_recomputed_pass_that_does_not_know_its_ids_says_so(where, trains):
    """Reentrant: nothing else would tell."""
    model = _model()
    if not trains:
        for m in model.modules():
            if isinstance(m, A.AdapterLinear):
                m.requires_grad_(False)
    x = _x()
    with A.use_adapters([2, -1, 0, 2]):
        y = checkpoint(model[0], x, use_reentrant=True)
        if where == "inside":
            with pytest.raises(RuntimeError, match="keep_adapters"):
                _grads(model, x, y)
    if where == "outside":
        with pytest.raises(RuntimeError, match="keep_adapters"):
            _grads(model, x, y)
    elif where == "inside another":
        with A.use_adapters([1, 1, 1, 1]), pytest.raises(RuntimeError, match="keep_adapters"):
            _grads(model, x, y)


@pytest.mark.parametrize("reentrant", [True, False])
def test_a_model_that_never_used_its_adapters_recomputes_the_plain_pass(reentrant):
    model = _model()
    x = _x()
    want = _grads(model, x, model[0](x))[0]
    x = _x()
    assert torch.equal(_grads(model, x, checkpoint(model[0], x, use_reentrant=reentrant))[0], want)


@pytest.mark.parametrize("way", list(_ways()))
def test_a_plain_pass_stays_plain(way):
    """Kept: no ids at all, whatever is in use when the pass is made again."""
    model = _model()
    x = _x()
    want = _grads(model, x, model[0](x))[0]
    with A.use_adapters([0] * 4):
        model[0](x)
    x = _x()
    y = _ways()[way](model[0], x)
    with A.use_adapters([1] * 4):
        assert torch.equal(_grads(model, x, y)[0], want)


def test_ids_chosen_within_the_recomputed_function_hold():
    model = _model()
    ids = [1, 0, -1, 2]

    def run(x):
        with A.use_adapters(ids):
            return model[0](x)

    x = _x()
    want = _grads(model, x, run(x))
    for reentrant in (True, False):
        x = _x()
        got = _grads(model, x, checkpoint(run, x, use_reentrant=reentrant))
        assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_packed_rows_are_kept():
    model = _model()
    at = torch.tensor([0, 1, 4, 5, 7])
    x = torch.randn(1, 5, 6, generator=torch.Generator().manual_seed(2)).requires_grad_()

    def passed(run):
        with A.use_adapters([2, 0]), A.packed_rows(at, 2, 4):
            return run(x)

    want = _grads(model, x, passed(model[0]))
    want = [g.clone() for g in want]
    x.grad = None
    for way in _ways().values():
        got = _grads(model, x, passed(lambda t: way(model[0], t)))
        assert all(torch.equal(g, w) for g, w in zip(got, want))
        x.grad = None


def test_kept_functions_leave_what_is_in_use_as_it_was():
    kept = A.keep_adapters(lambda: A._ACTIVE.ids)
    with A.use_adapters([1]):
        inside = A.keep_adapters(lambda: A._ACTIVE.ids.tolist())
        assert kept() is None and A._ACTIVE.ids.tolist() == [1]
    assert inside() == [1] and A._ACTIVE.ids is None
    with pytest.raises(ZeroDivisionError):
        A.keep_adapters(lambda: 1 / 0)()
    assert A._ACTIVE.ids is None


@pytest.mark.parametrize("way", list(_ways()))
def test_gradients_may_be_asked_for_more_than_once(way):
    model = _model()
    x = _x()
    params = [x] + [p for p in model[0].parameters() if p.requires_grad]
    with A.use_adapters([2, -1, 0, 2]):
        want = torch.autograd.grad(model[0](x).square().sum(), params)
        loss = _ways()[way](model[0], x).square().sum()
    if way == "reentrant":                           # such a checkpoint knows backward() alone
        for turn in (1, 2):
            loss.backward(retain_graph=True)
            assert all(torch.allclose(p.grad, turn * w) for p, w in zip(params, want))
    else:
        for _ in range(3):
            assert all(torch.equal(g, w) for g, w in zip(torch.autograd.grad(loss, params, retain_graph=True), want))
    assert A._ACTIVE.ids is None and A._ACTIVE.before is None
