"""What callers do with the projection with adapters: change its result in place, call it under autocast, give it rows that hold infinities."""
import pytest
import torch
from torch import nn

from turbodeberta_b200 import adapters as A
from turbodeberta_b200.ops.lora import lora_linear

pytestmark = pytest.mark.gpu
F, B = torch.float32, torch.bfloat16
HALF = {F: 2.0 ** -24, B: 2.0 ** -8, torch.float16: 2.0 ** -11}


def inputs(rows, cols, features, rank, n, dtype, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    r = lambda *s, k=1.0: (torch.randn(*s, device="cuda", generator=g) * k).to(dtype)  # noqa: E731
    ids = torch.randint(-1, n, (rows,), device="cuda", generator=g, dtype=torch.int32)
    return dict(x=r(rows, cols), w=r(features, cols, k=cols ** -0.5), bias=r(features), a=r(n, rank, cols, k=cols ** -0.5), b=r(n, features, rank), ids=ids,
                dy=r(rows, features))


def call(p, x=None, a=None, b=None):
    return lora_linear(p["x"] if x is None else x, p["w"], p["bias"], p["a"] if a is None else a, p["b"] if b is None else b, 0.75, p["ids"])


# 20 rows: the few-token kernel in bf16; 100 the tile kernel; columns of 63: CUDA cores beside the library's product in either type
@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("rows,cols,lead", [(20, 64, None), (100, 64, None), (100, 64, (4, 25)), (100, 63, None), (100, 63, (4, 25)), (1, 64, ())])
def test_the_result_may_be_changed_in_place(rows, cols, lead, dtype):
    p = inputs(rows, cols, 128, 8, 3, dtype)
    shape = (rows,) if lead is None else lead
    p["x"], p["dy"], p["ids"] = p["x"].view(*shape, cols), p["dy"].view(*shape, 128), p["ids"].view(shape)
    res = torch.randn_like(p["dy"])
    grads = []
    for change in (lambda y: y + res, lambda y: y.add_(res), lambda y: nn.functional.relu(y), lambda y: nn.functional.relu(y, inplace=True)):
        leaves = [p[k].clone().requires_grad_() for k in "xab"]
        y = change(call(p, *leaves))
        assert y.shape == p["dy"].shape
        grads.append((y.detach(), *torch.autograd.grad(y, leaves, p["dy"])))
    for one, two in (grads[:2], grads[2:]):
        assert all(torch.equal(s, t) for s, t in zip(one, two))


def test_rows_of_the_result_may_be_masked_in_place():
    p = inputs(100, 64, 128, 8, 3, B)
    out = []
    for change in (lambda y, m: y.masked_fill(m[:, None], 0), lambda y, m: y.masked_fill_(m[:, None], 0)):
        leaves = [p[k].clone().requires_grad_() for k in "xab"]
        out.append(torch.autograd.grad(change(call(p, *leaves), p["ids"] == 1), leaves, p["dy"]))
    assert all(torch.equal(s, t) for s, t in zip(*out))
