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


# ------------------------------------------------------------------------------------------------------------------ autocast
@pytest.mark.parametrize("to", [B, torch.float16])
@pytest.mark.parametrize("dtype,cols", [(F, 64), (F, 63), (B, 64), (B, 63)])
def test_under_autocast_the_operator_keeps_its_types(dtype, cols, to):
    p = inputs(70, cols, 128, 8, 3, dtype)

    def step():
        leaves = [p[k].clone().requires_grad_() for k in "xab"]
        y = call(p, *leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, p["dy"]))

    want = step()
    with torch.autocast("cuda", dtype=to):
        got = step()
        with torch.no_grad():
            plain = call(p)
    assert all(torch.equal(g, w) for g, w in zip(got, want)) and torch.equal(plain, want[0])


@pytest.mark.parametrize("to", [B, torch.float16])
@pytest.mark.parametrize("weights,x_type", [(F, F), (B, F), (F, B), (F, torch.float16)])
def test_an_adapter_linear_under_autocast(weights, x_type, to):
    """As the nn.Linear in its place: inputs and weights of any types, the result in autocast's.  Bound: operands rounded to the type (half a step each, two
    factors in the base and three in the adapters' part), the result rounded once, sums of 64 products in fp32."""
    torch.manual_seed(0)
    layer = A.AdapterLinear(nn.Linear(64, 128), 3, 8, scaling=0.75).to("cuda", weights)
    with torch.no_grad():
        layer.lora_b.normal_()
    x = torch.randn(60, 64, device="cuda").to(x_type).requires_grad_()
    ids = torch.arange(60, device="cuda") % 4 - 1
    with torch.autocast("cuda", dtype=to):
        assert layer(x).dtype == to                  # without ids
        with A.use_adapters(ids):
            y = layer(x)
    assert y.dtype == to
    y.sum().backward()
    assert x.grad.dtype == x_type and layer.lora_a.grad.dtype == weights
    xd, w, bias, a, b = (t.detach().double() for t in (x, layer.base.weight, layer.base.bias, layer.lora_a, layer.lora_b))
    own = (ids >= 0).double()[:, None] * 0.75
    ai, bi = a[ids.clamp(min=0)], b[ids.clamp(min=0)]
    part = lambda x, a, b: torch.einsum("tor,trk,tk->to", b, a, x)  # noqa: E731
    want = xd @ w.T + bias + own * part(xd, ai, bi)
    h = HALF[to]
    size = xd.abs() @ w.abs().T * ((1 + h) ** 2 - 1) + bias.abs() * h + own * part(xd.abs(), ai.abs(), bi.abs()) * ((1 + h) ** 3 - 1 + 2.0 ** -16)
    sums = 2 * 72 * 2.0 ** -24 * (xd.abs() @ w.abs().T + own * part(xd.abs(), ai.abs(), bi.abs()))
    off = size + sums
    assert ((y.double() - want).abs() <= off + (want.abs() + off) * h).all()


def test_a_model_with_adapters_under_autocast():
    """An fp32 model under bf16 autocast: each request as far from the fp32 model with its adapter merged in as that model itself gets under autocast."""
    import copy
    from transformers import DebertaV2Config
    from transformers.models.deberta_v2 import modeling_deberta_v2 as hf
    from tests import util
    from turbodeberta_b200 import model as M
    torch.manual_seed(1)
    cfg = DebertaV2Config(vocab_size=500, hidden_size=256, num_hidden_layers=2, num_attention_heads=4, intermediate_size=512, relative_attention=True,
                          position_buckets=256, max_relative_positions=512, pos_att_type=["p2c", "c2p"], norm_rel_ebd="layer_norm", type_vocab_size=0,
                          position_biased_input=False, share_att_key=True)
    plain = M.patch_model(hf.DebertaV2Model(cfg)).eval().cuda()
    model = copy.deepcopy(plain)
    layers = A.add_adapters(model, 2, 4, scaling=1.5)
    with torch.no_grad():
        for layer in layers.values():
            layer.lora_b.normal_(0, 0.1)
    ids = torch.randint(0, 500, (3, 80), device="cuda")
    mask = (torch.arange(80, device="cuda") < torch.tensor([[80], [33], [57]], device="cuda")).long()
    which = [1, -1, 0]
    with torch.no_grad():
        with torch.autocast("cuda", dtype=B), A.use_adapters(which):
            got = model(input_ids=ids, attention_mask=mask).last_hidden_state
        for i, k in enumerate(which):
            one = copy.deepcopy(plain)
            for name, layer in layers.items():
                if k >= 0:
                    one.get_submodule(name).weight += layer.scaling * (layer.lora_b[k] @ layer.lora_a[k])
            v = mask[i].bool()
            best = one(input_ids=ids, attention_mask=mask).last_hidden_state[i][v]
            with torch.autocast("cuda", dtype=B):
                merged = one(input_ids=ids, attention_mask=mask).last_hidden_state[i][v]
            assert (got[i][v].float() - best).norm() <= util.MODEL_BF16_VS_EAGER_FACTOR * (merged.float() - best).norm()


# --------------------------------------------------------------------------------------------------------------- infinities
@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("rows", [20, 100])
@pytest.mark.parametrize("rank", [1, 8, 16, 24])
def test_rows_with_infinities_have_the_formulas_infinities(rank, rows, dtype):
    """All factors and weights positive: a row with one infinity has infinite results, and no zero that pads a rank makes a NaN of them."""
    p = inputs(rows, 64, 128, rank, 2, dtype)
    for k in ("w", "a", "b"):
        p[k] = p[k].abs() + 0.01
    p["ids"] = torch.zeros(rows, dtype=torch.int32, device="cuda")
    p["x"][3, 5] = float("inf")
    p["dy"][7, 9] = float("inf")
    leaves = [p[k].clone().requires_grad_() for k in "xab"]
    y = call(p, *leaves)
    dx, = torch.autograd.grad(y, leaves[:1], p["dy"])
    others = torch.arange(rows, device="cuda")
    assert torch.isposinf(y[3]).all() and torch.isfinite(y[others != 3]).all()
    assert torch.isposinf(dx[7]).all() and torch.isfinite(dx[others != 7]).all()
