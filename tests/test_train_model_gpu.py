"""The training path's operators and adapters at work in the model.

Tolerance of fp32 models: util.MODEL_FP32_REL_TOL of the largest value (see there): the two sides run the same matrix products, sums in other orders.
"""
import copy

import pytest
import torch
from torch import nn
from transformers import DebertaV2Config
from transformers.models.deberta_v2 import modeling_deberta_v2 as hf

from tests import util
from turbodeberta_b200 import adapters as A
from turbodeberta_b200 import model as M
from turbodeberta_b200.ops.layer_norm import dropout_add_layer_norm
from turbodeberta_b200.ops.lora import lora_linear

pytestmark = pytest.mark.gpu
TOL = util.MODEL_FP32_REL_TOL


def _cfg(**more):
    return DebertaV2Config(**{**dict(vocab_size=500, hidden_size=128, num_hidden_layers=2, num_attention_heads=2, intermediate_size=256, relative_attention=True,
                                     position_buckets=256, max_relative_positions=512, pos_att_type=["p2c", "c2p"], norm_rel_ebd="layer_norm",
                                     type_vocab_size=0, position_biased_input=False, share_att_key=True), **more})


def close(got, want, what):
    got, want = got.double(), want.double()
    assert torch.isfinite(got).all() and (got - want).abs().max() <= TOL * want.abs().max(), (what, (got - want).abs().max().item(), want.abs().max().item())


def _batch(device="cuda"):
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(0, 500, (4, 90), generator=g)
    mask = torch.zeros(4, 90, dtype=torch.long)
    for b, n in enumerate([90, 1, 37, 64]):
        mask[b, :n] = 1
    return ids.to(device), mask.to(device)


def _freeze_below_the_last_attention(model):
    """The attention has no backward pass: train the last layer's output halves and the head."""
    model.requires_grad_(False)
    last = model.deberta.encoder.layer[-1]
    for part in (last.attention.output, last.intermediate, last.output, *(m for n, m in model.named_children() if n != "deberta")):
        part.requires_grad_(True)
    model.deberta.embeddings.requires_grad_(False)   # a masked-LM head shares its matrix with them
    return model


def _step(model, ids, mask, labels):
    model.zero_grad()
    loss = model(input_ids=ids, attention_mask=mask, labels=labels).loss
    loss.backward()
    return loss.detach(), {n: p.grad.clone() for n, p in model.named_parameters() if p.grad is not None}


@pytest.mark.parametrize("head", [M.FlashDebertaV2ForSequenceClassification, M.FlashDebertaV2ForTokenClassification, M.FlashDebertaV2ForMaskedLM])
def test_a_step_without_dropout_gives_the_stock_modules_gradients(head):
    torch.manual_seed(0)
    stock = head(_cfg(hidden_dropout_prob=0.0, attention_probs_dropout_prob=0.0, pooler_dropout=0.0)).cuda()
    with torch.no_grad():
        for p in stock.parameters():
            p.add_(torch.randn_like(p) * 0.02)       # norms that are not all ones
    own = M.patch_model(copy.deepcopy(stock), train_kernels=True)
    ids, mask = _batch()
    labels = torch.tensor([0, 1, 1, 0], device="cuda") if "Sequence" in head.__name__ else torch.where(mask.bool(), ids % 2, -100)
    results = [_step(_freeze_below_the_last_attention(m).train(), ids, mask, labels) for m in (stock, own)]
    close(results[1][0], results[0][0], "loss")
    assert results[0][1].keys() == results[1][1].keys() and len(results[0][1]) > 8
    for n in results[0][1]:
        close(results[1][1][n], results[0][1][n], n)


def test_steps_with_dropout_follow_torchs_seed():
    torch.manual_seed(0)
    model = M.patch_model(M.FlashDebertaV2ForSequenceClassification(_cfg(hidden_dropout_prob=0.2)), train_kernels=True).cuda()
    _freeze_below_the_last_attention(model).train()
    ids, mask = _batch()
    labels = torch.tensor([0, 1, 1, 0], device="cuda")
    runs = []
    for seed in (7, 7, 8):
        torch.manual_seed(seed)
        runs.append(_step(model, ids, mask, labels))
    assert torch.equal(runs[0][0], runs[1][0]) and not torch.equal(runs[0][0], runs[2][0])
    for n, g in runs[0][1].items():
        assert torch.equal(g, runs[1][1][n]), n
    model.eval()
    with torch.no_grad():                            # inference is what it was
        plain = copy.deepcopy(model)
        for m in plain.modules():
            for swapped, stock in ((type(model.deberta.encoder.layer[0].output), hf.DebertaV2Output),):
                if type(m) is swapped:
                    m.__class__ = stock
        assert torch.equal(model(input_ids=ids, attention_mask=mask).logits, plain(input_ids=ids, attention_mask=mask).logits)


def test_a_checkpointed_sublayer_end_makes_its_mask_again():
    from torch.utils.checkpoint import checkpoint
    torch.manual_seed(0)
    end = M.patch_model(hf.DebertaV2Model(_cfg(hidden_dropout_prob=0.3)), train_kernels=True).encoder.layer[0].output.cuda().train()
    h, x = torch.randn(50, 256, device="cuda"), torch.randn(50, 128, device="cuda", requires_grad=True)
    out = []
    for run in (lambda: end(h, x), lambda: checkpoint(end, h, x, use_reentrant=False)):
        torch.manual_seed(4)
        y = run()
        out.append((y.detach(), *torch.autograd.grad(y.square().sum(), [x, *end.parameters()])))
    assert all(torch.equal(a, b) for a, b in zip(*out))


def test_hooks_on_the_inner_modules_still_run():
    end = M.patch_model(hf.DebertaV2Model(_cfg()), train_kernels=True).encoder.layer[0].output.cuda().train()
    seen = []
    end.LayerNorm.register_forward_hook(lambda *a: seen.append(1))
    end(torch.randn(5, 256, device="cuda"), torch.randn(5, 128, device="cuda", requires_grad=True))
    assert seen


# ------------------------------------------------------------------------------------------------------------------ adapters
def _with_adapters(dtype=torch.float32, count=3, rank=4, **cfg):
    torch.manual_seed(1)
    plain = M.patch_model(hf.DebertaV2Model(_cfg(**cfg))).eval().to("cuda", dtype)
    model = copy.deepcopy(plain)
    layers = A.add_adapters(model, count, rank, scaling=1.5)
    with torch.no_grad():
        for layer in layers.values():
            layer.lora_b.normal_(0, 0.1)
    return plain, model, layers


def _merged(plain, layers, index):
    """The model whose weights have the adapter in them."""
    out = copy.deepcopy(plain)
    with torch.no_grad():
        for name, layer in layers.items():
            out.get_submodule(name).weight += layer.scaling * (layer.lora_b[index].double() @ layer.lora_a[index].double()).to(layer.lora_b.dtype)
    return out


@pytest.mark.parametrize("route", ["packed", "padded", "full"])
def test_a_batch_of_adapters_is_each_request_with_its_own_model(route):
    plain, model, layers = _with_adapters()
    ids, mask = _batch()
    if route == "full":
        mask = torch.ones_like(mask)
    model.encoder.pack_padded_batches = plain.encoder.pack_padded_batches = route != "padded"
    which = [2, -1, 0, 2]
    with torch.no_grad():
        with A.use_adapters(which):
            got = model(input_ids=ids, attention_mask=mask).last_hidden_state
        assert torch.equal(model(input_ids=ids[:1], attention_mask=mask[:1]).last_hidden_state,
                           model(input_ids=ids[:1], attention_mask=mask[:1]).last_hidden_state)
        for i, a in enumerate(which):
            one = plain if a < 0 else _merged(plain, layers, a)
            want = one(input_ids=ids, attention_mask=mask).last_hidden_state[i]
            v = mask[i].bool()
            close(got[i][v], want[v], f"request {i}")
            if a >= 0:
                other = plain(input_ids=ids, attention_mask=mask).last_hidden_state[i]
                assert (other[v] - want[v]).abs().max() > 100 * TOL * want[v].abs().max()
        close(model(input_ids=ids, attention_mask=mask).last_hidden_state, plain(input_ids=ids, attention_mask=mask).last_hidden_state, "outside")
        with pytest.raises(ValueError):
            with A.use_adapters([0, 1]):
                model(input_ids=ids, attention_mask=mask)


def test_a_bf16_batch_of_adapters():
    """bf16 rounds every layer's values, so the batch is held against the fp32 models as the merged bf16 models are."""
    plain, model, layers = _with_adapters(torch.bfloat16, hidden_size=256, num_attention_heads=4, intermediate_size=512)
    ids, mask = _batch()
    which = [1, 0, -1, 1]
    with torch.no_grad():
        with A.use_adapters(torch.tensor(which, device="cuda")):
            got = model(input_ids=ids, attention_mask=mask).last_hidden_state
        exact = copy.deepcopy(plain).float()
        wide = {n: copy.deepcopy(m).float() for n, m in layers.items()}
        for i, a in enumerate(which):
            v = mask[i].bool()
            best = (exact if a < 0 else _merged(exact, wide, a))(input_ids=ids, attention_mask=mask).last_hidden_state[i][v]
            merged = (plain if a < 0 else _merged(plain, layers, a))(input_ids=ids, attention_mask=mask).last_hidden_state[i][v]
            assert (got[i][v].float() - best).norm() <= util.MODEL_BF16_VS_EAGER_FACTOR * (merged.float() - best).norm()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_adapters_train_behind_the_last_attention(dtype):
    """Projection with adapters, dropout, residual and norm as they are used together, against the formulas in autograd."""
    torch.manual_seed(2)
    model = M.patch_model(hf.DebertaV2Model(_cfg(hidden_dropout_prob=0.0)), train_kernels=True).to("cuda", dtype).train().requires_grad_(False)
    last = "encoder.layer.1."
    layers = A.add_adapters(model, 2, 4, targets=(last + "attention.output.dense", last + "output.dense"))
    with torch.no_grad():
        for layer in layers.values():
            layer.lora_b.normal_(0, 0.1)
    ids, mask = _batch()
    mask = torch.ones_like(mask)
    which = torch.tensor([1, 0, -1, 1], device="cuda")
    with A.use_adapters(which):
        y = model(input_ids=ids, attention_mask=mask).last_hidden_state
    dy = torch.randn_like(y)
    params = [p for layer in layers.values() for p in (layer.lora_a, layer.lora_b)]
    grads = torch.autograd.grad(y, params, dy)

    class Plain(nn.Module):
        def __init__(self, layer):
            super().__init__()
            self.base, self.a, self.b = copy.deepcopy(layer.base).float(), layer.lora_a.detach().float().requires_grad_(), layer.lora_b.detach().float().requires_grad_()
            self.scaling = layer.scaling

        def forward(self, x):
            x = x.float()
            keep = (which >= 0).float()[:, None, None]
            a, b = self.a[which.clamp(min=0)], self.b[which.clamp(min=0)]
            return self.base(x) + keep * self.scaling * (x @ a.transpose(1, 2) @ b.transpose(1, 2))

    # the last layer once more in fp32 and elementary modules, from what its attention gives
    layer = model.encoder.layer[1]
    kept = {}
    hook = layer.attention.output.register_forward_pre_hook(lambda m, args: kept.update(context=args[0].detach(), hidden=args[1].detach()))
    with A.use_adapters(which):
        model(input_ids=ids, attention_mask=mask)
    hook.remove()
    first, second = Plain(layers[last + "attention.output.dense"]), Plain(layers[last + "output.dense"])
    norm = lambda m, x: nn.functional.layer_norm(x, m.normalized_shape, m.weight.float(), m.bias.float(), m.eps)  # noqa: E731
    mid = norm(layer.attention.output.LayerNorm, first(kept["context"]) + kept["hidden"].float())
    up = nn.functional.gelu(nn.functional.linear(mid, layer.intermediate.dense.weight.float(), layer.intermediate.dense.bias.float()))
    out = norm(layer.output.LayerNorm, second(up) + mid)
    want = torch.autograd.grad(out, [first.a, first.b, second.a, second.b], dy.float())
    for got, w in zip((y, *grads), (out, *want)):
        if dtype == torch.float32:
            close(got, w.detach(), "fp32")
        else:
            # seven roundings of half a step (2^-8 each at most) between the context and the result, five more on the way back, each of a value
            # that the next step weighs with others of its size: in the 2-norm no more than their sum
            assert (got.float() - w).norm() <= 12 * 2 ** -8 * w.norm()


def test_the_attention_still_has_no_backward_pass():
    model = M.patch_model(hf.DebertaV2Model(_cfg()), train_kernels=True).cuda().train()
    ids, mask = _batch()
    with pytest.raises(RuntimeError, match="forward-only"):
        model(input_ids=ids, attention_mask=mask).last_hidden_state.sum().backward()


def test_operators_in_a_row_captured():
    """A step of projection, dropout, residual and norm recorded into a graph while an eager graph of other leaves lives.  (One of the same leaves
    breaks the capture of a backward pass, of torch's own operators too: it keeps their accumulation on the stream that it was made on.)"""
    g = torch.Generator("cuda").manual_seed(0)
    r = lambda *s: (torch.randn(*s, device="cuda", generator=g) * 0.5).bfloat16()  # noqa: E731
    w, b, res, dy = r(128, 256), r(128), r(300, 128), r(300, 128)
    leaves = [r(300, 256), r(3, 8, 256), r(3, 128, 8), r(128), r(128)]
    twins = [t.clone().requires_grad_() for t in leaves]
    leaves = [t.requires_grad_() for t in leaves]
    ids = torch.randint(-1, 3, (300,), device="cuda", generator=g, dtype=torch.int32)
    seed = torch.tensor([4], device="cuda")

    def forward(leaves):
        y = lora_linear(leaves[0], w, b, leaves[1], leaves[2], 0.5, ids)
        return dropout_add_layer_norm(y, res, leaves[3], leaves[4], 1e-6, 0.1, seed)

    eager = forward(twins)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(forward(leaves), leaves, dy)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = forward(leaves)
        grads = torch.autograd.grad(y, leaves, dy)
    graph.replay()
    want = torch.autograd.grad(eager, twins, dy)
    torch.cuda.synchronize()
    assert torch.equal(y, eager) and all(torch.equal(a, c) for a, c in zip(grads, want))
