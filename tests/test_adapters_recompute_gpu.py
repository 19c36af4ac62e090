"""Checkpointed passes with adapters on the GPU, where autograd has a thread of its own: the bits of the pass that is not checkpointed."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint
from transformers import DebertaV2Config
from transformers.models.deberta_v2 import modeling_deberta_v2 as hf

from turbodeberta_b200 import adapters as A
from turbodeberta_b200 import model as M

pytestmark = pytest.mark.gpu


def _model(dtype):
    torch.manual_seed(3)
    cfg = DebertaV2Config(vocab_size=500, hidden_size=128, num_hidden_layers=2, num_attention_heads=2, intermediate_size=256, relative_attention=True,
                          position_buckets=256, max_relative_positions=512, pos_att_type=["p2c", "c2p"], norm_rel_ebd="layer_norm", type_vocab_size=0,
                          position_biased_input=False, share_att_key=True, hidden_dropout_prob=0.1)
    model = M.patch_model(hf.DebertaV2Model(cfg), train_kernels=True).to("cuda", dtype).train().requires_grad_(False)
    last = "encoder.layer.1."
    layers = A.add_adapters(model, 3, 8, targets=(last + "attention.output.dense", last + "intermediate.dense", last + "output.dense"))
    with torch.no_grad():
        for layer in layers.values():
            layer.lora_b.normal_(0, 0.1)
    return model, [p for m in layers.values() for p in (m.lora_a, m.lora_b)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_checkpointed_model(dtype):
    model, params = _model(dtype)
    ids = torch.randint(0, 500, (4, 90), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    mask = (torch.arange(90, device="cuda") < torch.tensor([[90], [1], [37], [64]], device="cuda")).long()
    dy = None

    def step(inside):
        nonlocal dy
        torch.manual_seed(5)
        with A.use_adapters([2, -1, 0, 2]):
            y = model(input_ids=ids, attention_mask=mask).last_hidden_state
            dy = torch.randn_like(y) if dy is None else dy
            if inside:
                return [y.detach(), *torch.autograd.grad(y, params, dy)]
        return [y.detach(), *torch.autograd.grad(y, params, dy)]

    want = step(False)
    assert all(torch.isfinite(t).all() and t.any() for t in want)
    model.gradient_checkpointing_enable({"use_reentrant": False, "context_fn": A.recompute_contexts})
    for inside in (False, True):
        assert all(torch.equal(g, w) for g, w in zip(step(inside), want))


def test_a_checkpointed_part_in_both_forms():
    model, params = _model(torch.bfloat16)
    part = model.encoder.layer[1].output
    h, x = (torch.randn(4, 30, n, device="cuda").bfloat16() for n in (256, 128))
    params = [part.dense.lora_a, part.dense.lora_b]

    def step(run):
        torch.manual_seed(5)
        leaf = x.clone().requires_grad_()
        with A.use_adapters([2, -1, 0, 2]):
            y = run(leaf)
        y.backward(torch.ones_like(y) * torch.arange(128, device="cuda"))
        grads = [leaf.grad, *(p.grad for p in params)]
        for p in params:
            p.grad = None
        return [y.detach(), *grads]

    want = step(lambda leaf: part(h, leaf))
    for way in (lambda leaf: checkpoint(A.keep_adapters(part), h, leaf, use_reentrant=True),
                lambda leaf: checkpoint(A.keep_adapters(part), h, leaf, use_reentrant=False),
                lambda leaf: checkpoint(part, h, leaf, use_reentrant=False, context_fn=A.recompute_contexts)):
        assert all(torch.equal(g, w) for g, w in zip(step(way), want))
    with pytest.raises(RuntimeError, match="keep_adapters"):
        step(lambda leaf: checkpoint(part, h, leaf, use_reentrant=True))
