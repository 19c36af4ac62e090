"""Checkpointed parts of a model on the training path's kernels: the first pass, with or without gradients, and the one that is made again drop the same
elements, so a checkpointed step has the bits of the plain one."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint
from transformers import DebertaV2Config
from transformers.models.deberta_v2 import modeling_deberta_v2 as hf

from turbodeberta_b200 import model as M

pytestmark = pytest.mark.gpu


def _layer(dtype, **cfg):
    torch.manual_seed(0)
    cfg = DebertaV2Config(**{**dict(vocab_size=50, hidden_size=128, num_hidden_layers=1, num_attention_heads=2, intermediate_size=256, type_vocab_size=0,
                                    hidden_dropout_prob=0.3), **cfg})
    return M.patch_model(hf.DebertaV2Model(cfg), train_kernels=True).to("cuda", dtype).train()


def _step(part, inputs, run):
    leaves = [t.clone().requires_grad_() for t in inputs]
    torch.manual_seed(4)
    y = run(part, leaves)
    params = [p for p in part.parameters()]
    y.backward(torch.ones_like(y) * torch.arange(y.shape[-1], device="cuda"))
    out = [y.detach(), *(t.grad for t in leaves), *(p.grad for p in params)]
    for p in params:
        p.grad = None
    return out


WAYS = {"reentrant": lambda part, a: checkpoint(part, *a, use_reentrant=True), "other": lambda part, a: checkpoint(part, *a, use_reentrant=False)}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("way", list(WAYS))
@pytest.mark.parametrize("which", ["end", "dropout", "hooked end", "end without dropout"])
def test_a_checkpointed_part_drops_the_same_elements(which, way, dtype):
    model = _layer(dtype, **({"hidden_dropout_prob": 0.0} if which == "end without dropout" else {}))
    part = model.embeddings.dropout if which == "dropout" else model.encoder.layer[0].output
    if which == "hooked end":                        # then its modules run one by one
        part.LayerNorm.register_forward_hook(lambda *a: None)
    inputs = [torch.randn(50, n, device="cuda").to(dtype) for n in ((256,) if which == "dropout" else (256, 128))]
    want = _step(part, inputs, lambda p, a: p(*a))
    got = _step(part, inputs, WAYS[way])
    assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_a_pass_in_training_mode_drops_with_and_without_gradients_alike():
    part = _layer(torch.bfloat16).encoder.layer[0].output
    h, x = (torch.randn(50, n, device="cuda").bfloat16() for n in (256, 128))
    torch.manual_seed(1)
    want = part(h, x)
    torch.manual_seed(1)
    with torch.no_grad():
        assert torch.equal(part(h, x), want)
    part.eval()
    with torch.no_grad():                            # inference is torch's own
        assert torch.equal(part(h, x), torch.nn.functional.layer_norm(part.dense(h) + x, (128,), part.LayerNorm.weight, part.LayerNorm.bias, part.LayerNorm.eps))
