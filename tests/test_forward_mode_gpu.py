"""Forward-mode derivatives: the operators have none and say so; the model's modules then run torch's own, as they did before they had kernels."""
import pytest
import torch
import torch.autograd.forward_ad as fw
from transformers import DebertaV2Config
from transformers.models.deberta_v2 import modeling_deberta_v2 as hf

from turbodeberta_b200 import model as M
from turbodeberta_b200.ops.dropout import dropout
from turbodeberta_b200.ops.layer_norm import dropout_add_layer_norm, layer_norm
from turbodeberta_b200.ops.lora import lora_linear

pytestmark = pytest.mark.gpu


def _calls():
    r = lambda *s: torch.randn(*s, device="cuda")  # noqa: E731
    x, res, w, b = r(6, 16), r(6, 16), r(16), r(16)
    lora = [r(6, 16), r(8, 16), r(8), r(1, 2, 16), r(1, 8, 2), r(1).abs()]
    return [(lambda t: dropout(t, 0.5, 1), [x]), (lambda t, w, b: layer_norm(t, w, b), [x, w, b]),
            (lambda t, s, w, b: dropout_add_layer_norm(t, s, w, b, 1e-6, 0.5, 1), [x, res, w, b]),
            (lambda t, w, b, la, lb, s: lora_linear(t, w, b, la, lb, s), lora)]


@pytest.mark.parametrize("which", range(4))
def test_operators_refuse_dual_tensors(which):
    f, args = _calls()[which]
    for i in range(len(args)):
        with fw.dual_level():
            dual = [fw.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(args)]
            with pytest.raises(RuntimeError, match="forward-mode"):
                f(*dual)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                f(*dual)
    f(*args)


@pytest.mark.parametrize("which", range(4))
def test_operators_refuse_dual_gradients(which):
    f, args = _calls()[which]
    x = args[0].clone().requires_grad_()
    y = f(x, *args[1:])
    with fw.dual_level():
        dy = fw.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(y, x, dy)


@pytest.mark.parametrize("which", range(4))
def test_operators_refuse_function_transforms(which):
    f, args = _calls()[which]
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: f(t, *args[1:]), (args[0],), (torch.ones_like(args[0]),))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: f(t, *args[1:]).sum())(args[0])


def _layer(train_kernels):
    torch.manual_seed(0)
    cfg = DebertaV2Config(vocab_size=50, hidden_size=16, num_hidden_layers=1, num_attention_heads=2, intermediate_size=24, type_vocab_size=0,
                          hidden_dropout_prob=0.3)
    model = M.patch_model(hf.DebertaV2Model(cfg), train_kernels=train_kernels).cuda().train()
    return model.encoder.layer[0].output, model.embeddings.dropout


@pytest.mark.parametrize("frozen", [True, False])
def test_modules_have_the_tangents_of_torchs(frozen):
    h, x, t = (torch.randn(5, n, device="cuda") for n in (24, 16, 16))
    out = []
    for own in (False, True):
        end, drop = _layer(own)
        end.requires_grad_(not frozen)
        torch.manual_seed(2)
        with fw.dual_level():
            y = fw.unpack_dual(end(h, fw.make_dual(x, t)))
            z = fw.unpack_dual(drop(fw.make_dual(x, t)))
            n = fw.unpack_dual(end.LayerNorm(fw.make_dual(x, t)))
        out.append([*y, *z, *n])
        torch.manual_seed(2)
        out[-1] += torch.func.jvp(lambda u: end(h, u), (x,), (t,), )
        out[-1].append(torch.func.grad(lambda u: end.LayerNorm(u).square().sum())(x))
    assert all(s is not None and torch.equal(s, u) for s, u in zip(*out))
