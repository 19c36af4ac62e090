"""Which modules the joined end of a sublayer may stand for; the native call is replaced by a recorder, so no GPU is needed."""
import pytest
import torch
from torch import nn
from transformers import DebertaV2Config
from transformers.models.deberta_v2 import modeling_deberta_v2 as hf

from turbodeberta_b200 import model as M
from turbodeberta_b200 import training as T


@pytest.fixture
def joined(monkeypatch):
    """The joined call's arguments, of every time it is made; the conditions on types and devices are taken as met."""
    calls = []

    def record(x, residual, weight, bias, eps, p=0.0, seed=None, offset=0):
        calls.append(p)
        return nn.functional.layer_norm(x + residual, weight.shape, weight, bias, eps)

    monkeypatch.setattr(T, "dropout_add_layer_norm", record)
    monkeypatch.setattr(T, "layer_norm", lambda x, w, b, eps: nn.functional.layer_norm(x, w.shape, w, b, eps))
    monkeypatch.setattr(T, "_norm_applies", lambda norm, x: True)
    return calls


def _end():
    cfg = DebertaV2Config(vocab_size=50, hidden_size=16, num_hidden_layers=1, num_attention_heads=2, intermediate_size=24, type_vocab_size=0,
                          hidden_dropout_prob=0.5)
    return M.patch_model(hf.DebertaV2Model(cfg), train_kernels=True).encoder.layer[0].output.train()


def _inputs():
    g = torch.Generator().manual_seed(0)
    return torch.randn(3, 24, generator=g), torch.randn(3, 16, generator=g)


def test_stock_modules_are_joined(joined):
    end = _end()
    end(*_inputs())
    assert joined == [0.5]
    end.dropout.eval()
    end(*_inputs())
    end.dropout = nn.Identity()
    end(*_inputs())
    assert joined == [0.5, 0.0, 0.0]


def test_a_users_own_dropout_and_norm_run(joined):
    class Thrice(nn.Dropout):
        def forward(self, x):
            return x * 3

    class Shifted(nn.LayerNorm):
        def forward(self, x):
            return super().forward(x) + 1

    class Doubled(nn.Identity):
        def forward(self, x):
            return x * 2

    h, x = _inputs()
    for own, factor in ((Thrice(0.5), 3), (Doubled(), 2)):
        end = _end()
        end.dropout = own
        assert torch.equal(end(h, x), end.LayerNorm(end.dense(h) * factor + x))
    end = _end()
    norm = Shifted(16, eps=end.LayerNorm.eps)
    end.LayerNorm, end.dropout = norm, nn.Identity()
    assert torch.equal(end(h, x), norm(end.dense(h) + x))
    assert not joined


def test_a_forward_of_an_instance_runs(joined):
    h, x = _inputs()
    end = _end()
    end.dropout.forward = lambda t: t * 3
    assert torch.equal(end(h, x), end.LayerNorm(end.dense(h) * 3 + x))
    end = _end()
    end.dropout = nn.Identity()
    stock = end.LayerNorm.forward
    end.LayerNorm.forward = lambda t: stock(t) + 1
    assert torch.equal(end(h, x), stock(end.dense(h) + x) + 1)
    assert not joined


def test_hooks_of_one_module_and_of_all_run(joined):
    h, x = _inputs()
    end, seen = _end(), []
    handle = end.dropout.register_forward_hook(lambda *a: seen.append("one"))
    end(h, x)
    handle.remove()
    assert seen == ["one"] and not joined
    handle = nn.modules.module.register_module_forward_hook(lambda m, *a: seen.append(type(m).__name__))
    try:
        end(h, x)
    finally:
        handle.remove()
    assert "FlashDropout" in seen and "FlashLayerNorm" in seen and not joined
