"""Putting adapters into a model, loading them, and the classes of the training path; no GPU needed."""
import pytest
import torch
from torch import nn
from transformers import DebertaV2Config
from transformers.models.deberta_v2 import modeling_deberta_v2 as hf

from turbodeberta_b200 import adapters as A
from turbodeberta_b200 import model as M
from turbodeberta_b200 import training as T


def _cfg(**more):
    return DebertaV2Config(vocab_size=100, hidden_size=128, num_hidden_layers=2, num_attention_heads=2, intermediate_size=256, relative_attention=True,
                           position_buckets=256, max_relative_positions=512, pos_att_type=["p2c", "c2p"], norm_rel_ebd="layer_norm", type_vocab_size=0,
                           position_biased_input=False, **{"share_att_key": True, **more})


def test_adapters_take_the_linears_places():
    model = M.patch_model(hf.DebertaV2Model(_cfg()))
    layers = A.add_adapters(model, count=3, rank=4, scaling=2.0)
    assert len(layers) == 2 * 4 and "encoder.layer.1.attention.self.value_proj" in layers and "encoder.layer.0.output.dense" in layers
    for name, layer in layers.items():
        assert model.get_submodule(name) is layer and not layer.base.weight.requires_grad and layer.lora_a.requires_grad
        assert layer.lora_a.shape == (3, 4, layer.in_features) and not layer.lora_b.any()
    assert isinstance(model.encoder.layer[0].attention.self.key_proj, nn.Linear)
    with pytest.raises(ValueError, match="adapters already"):
        A.add_adapters(model, 1, 1)
    x = torch.randn(3, 128)
    one = model.encoder.layer[0].attention.output.dense
    assert torch.equal(one(x), one.base(x))          # outside use_adapters


def test_projections_that_make_the_tables_are_refused():
    for target in ("query_proj", "key_proj"):
        with pytest.raises(ValueError, match="relative-position tables"):
            A.add_adapters(M.patch_model(hf.DebertaV2Model(_cfg())), 1, 1, targets=(target,))
    apart = M.patch_model(hf.DebertaV2Model(_cfg(share_att_key=False)))
    with pytest.raises(ValueError, match="relative-position tables"):
        A.add_adapters(apart, 1, 1, targets=("pos_key_proj",))
    assert len(A.add_adapters(apart, 1, 1, targets=("self.query_proj", "self.key_proj"))) == 4
    with pytest.raises(ValueError, match="named like"):
        A.add_adapters(M.patch_model(hf.DebertaV2Model(_cfg())), 1, 1, targets=("nothing",))
    with pytest.raises(ValueError, match="positive"):
        A.add_adapters(M.patch_model(hf.DebertaV2Model(_cfg())), 0, 1)


def test_loading_an_adapter():
    model = M.patch_model(hf.DebertaV2Model(_cfg()))
    layers = A.add_adapters(model, count=3, rank=4, scaling=2.0)
    name = "encoder.layer.0.intermediate.dense"
    a, b = torch.randn(2, 128), torch.randn(256, 2)
    A.load_adapter(model, 1, {name: (a, b)}, scaling=1.0)
    got = layers[name]
    assert torch.equal(got.lora_a[1, :2], a) and not got.lora_a[1, 2:].any() and torch.equal(got.lora_b[1, :, :2], b * 0.5) and not got.lora_b[1, :, 2:].any()
    assert not layers["encoder.layer.0.output.dense"].lora_a[1].any()
    with pytest.raises(ValueError, match="no adapters at"):
        A.load_adapter(model, 1, {"pooler": (a, b)})
    with pytest.raises(ValueError, match="the model has 3"):
        A.load_adapter(model, 3, {})
    for bad in ((torch.zeros(5, 128), torch.zeros(256, 5)), (torch.zeros(2, 127), b), (a, torch.zeros(256, 3)), (a, torch.zeros(255, 2))):
        with pytest.raises(ValueError, match="do not fit"):
            A.load_adapter(model, 1, {name: bad})
    assert torch.equal(got.lora_a[1, :2], a)         # a refused one leaves the old one


def test_ids_of_a_thread_and_of_a_block():
    assert A._ACTIVE.ids is None
    with A.use_adapters([1, -1]):
        assert A._ACTIVE.ids.tolist() == [1, -1]
        with A.use_adapters(torch.tensor([0])):
            assert A._ACTIVE.ids.tolist() == [0]
            with A.packed_rows(torch.tensor([0, 1, 2]), 1, 4):
                assert A._ACTIVE.rows.tolist() == [[0, 0, 0]]
        assert A._ACTIVE.ids.tolist() == [1, -1] and A._ACTIVE.rows is None
        with A.packed_rows(torch.tensor([0, 3, 4, 7]), 2, 4):
            assert A._ACTIVE.rows.tolist() == [[1, 1, -1, -1]]
        with pytest.raises(ValueError, match="2 sequences, but the batch has 3"):
            with A.packed_rows(torch.tensor([0]), 3, 4):
                pass
    assert A._ACTIVE.ids is None
    for bad in (torch.tensor([0.5]), torch.tensor([[0]])):
        with pytest.raises(ValueError, match="one integer"):
            with A.use_adapters(bad):
                pass


def test_train_kernels_swap_stock_modules_only():
    class Own(nn.LayerNorm):
        pass

    model = hf.DebertaV2ForSequenceClassification(_cfg(num_labels=2))
    model.own = Own(4)
    before = list(model.state_dict())
    M.patch_model(model, train_kernels=True)
    layer = model.deberta.encoder.layer[0]
    assert type(layer.output) is T.FlashDebertaV2Output and type(layer.attention.output) is T.FlashDebertaV2SelfOutput
    assert type(layer.output.LayerNorm) is T.FlashLayerNorm and type(model.deberta.embeddings.dropout) is T.FlashDropout and type(model.own) is Own
    assert list(model.state_dict()) == before
    plain = M.patch_model(hf.DebertaV2Model(_cfg()))
    assert type(plain.encoder.layer[0].output) is hf.DebertaV2Output
    x = torch.randn(2, 128, requires_grad=True)      # on the CPU they are what they were
    assert torch.equal(layer.output.LayerNorm(x), nn.functional.layer_norm(x, (128,), layer.output.LayerNorm.weight, layer.output.LayerNorm.bias, layer.output.LayerNorm.eps))
    layer.eval()
    with torch.no_grad():
        h = torch.randn(2, 256)
        assert torch.equal(layer.output(h, x), layer.output.LayerNorm(layer.output.dense(h) + x))
