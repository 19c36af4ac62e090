"""Passes under torch.inference_mode where the encoder runs layer by layer (with adapters, or with a hook on a layer): masks made outside and inside of it."""
import pytest
import torch
from transformers import DebertaV2Config
from transformers.models.deberta_v2 import modeling_deberta_v2 as hf

from turbodeberta_b200 import adapters as A
from turbodeberta_b200 import model as M

pytestmark = pytest.mark.gpu
LENGTHS = {"full": [90, 90, 90, 90], "ragged": [90, 1, 37, 64]}


def _model(dtype=torch.float32):
    torch.manual_seed(0)
    cfg = DebertaV2Config(vocab_size=500, hidden_size=128, num_hidden_layers=2, num_attention_heads=2, intermediate_size=256, relative_attention=True,
                          position_buckets=256, max_relative_positions=512, pos_att_type=["p2c", "c2p"], norm_rel_ebd="layer_norm", type_vocab_size=0,
                          position_biased_input=False, share_att_key=True)
    return M.patch_model(hf.DebertaV2Model(cfg)).eval().to("cuda", dtype)


def _ids():
    return torch.randint(0, 500, (4, 90), device="cuda", generator=torch.Generator("cuda").manual_seed(2))


def _mask(lengths):
    return (torch.arange(90, device="cuda") < torch.tensor(lengths, device="cuda")[:, None]).long()


@pytest.mark.parametrize("with_adapters", [True, False])
@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("made", ["outside", "inside"])
@pytest.mark.parametrize("lengths", list(LENGTHS))
def test_a_pass_layer_by_layer(lengths, made, packed, with_adapters):
    model, ids = _model(), _ids()
    model.encoder.pack_padded_batches = packed
    if with_adapters:
        with torch.no_grad():
            for layer in A.add_adapters(model, 3, 4).values():
                layer.lora_b.normal_(0, 0.1)
    else:
        model.encoder.layer[0].register_forward_hook(lambda *a: None)
    chosen = [2, -1, 0, 2] if with_adapters else [-1] * 4
    with torch.no_grad(), A.use_adapters(chosen):
        want = model(input_ids=ids, attention_mask=_mask(LENGTHS[lengths])).last_hidden_state
    outside = _mask(LENGTHS[lengths])
    with torch.inference_mode(), A.use_adapters(chosen):
        mask = outside if made == "outside" else _mask(LENGTHS[lengths])
        for _ in range(2):
            got = model(input_ids=ids, attention_mask=mask).last_hidden_state
            assert torch.equal(got, want)


def test_a_mask_changed_in_inference_mode_is_looked_at_again():
    """Such a tensor counts no versions."""
    model, ids = _model(), _ids()
    model.encoder.layer[0].register_forward_hook(lambda *a: None)
    with torch.no_grad():
        want = [model(input_ids=ids, attention_mask=_mask(LENGTHS[k])).last_hidden_state for k in ("full", "ragged", "full")]
    with torch.inference_mode():
        mask = _mask(LENGTHS["full"])
        for k, w in zip(("full", "ragged", "full"), want):
            mask.copy_(_mask(LENGTHS[k]))
            assert torch.equal(model(input_ids=ids, attention_mask=mask).last_hidden_state, w)
