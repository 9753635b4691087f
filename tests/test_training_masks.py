"""CPU tests of the masks that a backbone with the fused attention takes: all that Hugging Face's encoder
takes, with its results."""

from __future__ import annotations

import pytest
import torch

from disentangled_flash import enable_deberta_training

pytest.importorskip("transformers")

from test_training_attention import _inputs, _model, calls  # noqa: E402, F401 (tests/ is on the path)


def _hidden():
    return torch.randn(3, 11, 64, generator=torch.Generator().manual_seed(2))


_, PADDING = _inputs()
MASKS = {
    "padding": PADDING, "one row for all": PADDING[1:2], "one value a sequence": PADDING[:, 3:4],
    "one value": PADDING[:1, :1], "numbers": PADDING * -3.5, "bool": PADDING.bool(),
    "queries": PADDING[:, None, :, None], "one row's queries": PADDING[1:2, None, :, None],
    "keys": PADDING[:, None, None, :], "pairs": PADDING[:, None, :, None] * PADDING[:, None, None, :],
    "3-D": (PADDING[:, :, None] * PADDING[:, None, :]).tril(), "a value of four dimensions":
    PADDING[:, None, 3:4, None],
}


@pytest.mark.parametrize("kind", MASKS)
def test_on_the_cpu_it_is_torchs(kind):
    model = _model(conv_kernel_size=0).eval()
    want = model.encoder(_hidden(), MASKS[kind]).last_hidden_state
    fused = enable_deberta_training(model, attention="hip").eval()
    assert torch.equal(fused.encoder(_hidden(), MASKS[kind]).last_hidden_state, want)


@pytest.mark.parametrize("kind", [k for k, m in MASKS.items() if m.dim() == 2])
def test_padding_masks_are_fused(calls, kind):  # noqa: F811
    """What the operator is called with is the mask of every token; padded queries' rows apart (1 / L of
    all keys either way) the result is the module's."""

    given = MASKS[kind]
    model = _model(conv_kernel_size=0).eval()
    want = model.encoder(_hidden(), given).last_hidden_state
    fused = enable_deberta_training(model, attention="hip").eval()
    got = fused.encoder(_hidden(), given).last_hidden_state
    kept = given.bool().expand(3, 11)
    assert len(calls) == 2 and all(torch.equal(c["mask"], kept) for c in calls)
    assert torch.allclose(got[kept], want[kept], atol=2e-6)


@pytest.mark.parametrize("kind", [k for k, m in MASKS.items() if m.dim() > 2])
def test_other_masks_are_not_fused(calls, kind):  # noqa: F811
    fused = enable_deberta_training(_model(conv_kernel_size=0), attention="hip").eval()
    fused.encoder(_hidden(), MASKS[kind])
    assert not calls


def test_masks_that_do_not_fit_are_refused(calls):  # noqa: F811
    fused = enable_deberta_training(_model(conv_kernel_size=0), attention="hip").eval()
    for mask in (PADDING[:2], PADDING[:, :5]):
        with pytest.raises(RuntimeError):
            fused.encoder(_hidden(), mask)
    assert not calls


def test_a_layer_called_by_itself():
    """Its attention takes Hugging Face's masks, in which no padding mask hides."""

    mask = PADDING[:, None, :, None]
    model = _model().eval()
    table = model.encoder.get_rel_embedding()
    want = model.encoder.layer[0].attention(_hidden(), mask, rel_embeddings=table)[0]
    fused = enable_deberta_training(model, attention="hip").eval()
    got = fused.encoder.layer[0].attention(_hidden(), mask, rel_embeddings=table)[0]
    assert torch.equal(got, want)


def test_relative_positions_by_name():
    """The encoder's methods take their arguments by name too."""

    model = enable_deberta_training(_model(), attention="hip")
    hidden = _hidden()
    places = torch.ones(1, 11, 11, dtype=torch.long)
    assert model.encoder.get_rel_pos(hidden, relative_pos=places) is places
    assert model.encoder.get_rel_pos(hidden, None, places) is places
    assert model.encoder.get_rel_pos(hidden_states=hidden, query_states=None,
                                     relative_pos=places) is places
    assert model.encoder.get_rel_pos(hidden, query_states=hidden) is None
    mask = model.encoder.get_attention_mask(attention_mask=PADDING)
    assert torch.equal(mask.flatten(1), PADDING)
    pairs = model.encoder.get_attention_mask(attention_mask=MASKS["3-D"])
    assert torch.equal(pairs, MASKS["3-D"][:, None])
