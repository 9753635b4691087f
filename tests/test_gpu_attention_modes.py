"""A backbone with the fused attention, as programs call it: validation before training, other forms of
masks, moved and copied models."""

from __future__ import annotations

import pytest
import torch

from test_gpu_attention_use import _batch, _grads, _model  # noqa: E402 (tests/ is on the path)

pytestmark = pytest.mark.gpu

pytest.importorskip("transformers")


@pytest.mark.parametrize("changed", [{}, {"position_buckets": -1, "max_relative_positions": 40}],
                         ids=str)
def test_training_after_a_validation_in_inference_mode(changed):
    """A length that is first met in inference mode trains as any other."""

    ids, mask = _batch()
    want, want_grads = _grads(_model(**changed), ids, mask)
    model = _model(**changed).eval()
    with torch.inference_mode():
        model(ids, attention_mask=mask)
    got, grads = _grads(model.train(), ids, mask)
    # (As between two runs of one model: torch's products differ by 1e-6.)
    assert float((got - want).abs().max()) < 1e-5 * float(want.abs().max())
    assert set(grads) == set(want_grads)
    for name, g in grads.items():
        w = want_grads[name]
        assert float((g - w).abs().max()) <= 1e-4 * float(w.abs().max()) + 1e-6, name
