"""``training.orthogonalize`` at the ends of its range, held to the bound of ``test_gpu_orthogonalize``: twice
the error of fp32 iterations with fp16 operands, the result's rounding and fp32 sums."""

from __future__ import annotations

import pytest
import torch

from test_gpu_orthogonalize import DTYPES, _check, _normal  # noqa: E402 (tests/ is on the path)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,scale", [("fp32", 1e-40), ("fp32", 1e-37), ("bf16", 1e-38), ("fp32", 3e36),
                                        ("bf16", 3e36), ("fp16", 1e-5)])
@pytest.mark.parametrize("shape", [(140, 96), (96, 140), (90, 31)], ids=str)
def test_norms_at_the_ends_of_the_range(kind, scale, shape):
    """Elements of any size, subnormal ones too, and norms past fp32's range; eps = 0."""

    update = (_normal(11, shape, torch.float32).double() * 1e3 * scale).to(DTYPES[kind])
    assert bool((update != 0).any()) and bool(torch.isfinite(update).all())
    _check(update, eps=0.0)
