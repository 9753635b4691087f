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


@pytest.mark.parametrize("rows", [4, 16, 256])
@pytest.mark.parametrize("value,coefficients", [
    (13.0, (-4.775, 2.0315)),  # B reaches 57214
    (12.0, (-400.0, 0.0)),     # and -57600
    (250.0, (0.0, 0.0)),       # A 62500
    (250.0, (1.0, 0.0)),       # and B
])
def test_singular_values_near_the_most_that_fp16_holds(rows, value, coefficients):
    """All singular values of the first X are 1 / sqrt(rows); `a` brings them to `value`, and the
    second step's A and B come near 65504."""

    b, c = coefficients
    first = rows ** -0.5
    a = value / first - b * first ** 2 - c * first ** 4
    gen = torch.Generator(device="cuda").manual_seed(rows)
    update = torch.linalg.qr(torch.randn(rows + 60, rows, device="cuda", generator=gen))[0]
    assert abs(b * value ** 2 + c * value ** 4) < 65504 and value < 255
    _check(update, steps=2, coefficients=(a, b, c), eps=0.0)


@pytest.mark.parametrize("shape", [(5, 64, 96), (3, 300, 200), (2, 513, 1025)], ids=str)
def test_calls_are_repeatable(shape):
    from disentangled_flash.training import orthogonalize

    update = _normal(5, shape, torch.bfloat16, rank=9)
    want = orthogonalize(update)
    for _ in range(3):
        assert torch.equal(orthogonalize(update), want)
