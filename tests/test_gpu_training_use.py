"""The training operators on the GPU in programs: transforms, checkpoints, changed modules, other
layouts and ids."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import training_reference as ref  # noqa: E402 (tests/ is on the path)

pytestmark = pytest.mark.gpu

SITE = 11


def _rng():
    return torch.tensor([0x1234567890ABCDEF, 7], device="cuda")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, shape, dtype, scale=1.0, at=0.0):
    return (torch.randn(shape, device="cuda", generator=gen) * scale + at).to(dtype)


@pytest.mark.parametrize("which", range(3))
def test_tangents_of_a_gradient_are_refused(which):
    """A tangent that only enters through the output's gradient must not be lost."""

    from disentangled_flash import training

    x = torch.randn(3, 16, device="cuda", requires_grad=True)
    w, b = torch.ones(16, device="cuda"), torch.zeros(16, device="cuda")
    with forward_ad.dual_level():
        y = (
            lambda: training.dropout(x, 0.5, _rng()),
            lambda: training.layer_norm(x, w, b, 1e-5),
            lambda: training.embedding(torch.arange(3, device="cuda"), x),
        )[which]()
        dy = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(y, x, dy)
