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


def test_vmap_with_an_rng_for_every_sample():
    """The samples' values are those of calls by themselves."""

    from disentangled_flash import training

    x = torch.randn(4, 6, 72, device="cuda")
    w, b = torch.rand(2, 72, device="cuda")
    rngs = torch.stack([_rng() + i for i in range(4)])

    def tail(t, r):
        return training.layer_norm(training.dropout(t, 0.3, r, 1), w, b, 1e-5, t, 0.5, r, SITE)

    got = torch.func.vmap(tail)(x, rngs)
    for i in range(4):
        assert torch.equal(got[i], tail(x[i], rngs[i]))
    assert not torch.equal(torch.func.vmap(tail)(x[:1].expand(2, 6, 72), rngs[:2])[0],
                           tail(x[0], rngs[1]))
    table = torch.randn(9, 72, device="cuda")
    ids = torch.arange(8, device="cuda").view(4, 2)
    assert torch.equal(torch.func.vmap(lambda i: training.embedding(i, table))(ids), table[ids])
