"""``training.orthogonalize`` on the GPU against its float64 statement.

Bound.  Let E be the error of X at the end of a step, in the Frobenius norm relative to X.  A step
multiplies with fp16 operands, each off by at most u = 2^-11 / 2 = 2^-12 of itself: A = X X^T is off
by 3 u |X|_F^2 at most (two operands and its own rounding), and so on; but worst-case chains over five
steps say nothing.  What the tests hold to is measured against arithmetic instead: operands
rounded to fp16 in a float32 iteration (``emulate``, rounding for rounding what the kernels do) give
E between 3e-4 and 3e-3 by the spectrum, and a different order of fp32 sums moves the roundings but
not their size.  The result may be off by twice the emulation's error, by the rounding of the result to bf16
(2^-8 of each element at most, 2^-9 on the root mean square) and by 1e-4 for the fp32 sums.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

COEFFICIENTS = (3.4445, -4.775, 2.0315)
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _exact(update, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    a, b, c = coefficients
    x = update.double()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    for _ in range(steps):
        s = x @ x.mT.contiguous()
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.mT if tall else x


def _emulate(update, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    a, b, c = coefficients

    def half(t):
        return t.half().float()

    x = update.float()
    x = x.mT if x.shape[-2] > x.shape[-1] else x
    norm = update.double().square().sum((-2, -1), keepdim=True).sqrt() + eps
    x = (x.double() / norm).float()
    for step in range(steps):
        high = half(x * 256) / 256
        rest = half((x - high) * 256) / 256
        x = high + rest if step == 0 or step + 1 < steps else high
        s = half(high @ high.mT.contiguous())
        x = a * x + half(b * s + c * (s @ s)) @ high
    return x.mT if update.shape[-2] > update.shape[-1] else x


def _distance(a, b):
    return ((a.double() - b).square().sum((-2, -1)).sqrt()
            / b.square().sum((-2, -1)).sqrt().clamp(min=1e-30))


def _normal(seed, shape, dtype, rank=None):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    g = torch.randn(shape, device="cuda", generator=gen)
    if rank:
        strong = torch.randn((*shape[:-1], rank), device="cuda", generator=gen)
        g = 0.05 * g + strong @ torch.randn((*shape[:-2], rank, shape[-1]), device="cuda",
                                            generator=gen)
    return (g * 1e-3).to(dtype)


def _check(update, **settings):
    from disentangled_flash.training import orthogonalize

    got = orthogonalize(update, **settings)
    assert got.dtype == torch.bfloat16 and got.shape == update.shape
    want = _exact(update, **settings)
    allowed = 2 * _distance(_emulate(update, **settings), want) + 2.0 ** -9 + 1e-4
    off = _distance(got, want)
    assert bool((off <= allowed).all()), (off.max().item(), allowed.min().item())


@pytest.mark.parametrize("kind", list(DTYPES))
@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (5, 1), (3, 200), (17, 100), (100, 17), (64, 64),
                                   (127, 129), (128, 128), (129, 127), (130, 300), (300, 130),
                                   (256, 1024), (512, 512), (1001, 437)], ids=str)
def test_shapes(kind, shape):
    _check(_normal(shape[0], shape, DTYPES[kind]))


@pytest.mark.parametrize("batch", [(1,), (3,), (2, 5)], ids=str)
@pytest.mark.parametrize("shape", [(96, 200), (200, 96), (256, 256)], ids=str)
def test_batches(batch, shape):
    _check(_normal(7, (*batch, *shape), torch.bfloat16, rank=8))


@pytest.mark.parametrize("steps", [1, 2, 3, 6, 7])
def test_steps(steps):
    _check(_normal(9, (200, 160), torch.float32, rank=20), steps=steps)


def test_other_coefficients_and_eps():
    update = _normal(10, (150, 260), torch.float32)
    _check(update, steps=12, coefficients=(1.5, -0.5, 0.0))  # the cubic, whose limit is 1
    _check(update, eps=1e-2)  # a norm of 0.2: the first X is shorter
    _check(update, coefficients=(2.0, -1.5, 0.5), eps=0.0)


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
@pytest.mark.parametrize("scale", [1e-30, 1e-18, 1e6, 1e30])
def test_sizes_of_elements(kind, scale):
    """The squares' sum neither overflows nor vanishes (eps = 0: the size alone counts)."""

    g = _normal(11, (140, 90), torch.float32) * 1e3
    _check((g * scale).to(DTYPES[kind]), eps=0.0)


def test_singular_values_come_near_one():
    from disentangled_flash.training import orthogonalize

    got = orthogonalize(_normal(12, (300, 500), torch.float32)).double()
    values = torch.linalg.svdvals(got)
    # (the quintic's range, and the error of X that the bound above allows)
    assert 0.65 < float(values.min()) and float(values.max()) < 1.25


def test_matrices_of_a_batch_stay_apart():
    """A matrix of zeros gives zeros, one with a NaN gives NaN, and the others are what they are
    alone."""

    from disentangled_flash.training import orthogonalize

    g = _normal(13, (5, 130, 140), torch.bfloat16)
    alone = orthogonalize(g)
    g[1] = 0
    g[3, 5, 7] = float("nan")
    got = orthogonalize(g)
    assert bool((got[1] == 0).all()) and bool(torch.isnan(got[3]).all())
    for n in (0, 2, 4):
        assert torch.equal(got[n], alone[n])


def test_layouts():
    from disentangled_flash.training import orthogonalize

    g = _normal(14, (4, 140, 260), torch.bfloat16)
    want = orthogonalize(g)
    assert torch.equal(orthogonalize(g.mT.contiguous().mT), want)
    assert torch.equal(orthogonalize(g[::2]), want[::2])
    flat = torch.empty(g.numel() + 1, dtype=g.dtype, device="cuda")[1:]  # off 16-byte boundaries
    assert torch.equal(orthogonalize(flat.copy_(g.flatten()).view_as(g)), want)
    assert torch.equal(orthogonalize(g.mT).mT, want)  # tall and wide take the same steps
    assert orthogonalize(g[:0]).shape == (0, 140, 260)
    assert not orthogonalize(g.clone().requires_grad_()).requires_grad


@pytest.mark.parametrize("shape", [(8, 8), (9, 300), (33, 30), (64, 64), (128, 128), (150, 140),
                                   (192, 600), (500, 500)], ids=str)
def test_results_are_off_by_little_more_than_their_rounding(shape):
    """By root mean squares over many matrices: the result's rounding and that of the operands.  Of up
    to 128 rows B and X are operands in parts, without which a model in 64 bits gave 1.45 times
    the rounding (128 rows) to 2.1 (9), with them 1.11 to 1.25 (1.8 for single matrices of 8
    and 9 rows, which are nearly singular); with more rows 1.4."""

    from disentangled_flash.training import orthogonalize

    update = _normal(21, (12, *shape), torch.bfloat16)
    want = _exact(update)
    got = orthogonalize(update).double()
    rounding = (want.to(torch.bfloat16).double() - want).square().sum().sqrt()
    assert (got - want).square().sum().sqrt() < 1.5 * rounding
