"""``training.attention`` on the GPU against its float64 statement.

Every comparison is element by element against ``attention_reference``'s bounds, which are
derived there.
"""

from __future__ import annotations

import math

import pytest
import torch

import attention_reference as ref  # noqa: E402 (tests/ is on the path)
import training_reference as common

pytestmark = pytest.mark.gpu

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SEED, STEP, SITE = 0x1234567890ABCDEF, 7, 11


@pytest.fixture(params=list(DTYPES))
def dtype(request):
    return DTYPES[request.param]


def _rng(seed=SEED, step=STEP):
    return torch.tensor([seed, step], device="cuda")


def _lut(length, buckets=8, most=32):
    from disentangled_flash.position import compact_position_plan

    used, lut = compact_position_plan(length, position_buckets=buckets,
                                      max_relative_positions=most,
                                      position_embedding_size=buckets)
    return used.numel(), lut.cuda()


def _mask(kind, b, length, gen):
    if kind == "none":
        return None
    at = torch.arange(length, device="cuda")
    if kind == "ragged":
        kept = torch.randint(1, length + 1, (b, 1), device="cuda", generator=gen)
        return at[None] < kept
    if kind == "left":
        return at[None] >= torch.randint(0, length, (b, 1), device="cuda", generator=gen)
    if kind == "one":
        return at[None] == torch.randint(0, length, (b, 1), device="cuda", generator=gen)
    mask = torch.rand(b, length, device="cuda", generator=gen) < 0.6
    if kind == "empty":
        mask[0] = False
    return mask


def _case(seed, b, length, h, d, dtype, modes="both", mask="ragged", slots=None):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=gen).to(dtype)

    count, lut = _lut(length) if slots is None else slots
    q, k, v = (normal(b, length, h, d).requires_grad_() for _ in range(3))
    pk = normal(h, count, d).requires_grad_() if modes in ("both", "c2p") else None
    pq = normal(h, count, d).requires_grad_() if modes in ("both", "p2c") else None
    scale = 1 / math.sqrt(d * (1 + (pk is not None) + (pq is not None)))
    return [q, k, v, pk, pq, lut, scale, _mask(mask, b, length, gen)], normal(b, length, h, d)


def _gradients(y, inputs, dout):
    names = ("dq", "dk", "dv", "dpos_key", "dpos_query")
    wanted = [(n, t) for n, t in zip(names, inputs) if t is not None and t.requires_grad]
    grads = torch.autograd.grad(y, [t for _, t in wanted], dout)
    return dict(zip([n for n, _ in wanted], grads))


def _check(case, p=0.0, site=SITE):
    from disentangled_flash.training import attention

    args, dout = case
    q, length = args[0], args[0].shape[1]
    y = attention(*args, p=p, rng=_rng(), site=site)
    shape = (q.shape[0], q.shape[2], length, length)
    mult = common.factor(shape, p, _rng(), site) if p else None
    want = ref.attention(*args, mult=mult, dout=dout)
    got = {"out": y.detach(), **_gradients(y, args[:5], dout)}
    assert set(got) == set(want)
    for name, value in got.items():
        assert value.dtype == q.dtype
        common.check(value, want[name], name)


LENGTHS = [1, 2, 3, 15, 16, 17, 31, 32, 33, 47, 63, 64, 65, 96, 127, 128, 129, 200, 257]


@pytest.mark.parametrize("length", LENGTHS)
@pytest.mark.parametrize("d", [32, 64, 128])
def test_lengths(dtype, length, d):
    _check(_case(length, 2, length, 2, d, dtype), p=0.2)


@pytest.mark.parametrize("mask", ["none", "ragged", "left", "holes", "one", "empty"])
@pytest.mark.parametrize("length", [20, 64, 150])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_masks(dtype, mask, length, p):
    _check(_case(3, 3, length, 2, 64, dtype, mask=mask), p=p)


@pytest.mark.parametrize("modes", ["both", "c2p", "p2c", "neither"])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("length", [40, 130])
def test_terms(dtype, modes, d, length):
    _check(_case(5, 2, length, 3, d, dtype, modes=modes, mask="holes"), p=0.1)


@pytest.mark.parametrize("p", [1e-9, 0.5, 0.9, 1.0])
def test_dropout_shares(dtype, p):
    _check(_case(7, 2, 75, 2, 64, dtype), p=p)


def test_batches_and_heads():
    for b, h in ((1, 1), (5, 7), (17, 3)):
        _check(_case(b, b, 70, h, 32, torch.bfloat16), p=0.1)


@pytest.mark.parametrize("kind", ["one slot", "all slots", "shuffled", "outside"])
def test_position_tables(dtype, kind):
    """Any table of places: every delta its own row, all one row, in no order, some outside."""

    length = 100
    gen = torch.Generator().manual_seed(2)
    count, lut = {"one slot": (1, torch.zeros(199)), "all slots": (199, torch.arange(199)),
                  "shuffled": (50, torch.randint(0, 50, (199,), generator=gen)),
                  "outside": (20, torch.randint(-9, 30, (199,), generator=gen))}[kind]
    _check(_case(11, 2, length, 2, 64, dtype, slots=(count, lut.to("cuda", torch.int32))), p=0.1)


def test_a_long_sequence(dtype):
    from disentangled_flash.position import compact_position_plan

    used, lut = compact_position_plan(1100, position_buckets=256, max_relative_positions=512,
                                      position_embedding_size=256)
    _check(_case(13, 1, 1100, 2, 64, dtype, slots=(used.numel(), lut.cuda())), p=0.1)


@pytest.mark.parametrize("half,length", [(torch.float16, 17), (torch.bfloat16, 1500)])
def test_gradients_are_off_by_little_more_than_their_roundings(half, length):
    """G is rounded once and a gradient once, independently: sqrt(2) of one rounding, by root mean
    squares.  The rows of G add up to 0, so that on shared slots the sums are smaller than their terms
    and G's share is larger: 1.47 by a model of the roundings in 64 bits.  An output that was
    rounded before D, or of rounded probabilities, made it 1.54 (17 tokens) and 1.63."""

    from disentangled_flash.training import attention

    args, dout = _case(23, 1, length, 12 if length < 100 else 2, 64, half, mask="none",
                       slots=_lut(length, 256, 512))
    y = attention(*args, p=0.1, rng=_rng(), site=SITE)
    shape = (1, args[0].shape[2], length, length)
    want = ref.attention(*args, mult=common.factor(shape, 0.1, _rng(), SITE), dout=dout)
    for name, value in {"out": y.detach(), **_gradients(y, args[:5], dout)}.items():
        exact = want[name][0].double().to(value.device)
        error = (value.double() - exact).square().sum().sqrt()
        rounding = (exact.to(half).double() - exact).square().sum().sqrt()
        assert error < (1.2 if name == "out" else 1.52) * rounding, (name, error / rounding)
