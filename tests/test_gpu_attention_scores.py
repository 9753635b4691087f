"""``training.attention`` with large scores: the range of bf16 inputs, and probabilities of the backward
pass that are the forward pass's."""

from __future__ import annotations

import math

import pytest
import torch

import attention_reference as ref  # noqa: E402 (tests/ is on the path)
from training_reference import U

pytestmark = pytest.mark.gpu


def _inputs(b, length, h, d, dtype, query, tables, slots=40):
    gen = torch.Generator(device="cuda").manual_seed(length + d)

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=gen)

    q = (query * normal(b, length, h, d)).to(dtype)
    k, v, dout = (normal(b, length, h, d).to(dtype) for _ in range(3))
    pk, pq = ((tables * normal(h, slots, d)).to(dtype) for _ in range(2))
    lut = torch.randint(0, slots, (2 * length - 1,), device="cuda", dtype=torch.int32, generator=gen)
    return [q, k, v, pk, pq, lut, 1 / math.sqrt(3 * d)], dout


def _scores(q, k, pk, pq, lut, scale):
    """``[B, H, L, L]`` in 64 bits, and the sums of the absolute values of its products."""

    def sums(q, k, pk, pq):
        q, k = (t.transpose(1, 2) for t in (q, k))
        pk, pq = (ref.expand(t, lut) for t in (pk, pq))
        s = q @ k.mT.contiguous() + ref.from_delta(q @ pk.mT.contiguous())
        return s + ref.from_delta((k @ pq.mT.contiguous()).flip(-1)).mT

    given = [t.double() for t in (q, k, pk, pq)]
    return sums(*given) * scale, sums(*(t.abs() for t in given)) * scale


def _gradients(args, dout):
    from disentangled_flash.training import attention

    leaves = [t.detach().requires_grad_() for t in args[:5]]
    out = attention(*leaves, *args[5:])
    return out.detach(), torch.autograd.grad(out, leaves, dout)


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_scores_past_the_range_of_16_bits(dtype, d):
    """Relative scores of some 100 000: a row takes the value of its largest score, and nothing
    overflows.

    A score of n products is off by (d + 6) U sum|t| at most (two roundings of the scaled sums, one of each
    of d products and two sums) on either side of a comparison; where a row's largest lies 32 and
    twice that above the next, all other probabilities together are below 100 exp(-32) < 2^-39, so the row of
    the output is V's, within half a step, and G vanishes but for the roundings of
    D_i and of dO_i.V_j: (d + 8) U |dO|.|V| each, in sums of d products, and 2^-38 of them."""

    args, dout = _inputs(2, 100, 2, d, dtype, 400, 400)
    q, k, v, pk, pq, lut, scale = args
    s, size = _scores(q, k, pk, pq, lut, scale)
    assert float(s.abs().max()) > 65504
    error = (d + 6) * U * size.amax(-1)
    top = s.topk(2, -1)
    sure = top.values[..., 0] - top.values[..., 1] > 32 + 2 * error
    assert float(sure.double().mean()) > 0.8
    out, grads = _gradients(args, dout)
    assert bool(torch.isfinite(out).all())
    for g in grads:
        assert bool(torch.isfinite(g).all())
    heads = v.double().transpose(1, 2)
    chosen = heads.gather(2, top.indices[..., :1].expand(heads.shape))
    got = out.double().transpose(1, 2)
    assert bool(((got - chosen).abs() <= 2.0 ** -22 * (chosen.abs() + 8))[sure].all())
    g = (2 * (d + 8) * U + 2.0 ** -37) * (dout.double().transpose(1, 2).abs() @ heads.abs().mT.contiguous())
    # dQ_i = scale sum_j G_ij (K_j + PK[t]): the terms' sizes, by the same sums.
    rows = ref.expand(pk.double().abs(), lut)
    allowed = scale * (g @ k.double().abs().transpose(1, 2) + ref.by_delta(g) @ rows)
    assert bool((grads[0].double().transpose(1, 2).abs() <= 1.05 * allowed + 1e-30)[sure].all())


@pytest.mark.parametrize("scores", [4.0, 40.0, 400.0, 4000.0])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("d", [64, 128])
def test_probabilities_of_the_backward_pass_add_up_to_1(dtype, d, scores):
    """With dO_i the i-th unit vector the sum over keys of dV_j is the row sum of query i's
    probabilities, as the backward pass has them.

    A probability is rounded to the dtype (u of itself, or half a subnormal's step) and so is dV: 2 u and
    64 floors.  Scores of both passes are the same operations on the same numbers, so that
    their difference from the statistic is off by that one's rounding and the difference's, 4 U max|s| log2 e
    with the exponential's own 4 U, and by the sums' 2 L U."""

    length = 64
    args, _ = _inputs(1, length, 2, d, dtype, 1, 1)
    s, _ = _scores(*args[:2], *args[3:])
    args[6] *= scores / float(s.abs().max())
    dout = torch.zeros(1, length, 2, d, device="cuda", dtype=dtype)
    dout[0, torch.arange(length), :, torch.arange(length)] = 1
    _, grads = _gradients(args, dout)
    rows = grads[2].double().sum((0, 1))[:, :length]  # [H, query]
    info = torch.finfo(dtype)
    u = 0.0 if dtype == torch.float32 else info.eps / 2
    allowed = 2 * u + 2 * length * info.tiny * info.eps \
        + U * (8 * scores * 1.4427 + 2 * length + 16)
    assert float((rows - 1).abs().max()) <= allowed, ((rows - 1).abs().max().item(), allowed)


@pytest.mark.parametrize("size", [1.0, 30.0])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("d", [32, 64, 128])
def test_statistics_are_those_of_fp32_scores(d, dtype, size):
    """A row's log2 of the sum of its exponentials is off by the largest error of its scores, (d + 6) U sum|t|,
    by (L + 32) U of a sum of L exponentials, and by the roundings of the result, its parts and its base, 4 U
    of its size and of 1."""

    from disentangled_flash import training

    length = 90
    args, _ = _inputs(2, length, 3, d, dtype, size, 2)
    q, k, v, pk, pq, lut, scale = args
    training._load()
    lse = torch.ops.disentangled_flash.attention_train(q, k, v, pk, pq, lut, None, None, scale, 0.0,
                                                       0)[2]
    s, sums = _scores(q, k, pk, pq, lut, scale)
    want = torch.logsumexp(s, -1) / math.log(2)
    allowed = 1.4427 * ((d + 6) * U * sums.amax(-1) + (length + 32) * U) + 4 * U * (want.abs() + 1)
    assert bool(((lse.double() - want).abs() <= allowed).all())
