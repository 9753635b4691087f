"""CPU tests of ``training.attention``: the float64 statement that the GPU tests compare with, and
the refusals of the Python and the C interface."""

from __future__ import annotations

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import attention_reference as ref  # noqa: E402 (tests/ is on the path)


def _inputs(b=2, length=11, h=3, d=4, slots=5, dtype=torch.float64):
    gen = torch.Generator().manual_seed(0)

    def normal(*shape):
        return torch.randn(shape, generator=gen, dtype=torch.float64).to(dtype)

    lut = torch.randint(-1, slots + 1, (2 * length - 1,), generator=gen, dtype=torch.int32)
    mask = torch.rand(b, length, generator=gen) < 0.7
    mult = (torch.rand(b, h, length, length, generator=gen) < 0.8).double() / 0.8
    args = [normal(b, length, h, d) for _ in range(3)] + [normal(h, slots, d) for _ in range(2)]
    return args, lut, mask, mult, normal(b, length, h, d)


def _by_pairs(args, lut, scale, mask, mult):
    """The definition, pair by pair."""

    q, k, v, pk, pq = args
    b, length, h, d = q.shape
    out = torch.zeros(b, length, h, d, dtype=torch.float64)
    for n in range(b):
        for head in range(h):
            for i in range(length):
                if not mask[n, i]:
                    weights = torch.full((length,), 1.0 / length, dtype=torch.float64)
                else:
                    s = []
                    for j in range(length):
                        t = int(lut[i - j + length - 1])
                        x = q[n, i, head] @ k[n, j, head]
                        if 0 <= t < pk.shape[1]:
                            x = x + q[n, i, head] @ pk[head, t] + k[n, j, head] @ pq[head, t]
                        s.append(x * scale if mask[n, j] else torch.tensor(-torch.inf).double())
                    weights = torch.softmax(torch.stack(s), 0)
                out[n, i, head] = (weights * mult[n, head, i]) @ v[n, :, head]
    return out


def test_statement_is_the_definition():
    args, lut, mask, mult, _ = _inputs()
    got, bound = ref.attention(*args, lut, 0.4, mask, mult)["out"]
    assert torch.allclose(got, _by_pairs(args, lut, 0.4, mask, mult), rtol=1e-12, atol=1e-12)
    assert bool(torch.isfinite(bound).all()) and float(bound.max()) < 1e-4


def test_statement_gradients_are_autograds():
    args, lut, mask, mult, dout = _inputs()
    leaves = [a.clone().requires_grad_() for a in args]
    grads = torch.autograd.grad(_by_pairs(leaves, lut, 0.4, mask, mult), leaves, dout)
    want = ref.attention(*args, lut, 0.4, mask, mult, dout)
    for name, grad in zip(("dq", "dk", "dv", "dpos_key", "dpos_query"), grads):
        value, bound = want[name]
        assert torch.allclose(value, grad, rtol=1e-11, atol=1e-11), name
        assert bool(torch.isfinite(bound).all()) and float(bound.max()) < 1e-3, name


def test_statement_gradients_are_differences():
    args, lut, mask, mult, dout = _inputs()
    want = ref.attention(*args, lut, 0.4, mask, mult, dout)
    gen = torch.Generator().manual_seed(1)
    for n, name in enumerate(("dq", "dk", "dv", "dpos_key", "dpos_query")):
        direction = torch.randn(args[n].shape, generator=gen, dtype=torch.float64)
        step, values = 1e-5, []
        for sign in (1, -1):
            moved = [a + sign * step * direction if m == n else a for m, a in enumerate(args)]
            values.append((ref.attention(*moved, lut, 0.4, mask, mult)["out"][0] * dout).sum())
        difference = (values[0] - values[1]) / (2 * step)
        analytic = (want[name][0] * direction).sum()
        # The difference is off by step^2 / 6 of the third derivative and 1e-16 / step of the output.
        assert abs(difference - analytic) < 1e-7 * (1 + abs(analytic)), name


# ---- refusals ------------------------------------------------------------------------


def test_attention_wants_gpu_tensors():
    from disentangled_flash.training import attention

    x = torch.zeros(1, 4, 2, 64)
    with pytest.raises(RuntimeError, match="GPU"):
        attention(x, x, x, None, None, torch.zeros(7, dtype=torch.int32), 1.0)


def test_attention_refusals():
    from disentangled_flash.training import attention

    with FakeTensorMode():
        def t(*shape, dtype=torch.float16, device="cuda"):
            return torch.empty(shape, dtype=dtype, device=device)

        x, table = t(2, 8, 3, 64), t(3, 5, 64)
        lut, mask = t(15, dtype=torch.int32), t(2, 8, dtype=torch.bool)
        rng = t(2, dtype=torch.int64)
        good = dict(query=x, key=x, value=x, pos_key=table, pos_query=table, delta_to_slot=lut,
                    scale=0.1, mask=mask, p=0.1, rng=rng)
        assert attention(**good).shape == x.shape
        assert attention(**{**good, "pos_key": None, "mask": None, "p": 0}).shape == x.shape
        for error, match, changed in (
            (TypeError, "not fp16", {"query": x.double()}),
            (ValueError, "query must be", {"query": t(2, 8, 192)}),
            (ValueError, "query must be", {"query": t(2, 8, 3, 48)}),
            (ValueError, "query must be", {"query": t(2, 8, 0, 64)}),
            (ValueError, "16384", {"query": t(1, 16385, 3, 64)}),
            (ValueError, "key must match", {"key": t(2, 9, 3, 64)}),
            (ValueError, "value must match", {"value": x.float()}),
            (ValueError, "value must match", {"value": t(2, 8, 3, 64, device="cpu")}),
            (ValueError, "pos_key must be", {"pos_key": t(5, 3, 64)}),
            (ValueError, "pos_query must be", {"pos_query": t(3, 0, 64)}),
            (TypeError, "pos_query dtype", {"pos_query": table.bfloat16()}),
            (ValueError, "pos_key is on", {"pos_key": t(3, 5, 64, device="cpu")}),
            (ValueError, "slots", {"pos_query": t(3, 6, 64)}),
            (TypeError, "int32", {"delta_to_slot": lut.long()}),
            (TypeError, "int32", {"delta_to_slot": lut[None]}),
            (ValueError, "2L-1", {"delta_to_slot": lut[1:]}),
            (ValueError, "delta_to_slot is on", {"delta_to_slot": t(15, dtype=torch.int32,
                                                                    device="cpu")}),
            (ValueError, "mask must be", {"mask": mask.float()}),
            (ValueError, "mask must be", {"mask": t(2, 8, 8, dtype=torch.bool)}),
            (ValueError, "mask is on", {"mask": t(2, 8, dtype=torch.bool, device="cpu")}),
            (ValueError, "scale", {"scale": 0.0}), (ValueError, "scale", {"scale": float("nan")}),
            (ValueError, "scale", {"scale": -1.0}), (ValueError, "scale", {"scale": float("inf")}),
            (ValueError, "probability", {"p": 1.5}),
            (ValueError, "needs rng", {"rng": None}),
            (ValueError, "int64", {"rng": rng.int()}),
            (ValueError, "site", {"site": -1}),
        ):
            with pytest.raises(error, match=match):
                attention(**{**good, **changed})


@pytest.fixture(scope="module")
def lib():
    from disentangled_flash import _lib

    return _lib.load()


def _struct(**changed):
    from disentangled_flash import _lib

    a = _lib.AttentionTrain()
    for name in ("query", "key", "value", "pos_key", "pos_query", "delta_to_slot", "mask"):
        setattr(a, name, 1 << 20)  # (never read: every call here is refused)
    for name in ("query_strides", "key_strides", "value_strides"):
        setattr(a, name, (ctypes.c_int64 * 3)(8 * 192, 64, 192))
    a.pos_key_strides = a.pos_query_strides = (ctypes.c_int64 * 2)(5 * 64, 64)
    a.B, a.H, a.L, a.D, a.S, a.dtype, a.scale, a.p = 2, 3, 8, 64, 5, 0, 0.1, 0.0
    for name, value in changed.items():
        setattr(a, name, value)
    return a


def test_c_attention_refusals(lib):
    null, shape, head_dim, dtype, align, large = -1, -2, -3, -4, -5, -6
    strides = (ctypes.c_int64 * 3)(8 * 192, 64, 196)
    at = 1 << 20
    for code, changed in (
        (null, {"query": None}), (null, {"value": None}), (null, {"delta_to_slot": None}),
        (null, {"S": 0}), (shape, {"B": -1}), (shape, {"H": 0}), (shape, {"L": 0}),
        (shape, {"S": -1}), (shape, {"p": 1.1}), (shape, {"p": float("nan")}),
        (shape, {"scale": 0.0}), (shape, {"scale": float("nan")}), (shape, {"scale": float("inf")}),
        (head_dim, {"D": 48}), (dtype, {"dtype": 3}), (align, {"key": at + 8}),
        (align, {"pos_query": at + 2}), (align, {"delta_to_slot": at + 2}),
        (align, {"query_strides": strides}), (large, {"L": 16385}),
        (large, {"B": 1 << 20}), (large, {"S": 1 << 21}),
    ):
        a = _struct(**changed)
        assert lib.dflash_attention_train_fwd(a, None, 0, at, None, None, None, None) == code, changed
        assert lib.dflash_attention_train_bwd_workspace_bytes(a) == 0, changed
        assert lib.dflash_attention_train_bwd(a, at, at, at, None, at, at, at, at, None, None, at,
                                              1 << 40, None) == code, changed
    a = _struct()
    fwd, bwd = lib.dflash_attention_train_fwd, lib.dflash_attention_train_bwd
    assert fwd(a, None, 0, None, None, None, None, None) == null
    assert fwd(a, None, 0, at + 8, None, None, None, None) == align
    assert fwd(a, None, 0, at, at + 8, None, None, None) == align
    dropping = _struct(p=0.1)
    assert fwd(dropping, None, 0, at, None, None, at, None) == null
    assert fwd(dropping, at, 0, at, None, None, None, None) == null
    assert fwd(dropping, at, 0, at, None, None, at + 4, None) == align
    size = lib.dflash_attention_train_bwd_workspace_bytes(a)
    assert size > 0
    good = [at] * 3 + [None] + [at] * 7 + [size, None]
    for n, value, code in ((0, None, null), (1, None, null), (2, None, null), (4, None, null),
                           (6, None, null), (0, at + 8, align), (1, at + 8, align),
                           (2, at + 2, align), (9, at + 4, align), (10, None, null),
                           (11, size - 1, -7)):
        args = list(good)
        args[n] = value
        assert bwd(a, *args) == code, n
    args = list(good)
    assert bwd(dropping, *args) == null  # the bits
    assert bwd(_struct(pos_key=None), *args) == null  # a gradient of no table
    assert fwd(_struct(B=0), None, 0, None, None, None, None, None) == 0
    assert lib.dflash_attention_train_bits_bytes(2, 3, 65) == 2 * 3 * 65 * 16
    assert lib.dflash_attention_train_bits_bytes(0, 3, 65) == 0
