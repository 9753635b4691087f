"""CPU tests of ``training.Muon``: its state beside that of ``torch.optim.Muon``, and steps that are
refused before anything changes."""

from __future__ import annotations

import copy
import pickle

import pytest
import torch
from torch import nn

from disentangled_flash import training

pytest.importorskip("transformers")

from test_training_attention import _exact  # noqa: E402 (tests/ is on the path)

SHAPES = ((6, 4), (3, 7), (6, 4), (5, 5))


@pytest.fixture(autouse=True)
def _on_the_cpu(monkeypatch):
    monkeypatch.setattr(training, "orthogonalize", lambda update, steps, coefficients, eps: _exact(
        update, steps, coefficients, eps).to(torch.bfloat16))
    monkeypatch.setattr(training, "_check_floating", lambda *a: None)


def _params(seed=0):
    gen = torch.Generator().manual_seed(seed)
    return [nn.Parameter(torch.randn(s, generator=gen)) for s in SHAPES]


def _steps(optimizers, count, seed, momenta=None):
    """The same gradients to the parameters of every optimizer."""

    gen = torch.Generator().manual_seed(seed)
    for n in range(count):
        grads = [torch.randn(s, generator=gen) for s in SHAPES]
        for optimizer in optimizers:
            if momenta:
                optimizer.param_groups[0]["momentum"] = momenta[n]
            for p, g in zip(optimizer.param_groups[0]["params"], grads):
                p.grad = g.clone()
            optimizer.step()


def _buffers(optimizer):
    return [optimizer.state[p]["momentum_buffer"] for p in optimizer.param_groups[0]["params"]]


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("adjust", [None, "match_rms_adamw"])
def test_average_is_torchs_rule(nesterov, adjust):
    """States bit for bit, with a momentum that changes.  torch's products of bf16 are off by up to
    5e-2 of a step, these by 2^-8: steps agree to 0.1 of their size."""

    settings = dict(lr=0.1, weight_decay=0.0, nesterov=nesterov, adjust_lr_fn=adjust)
    theirs = torch.optim.Muon(_params(), **settings)
    ours = training.Muon(_params(), average=True, **settings)
    for n in range(5):
        before = [[p.detach().clone() for p in o.param_groups[0]["params"]] for o in (theirs, ours)]
        _steps((theirs, ours), 1, seed=n, momenta=[0.5 + 0.1 * n])
        assert all(map(torch.equal, _buffers(ours), _buffers(theirs)))
        moved = [[p.detach() - b for p, b in zip(o.param_groups[0]["params"], was)]
                 for o, was in zip((theirs, ours), before)]
        for a, b in zip(*moved):
            assert float((a - b).norm()) < 0.1 * float(a.norm())


@pytest.mark.parametrize("nesterov", [True, False])
def test_both_rules_take_the_same_steps(nesterov):
    """While momentum stays what it is: up to the roundings of fp32 sums and of the result to bf16, by
    half a step, 2^-8, of an element, and eps."""

    found = []
    for average in (False, True):
        params = _params()
        _steps([training.Muon(params, lr=0.1, nesterov=nesterov, average=average)], 4, seed=3)
        found.append([p.detach() for p in params])
    for a, b in zip(*found):
        # Four steps of 0.1 with elements up to 1.2 sqrt(1.5), each off by a step of bf16.
        assert float((a - b).abs().max()) < 4 * 0.1 * 1.5 * 2 ** -7


def test_states_move_to_torchs_and_back():
    theirs = torch.optim.Muon(_params(), lr=0.1)
    _steps([theirs], 3, seed=1)
    state = theirs.state_dict()
    ours = training.Muon(_params(), lr=0.3)
    with pytest.raises(ValueError, match="average"):
        ours.load_state_dict(state)
    assert not ours.state and ours.param_groups[0]["lr"] == 0.3
    state = copy.deepcopy(state)
    state["param_groups"][0]["average"] = True
    ours.load_state_dict(state)
    assert ours.param_groups[0]["average"] is True and ours.param_groups[0]["lr"] == 0.1
    _steps((theirs, ours), 3, seed=2)
    assert all(map(torch.equal, _buffers(ours), _buffers(theirs)))
    back = torch.optim.Muon(_params())
    back.load_state_dict(copy.deepcopy(ours.state_dict()))
    _steps((back, ours), 2, seed=3)
    assert all(map(torch.equal, _buffers(ours), _buffers(back)))


@pytest.mark.parametrize("average", [True, False])
def test_own_states_keep_their_rule(average):
    ours = training.Muon(_params(), average=average)
    _steps([ours], 2, seed=1)
    other = training.Muon(_params(), average=not average)
    other.load_state_dict(copy.deepcopy(ours.state_dict()))
    pickled = pickle.loads(pickle.dumps(ours))
    _steps((ours, other, pickled), 2, seed=2)
    for o in (other, pickled):
        assert o.param_groups[0]["average"] is average
        assert all(map(torch.equal, _buffers(o), _buffers(ours)))


def test_averages_stay_in_the_range_of_their_gradients():
    for average in (False, True):
        p = nn.Parameter(torch.zeros(3, 4, dtype=torch.float16))
        optimizer = training.Muon([p], average=average)
        for _ in range(60):
            p.grad = torch.full_like(p, 6000)
            optimizer.step()
        buffer = optimizer.state[p]["momentum_buffer"]
        assert bool(torch.isfinite(buffer).all()) == average
        if average:
            assert bool((buffer <= 6000).all()) and bool(torch.isfinite(p).all())


def _two_groups(bad, **settings):
    good = nn.Parameter(torch.ones(3, 4))
    optimizer = training.Muon([{"params": [good]}, {"params": [bad], **settings}], lr=0.1)
    good.grad, bad.grad = torch.ones_like(good), torch.ones_like(bad)
    return optimizer, good


def _unchanged(optimizer, good):
    return not optimizer.state and torch.equal(good, torch.ones(3, 4))


@pytest.mark.parametrize("settings", [{"ns_steps": 0}, {"eps": -1.0}, {"eps": float("nan")}], ids=str)
def test_a_refused_step_changes_no_group(settings):
    optimizer, good = _two_groups(nn.Parameter(torch.ones(2, 2)), **settings)
    with pytest.raises(ValueError):
        optimizer.step()
    assert _unchanged(optimizer, good)
    optimizer.param_groups[1].update(ns_steps=5, eps=1e-7)
    optimizer.step()
    assert len(optimizer.state) == 2 and not _unchanged(optimizer, good)


def test_a_refused_parameter_changes_no_group(monkeypatch):
    def check(name, tensor):
        if tensor.shape == (2, 2):
            raise RuntimeError("must be on a GPU")

    monkeypatch.setattr(training, "_check_floating", check)
    optimizer, good = _two_groups(nn.Parameter(torch.ones(2, 2)))
    with pytest.raises(RuntimeError, match="GPU"):
        optimizer.step()
    assert _unchanged(optimizer, good)
    optimizer, good = _two_groups(nn.Parameter(torch.ones(2, 3)))
    optimizer.param_groups[1]["params"][0].grad = torch.ones(2, 3).to_sparse()
    with pytest.raises(RuntimeError, match="sparse"):
        optimizer.step()
    assert _unchanged(optimizer, good)


def test_sizes_that_are_refused(monkeypatch):
    from torch._subclasses.fake_tensor import FakeTensorMode

    monkeypatch.undo()
    with FakeTensorMode():
        for shape in ((65536, 2, 3), (2, 2 ** 20 + 1, 2), (3, 2 ** 19, 2 ** 18)):
            with pytest.raises(ValueError, match="at most"):
                training.orthogonalize(torch.empty(shape, device="cuda"))
        assert training.orthogonalize(torch.empty(65535, 2, 3, device="cuda")).shape[0] == 65535
    with FakeTensorMode():
        many = [nn.Parameter(torch.empty(2 ** 20 + 1, 1, device="cuda"))]
        optimizer = training.Muon(many)
        many[0].grad = torch.empty_like(many[0])
        with pytest.raises(ValueError, match="at most"):
            optimizer.step()
        assert not optimizer.state


def test_groups_of_a_shape_keep_their_settings():
    """Parameters of one shape in two groups: each group's own rate and momentum."""

    def steps(optimizer, params):
        gen = torch.Generator().manual_seed(7)
        for _ in range(3):
            for p in params:
                p.grad = torch.randn(p.shape, generator=gen)
            optimizer.step()
        return [p.detach() for p in params]

    a = [nn.Parameter(torch.ones(3, 4)) for _ in range(2)]
    both = steps(training.Muon([{"params": a[:1], "lr": 0.1}, {"params": a[1:], "lr": 0.2,
                                                               "momentum": 0.5}]), a)
    for n, settings in ((0, {"lr": 0.1}), (1, {"lr": 0.2, "momentum": 0.5})):
        b = [nn.Parameter(torch.ones(3, 4)) for _ in range(2)]
        alone = steps(training.Muon(b, **settings), b)
        assert torch.equal(alone[n], both[n])


@pytest.mark.parametrize("average", [True, False])
def test_a_momentum_that_is_a_tensor(average):
    found = []
    for momentum in (0.75, torch.tensor(0.75)):
        params = _params()
        optimizer = training.Muon(params, average=average)
        _steps([optimizer], 3, seed=4, momenta=[momentum] * 3)
        found.append([p.detach() for p in params] + _buffers(optimizer))
    assert all(map(torch.equal, *found))
