"""``training.Muon`` on the GPU beside ``torch.optim.Muon``."""

from __future__ import annotations

import copy

import pytest
import torch
from torch import nn

pytestmark = pytest.mark.gpu

SHAPES = ((96, 160), (160, 96), (96, 160), (200, 200))


def _params(dtype):
    gen = torch.Generator(device="cuda").manual_seed(0)
    return [nn.Parameter(torch.randn(s, device="cuda", generator=gen).to(dtype)) for s in SHAPES]


@pytest.mark.parametrize("dtype,nesterov", [(torch.float32, True), (torch.float32, False),
                                            (torch.bfloat16, True)], ids=str)
def test_average_is_torchs_rule(dtype, nesterov):
    """States bit for bit; steps of the parameters, which torch takes by bf16 products (up to 5e-2 off, and
    these 2.3e-3), to 0.1 of their size, and half a step of the parameters' dtype for each of decay and
    update.  (Without nesterov torch divides a bf16 momentum_buffer itself by its norm at every step, so
    its state is no witness there.)"""

    from disentangled_flash import training

    settings = dict(lr=0.1, weight_decay=0.1, nesterov=nesterov)
    theirs = torch.optim.Muon(_params(dtype), **settings)
    ours = training.Muon(_params(dtype), average=True, **settings)
    gen = torch.Generator(device="cuda").manual_seed(1)
    u = torch.finfo(dtype).eps / 2
    for step in range(4):
        if step == 2:  # the state goes from one to the other
            state = copy.deepcopy(theirs.state_dict())
            state["param_groups"][0]["average"] = True
            ours.load_state_dict(state)
        weights = [p.detach().clone() for p in theirs.param_groups[0]["params"]]
        grads = [torch.randn(s, device="cuda", generator=gen).to(dtype) for s in SHAPES]
        for optimizer in (theirs, ours):
            for p, w, g in zip(optimizer.param_groups[0]["params"], weights, grads):
                p.data.copy_(w)
                p.grad = g.clone()
            optimizer.step()
        for w, a, b in zip(weights, *(o.param_groups[0]["params"] for o in (theirs, ours))):
            assert torch.equal(theirs.state[a]["momentum_buffer"], ours.state[b]["momentum_buffer"])
            a, b, w = a.detach().double(), b.detach().double(), w.double()
            allowed = 0.1 * (a - w).norm() + 4 * u * w.norm()
            assert float((a - b).norm()) < float(allowed)
