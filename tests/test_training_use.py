"""CPU tests of the training operators in programs: transforms, compilers, checkpoints and modules
that change after ``enable_deberta_training``.  Kernels do not run here: operators meet fake GPU
tensors, or are recorded."""

from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad


@pytest.fixture(autouse=True)
def library():
    from disentangled_flash import _lib

    if not _lib.library_path().exists():
        pytest.skip("libdflash.so not built (run python __graft_entry__.py)")


def _fake_inputs():
    x, r = (torch.empty(3, 16, device="cuda") for _ in range(2))
    w, b = (torch.empty(16, device="cuda") for _ in range(2))
    table = torch.empty(10, 16, device="cuda")
    ids = torch.empty(3, dtype=torch.int64, device="cuda")
    rng = torch.empty(2, dtype=torch.int64, device="cuda")
    return x, r, w, b, table, ids, rng


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("which", range(6))
def test_tangents_are_refused(which, requires_grad):
    """Forward-mode derivatives are not implemented: a tangent must not be lost."""

    from disentangled_flash import training

    with FakeTensorMode(), forward_ad.dual_level():
        x, r, w, b, table, ids, rng = _fake_inputs()

        def dual(t):
            return forward_ad.make_dual(t.requires_grad_(requires_grad), torch.ones_like(t))

        call = (
            lambda: training.dropout(dual(x), 0.5, rng),
            lambda: training.layer_norm(dual(x), w, b, 1e-5),
            lambda: training.layer_norm(x, dual(w), b, 1e-5),
            lambda: training.layer_norm(x, w, dual(b), 1e-5),
            lambda: training.layer_norm(x, w, b, 1e-5, dual(r)),
            lambda: training.embedding(ids, dual(table)),
        )[which]
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call()


def test_tangents_through_functions_are_refused():
    from disentangled_flash import training

    with FakeTensorMode():
        x, r, w, b, table, ids, rng = _fake_inputs()
        for call, at in ((lambda t: training.dropout(t, 0.5, rng), x),
                         (lambda t: training.layer_norm(t, w, b, 1e-5), x),
                         (lambda t: training.embedding(ids, t), table)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.func.jvp(call, (at,), (torch.ones_like(at),))
