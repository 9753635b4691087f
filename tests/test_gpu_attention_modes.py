"""A backbone with the fused attention, as programs call it: validation before training, other forms of
masks, moved and copied models."""

from __future__ import annotations

import io

import pytest
import torch

from test_gpu_attention_train import _case, _rng  # noqa: E402 (tests/ is on the path)
from test_gpu_attention_use import _batch, _grads, _model

pytestmark = pytest.mark.gpu

pytest.importorskip("transformers")


@pytest.mark.parametrize("changed", [{}, {"position_buckets": -1, "max_relative_positions": 40}],
                         ids=str)
def test_training_after_a_validation_in_inference_mode(changed):
    """A length that is first met in inference mode trains as any other."""

    ids, mask = _batch()
    want, want_grads = _grads(_model(**changed), ids, mask)
    model = _model(**changed).eval()
    with torch.inference_mode():
        model(ids, attention_mask=mask)
    got, grads = _grads(model.train(), ids, mask)
    # (As between two runs of one model: torch's products differ by 1e-6.)
    assert float((got - want).abs().max()) < 1e-5 * float(want.abs().max())
    assert set(grads) == set(want_grads)
    for name, g in grads.items():
        w = want_grads[name]
        assert float((g - w).abs().max()) <= 1e-4 * float(w.abs().max()) + 1e-6, name


@pytest.mark.parametrize("kind", ["one row for all", "one value a sequence", "queries", "keys"])
def test_masks_that_are_broadcast(kind):
    """Against torch's attention: both in fp32, so 1e-4 of the largest (rows of kept queries, and all rows
    of masks that name queries or keys)."""

    ids, mask = _batch()
    given = {"one row for all": mask[1:2], "one value a sequence": mask[:, 60:61],
             "queries": mask[:, None, :, None], "keys": mask[:, None, None, :]}[kind]
    gen = torch.Generator(device="cuda").manual_seed(6)
    hidden = torch.randn(*ids.shape, 128, device="cuda", generator=gen)
    found = []
    for attention in ("torch", "hip"):
        model = _model(attention=attention, conv_kernel_size=0).eval()
        with torch.no_grad():
            found.append(model.encoder(hidden, given).last_hidden_state)
    kept = given.bool().expand(ids.shape) if given.dim() == 2 else torch.ones_like(ids).bool()
    want, got = (x[kept] for x in found)
    assert float((got - want).abs().max()) < 1e-4 * float(want.abs().max())


def test_a_model_saved_on_the_gpu_and_loaded_on_the_cpu():
    """And brought back: its tables of relative distances are made again."""

    ids, mask = _batch()
    model = _model()
    want, want_grads = _grads(model, ids, mask)
    store = io.BytesIO()
    model.zero_grad()
    torch.save(model, store)
    store.seek(0)
    loaded = torch.load(store, weights_only=False, map_location="cpu")
    assert not any(p.is_cuda for p in loaded.parameters())
    got, grads = _grads(loaded.cuda(), ids, mask)
    assert float((got - want).abs().max()) < 1e-5 * float(want.abs().max())
    assert set(grads) == set(want_grads)
    for name, g in grads.items():
        w = want_grads[name]
        assert float((g - w).abs().max()) <= 1e-4 * float(w.abs().max()) + 1e-6, name


def test_rows_of_a_head_that_lie_more_than_2_gib_apart():
    """Tokens outermost, in a tensor of more than 2 GiB: the rows are copied."""

    from disentangled_flash.training import attention

    length, width = 600, 2_000_000
    store = torch.zeros(length, width, dtype=torch.float16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(1)
    q, k, v, dout = (torch.randn(1, length, 2, 32, device="cuda", generator=gen).half()
                     for _ in range(4))
    pk = torch.randn(2, 9, 32, device="cuda", generator=gen).half()
    lut = torch.randint(0, 9, (2 * length - 1,), device="cuda", dtype=torch.int32, generator=gen)
    views = []
    for n, t in enumerate((q, k, v)):
        store[:, 64 * n:64 * n + 64] = t[0].flatten(1)
        views.append(store[:, 64 * n:64 * n + 64].view(1, length, 2, 32))
    found = []
    for tensors in ((q, k, v), views):
        leaves = [t.detach().requires_grad_() for t in (*tensors, pk)]
        out = attention(*leaves, None, lut, 0.1)
        found.append([out.detach(), *torch.autograd.grad(out, leaves, dout)])
    assert views[0].stride(1) * 2 * (length - 1) > 1 << 31
    assert all(map(torch.equal, *found))


def test_backbone_compiled_ahead_of_time():
    """Through torch.compile's joint graph of forward and backward, two lengths one after the other (the
    second may be traced with symbolic sizes)."""

    plain, model = (_model(dropout=0.1) for _ in range(2))
    torch._dynamo.reset()
    model.compile(backend="aot_eager")
    ids, mask = _batch()
    for length in (90, 50):
        given = ids[:, :length], mask[:, :length]
        want, want_grads = _grads(plain, *given)
        got, grads = _grads(model, *given)
        assert float((got - want).abs().max()) < 1e-5 * float(want.abs().max())
        assert set(grads) == set(want_grads)
        for name, g in grads.items():
            w = want_grads[name]
            assert float((g - w).abs().max()) <= 1e-4 * float(w.abs().max()) + 1e-6, name


def test_operator_compiled_ahead_of_time():
    from disentangled_flash.training import attention

    args, dout = _case(1, 2, 100, 2, 64, torch.bfloat16)
    rng = _rng()

    def twice(*args):
        return attention(*args, p=0.1, rng=rng, site=3) * 2

    torch._dynamo.reset()
    found = []
    for call in (twice, torch.compile(twice, backend="aot_eager", fullgraph=True)):
        y = call(*args)
        found.append([y.detach(), *torch.autograd.grad(y, args[:5], dout)])
    assert all(map(torch.equal, *found))


def test_captured_step_of_a_backbone():
    """Every replay drops other places and equals the eager step of another model with that counter.  (No
    convolution; gradients of matrices only: torch's own sums record memsets, which replays do not
    repeat reliably.)"""

    ids, mask = _batch()
    model, eager = (_model(torch.bfloat16, dropout=0.2, conv_kernel_size=0) for _ in range(2))
    gen = torch.Generator(device="cuda").manual_seed(5)
    direction = torch.randn(*ids.shape, 128, device="cuda", generator=gen).bfloat16() * mask[..., None]

    def step(model):
        matrices = [p for n, p in model.named_parameters() if "proj.weight" in n]
        hidden = model(ids, attention_mask=mask).last_hidden_state
        return [hidden.detach(), *torch.autograd.grad(hidden, matrices, direction)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(model)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outputs = step(model)
    torch.cuda.current_stream().wait_stream(side)
    model.dropout_state.counter[1] = 30
    seen = []
    for n in range(4):
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outputs]
        eager.dropout_state.counter[1] = 30 + n
        want = step(eager)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            # (torch's products may be other ones in a capture: sums of bf16 in another order.)
            assert float((a.float() - b.float()).norm()) < 2e-2 * float(b.float().norm())
        seen.append(got[0])
    for n in range(4):
        assert all(not torch.equal(seen[n], seen[m]) for m in range(n))
