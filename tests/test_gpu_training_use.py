"""The training operators on the GPU in programs: transforms, checkpoints, changed modules, other
layouts and ids."""

from __future__ import annotations

import copy
import functools

import pytest
import torch
from torch import nn
from torch.autograd import forward_ad
from torch.utils.checkpoint import checkpoint

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


# ---- a model -------------------------------------------------------------------------


def _backbone(p, **over):
    from transformers import DebertaV2Config, DebertaV2Model

    torch.manual_seed(5)
    return DebertaV2Model(DebertaV2Config(
        vocab_size=100, hidden_size=64, num_hidden_layers=2, num_attention_heads=2,
        intermediate_size=128, hidden_act="gelu", type_vocab_size=2, max_position_embeddings=64,
        relative_attention=True, position_buckets=16, pos_att_type=["p2c", "c2p"],
        norm_rel_ebd="layer_norm", share_att_key=True, conv_kernel_size=3, conv_act="gelu",
        position_biased_input=True, hidden_dropout_prob=p, attention_probs_dropout_prob=p,
        **over)).cuda()


def _batch():
    gen = torch.Generator().manual_seed(2)
    return torch.randint(1, 100, (3, 24), generator=gen).cuda()


def _grads(model):
    return {n: p.grad.clone() for n, p in model.named_parameters() if p.grad is not None}


def _same_gradients(got, want):
    """torch adds the gradients of the attention's gathers with atomics, and a compiled graph may
    decompose its operators otherwise: 1000 half steps of the largest, where other masks would
    change a gradient by its own size."""

    assert got.keys() == want.keys()
    for name in want:
        size = want[name].abs().max().item()
        assert (got[name] - want[name]).abs().max().item() <= 1000 * ref.U * size, name


@pytest.mark.parametrize("compiled", [False, True])
def test_layers_in_training_in_a_backbone_in_eval_mode(compiled):
    """Each forward draws new masks, and its gradients are those of its masks."""

    from disentangled_flash import enable_deberta_training

    ids = _batch()
    model = enable_deberta_training(_backbone(0.3), seed=4).eval()
    twin = copy.deepcopy(model)
    for m in (model, twin):
        m.encoder.layer[1].train()
    call = torch.compile(model, backend="aot_eager") if compiled else model
    seen = []
    for step in range(1, 4):
        out = call(ids).last_hidden_state
        out.square().sum().backward()
        seen.append(out.detach())
        assert model.dropout_state.counter.tolist() == [4, step]
        twin.dropout_state.counter[1] = step - 1
        twin(ids).last_hidden_state.square().sum().backward()
        _same_gradients(_grads(model), _grads(twin))
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


def _gradients(model, ids, call, forwards=2):
    """Two forwards before the backward pass over both, and one by itself."""

    model.zero_grad()
    outs = [call(ids.roll(i, 0)) for i in range(forwards)]
    sum((out * (i + 1)).square().sum() for i, out in enumerate(outs)).backward()
    call(ids).square().sum().backward()
    return _grads(model)


@pytest.mark.parametrize("how", ["plain", "reentrant", "with its head", "nested", "compiled",
                                 "eval mode"])
def test_checkpointed_backbone_has_the_gradients_of_its_masks(how):
    """The same gradients as without torch.utils.checkpoint; an nn.Dropout of the program in the
    region keeps its masks too.  (Other masks would change a gradient by its own size.)"""

    from disentangled_flash import enable_deberta_training

    ids = _batch()
    grads = []
    for checkpointed in (False, True):
        model = enable_deberta_training(_backbone(0.3), seed=8).train()
        if how == "eval mode":
            model.eval().encoder.layer[1].train()
        own = nn.Dropout(0.5)
        head = nn.Linear(64, 64, device="cuda")
        leaf = torch.ones(1, device="cuda", requires_grad=True)
        call = torch.compile(model, backend="aot_eager") if how == "compiled" else model
        if how == "nested" and checkpointed:
            for layer in model.encoder.layer:
                layer.forward = functools.partial(checkpoint, layer.forward, use_reentrant=False)

        def region(ids, leaf):
            out = own(call(ids).last_hidden_state) * leaf
            return head(out) if how == "with its head" else out

        def step(ids):
            if checkpointed:
                return checkpoint(region, ids, leaf, use_reentrant=how == "reentrant")
            return region(ids, leaf)

        torch.manual_seed(9)
        grads.append(_gradients(model, ids, step))
        assert model.dropout_state.counter.tolist() == [8, 3]
    _same_gradients(grads[1], grads[0])


def test_checkpointed_backbone_without_its_generator_raises():
    from disentangled_flash import enable_deberta_training

    ids = _batch()
    model = enable_deberta_training(_backbone(0.3), seed=8).train()
    for out in (checkpoint(model, ids, use_reentrant=False, preserve_rng_state=False),
                checkpoint(model, input_ids=ids, use_reentrant=False)):
        with pytest.raises(RuntimeError, match="generator"):
            out.last_hidden_state.sum().backward()
    model(ids).last_hidden_state.sum().backward()
    assert model.dropout_state.counter.tolist() == [8, 3]


def test_output_block_whose_children_change():
    """Hooks put on later run, and what replaced a child is called.  (Between two norms in fp32:
    1e-5 is 42 half steps of values up to 4.)"""

    from disentangled_flash import enable_deberta_training

    block = enable_deberta_training(_backbone(0.0)).encoder.layer[0].output
    x, r = torch.randn(5, 128, device="cuda"), torch.randn(5, 64, device="cuda")
    want = block(x, r)
    seen = []
    handles = [child.register_forward_hook(lambda m, i, o: seen.append(type(m).__name__))
               for child in (block.LayerNorm, block.dropout)]
    torch.testing.assert_close(block(x, r), want, atol=1e-5, rtol=1e-5)
    assert seen == ["Dropout", "LayerNorm"]
    for handle in handles:
        handle.remove()
    assert torch.equal(block(x, r), want) and len(seen) == 2
    plain = block.LayerNorm
    block.LayerNorm = nn.RMSNorm(64, device="cuda")
    assert torch.equal(block(x, r), block.LayerNorm(block.dense(x) + r))
    block.LayerNorm = plain
    for drop in (nn.Identity(), nn.Dropout(1.0)):
        block.dropout = drop
        torch.testing.assert_close(block(x, r), plain(drop(block.dense(x)) + r), atol=1e-5,
                                   rtol=1e-5)


# ---- types ---------------------------------------------------------------------------

KINDS = [torch.float16, torch.bfloat16, torch.float32, torch.float64]


def _either(call):
    """The result, or None where torch refuses the types."""

    try:
        return call()
    except RuntimeError as error:
        assert "type" in str(error) or "Half" in str(error), error
        return None


def _close(got, want, half_steps):
    """Within so many half steps of the coarsest type on the way, bf16, at values up to 8."""

    assert got.dtype == want.dtype
    assert (got.double() - want.double()).abs().max().item() <= half_steps * 8 * 2.0 ** -8


@pytest.mark.parametrize("autocast", [False, True])
@pytest.mark.parametrize("weights", KINDS, ids=str)
@pytest.mark.parametrize("kind", KINDS, ids=str)
def test_norm_takes_the_types_that_torchs_takes(kind, weights, autocast):
    """The result and the gradients have the types that nn.LayerNorm's have, and their values.
    (16-bit rows beside fp32 weights, which it refuses outside autocast, are taken.)"""

    from disentangled_flash import training

    norm = nn.LayerNorm(64, device="cuda", dtype=weights)
    ours = training.LayerNorm(64, device="cuda", dtype=weights)
    results = []
    for module in (norm, ours):
        x = torch.randn(9, 64, device="cuda", generator=_gen(1)).to(kind).requires_grad_()
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
            y = _either(lambda: module(x))
        if y is not None:
            y.backward(torch.randn(9, 64, device="cuda", generator=_gen(2)).to(y.dtype))
            results.append((y, x.grad, module.weight.grad, module.bias.grad))
        else:
            results.append(None)
    if results[0] is None:
        assert results[1] is None or weights == torch.float32
        return
    for want, got in zip(*results):
        _close(got, want, 2 if torch.float64 not in (kind, weights) else 0.01)


@pytest.mark.parametrize("autocast", [False, True])
@pytest.mark.parametrize("weights", KINDS, ids=str)
@pytest.mark.parametrize("residual", KINDS, ids=str)
def test_output_block_takes_the_types_that_torchs_takes(weights, residual, autocast):
    from disentangled_flash import enable_deberta_training

    plain = _backbone(0.0).to(weights).train()
    ours = enable_deberta_training(copy.deepcopy(plain))
    results = []
    for model in (plain, ours):
        block = model.encoder.layer[0].output
        x = torch.randn(9, 128, device="cuda", generator=_gen(1)).to(weights)
        r = torch.randn(9, 64, device="cuda", generator=_gen(2)).to(residual).requires_grad_()
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
            y = _either(lambda: block(x, r))
        if y is not None:
            y.backward(torch.randn(9, 64, device="cuda", generator=_gen(3)).to(y.dtype))
            results.append((y, r.grad, block.LayerNorm.weight.grad, block.LayerNorm.bias.grad,
                            block.dense.bias.grad))
        else:
            results.append(None)
    if results[0] is None:
        assert results[1] is None
        return
    for want, got in zip(*results):
        # (A 16-bit product, sum and norm on the way; gradients of weights add 9 rows.)
        _close(got, want, 8)


@pytest.mark.parametrize("projected", [False, True])
def test_model_under_autocast(projected):
    """Hidden states keep the types that the unchanged model's have, fp32 between the blocks, and
    the values are as close to the fp32 model's as the unchanged model's are."""

    from disentangled_flash import enable_deberta_training

    ids = _batch()
    plain = _backbone(0.0, embedding_size=32) if projected else _backbone(0.0)
    plain.train()
    ours = enable_deberta_training(copy.deepcopy(plain))
    exact = plain(ids, output_hidden_states=True).hidden_states
    with torch.autocast("cuda", dtype=torch.bfloat16):
        want = plain(ids, output_hidden_states=True).hidden_states
        got = ours(ids, output_hidden_states=True).hidden_states
    got[-1].sum().backward()
    for e, w, g in zip(exact, want, got):
        assert g.dtype == w.dtype
        # A chain of two layers: three times the unchanged model's distance, at least 2 half steps.
        size = e.abs().max().item()
        assert (g - e).abs().max().item() <= 3 * (w - e).abs().max().item() + size * 2.0 ** -7


def test_model_in_double_precision():
    """Types that the operators lack stay torch's, dropout too."""

    from disentangled_flash import enable_deberta_training

    ids = _batch()
    plain = _backbone(0.0).double().train()
    ours = enable_deberta_training(copy.deepcopy(plain))
    want, got = (m(ids).last_hidden_state for m in (plain, ours))
    torch.testing.assert_close(got, want, rtol=1e-12, atol=1e-12)
    got.sum().backward()
    dropping = enable_deberta_training(_backbone(0.2).double().train())
    first, second = (dropping(ids).last_hidden_state for _ in range(2))
    assert first.dtype == torch.float64 and not torch.equal(first, second)
    first.sum().backward()


# ---- ids and addresses ---------------------------------------------------------------

BAD_IDS = {torch.int32: [-1, 30, 31, 2 ** 31 - 1, -2 ** 31, -30],
           torch.int64: [-1, 30, 31, 2 ** 31 - 1, -2 ** 31, -30, 1 << 40, -(1 << 40), 2 ** 63 - 1,
                         -2 ** 63, (1 << 32) + 4, -(1 << 32) + 4]}  # (low words inside the table)


@pytest.mark.parametrize("kind", list(BAD_IDS), ids=str)
@pytest.mark.parametrize("n", [200, 700, 9000, 40000])
@pytest.mark.parametrize("dtype,hidden", [(torch.bfloat16, 64), (torch.float32, 33)], ids=str)
def test_ids_outside_the_table_in_every_form(dtype, hidden, n, kind):
    """One launch, ranks, one run and merged runs: such ids give NaN and add to nothing, whatever
    their gradient rows hold, and neither do the padding's."""

    from disentangled_flash.training import embedding

    rows, gen = 30, _gen(n)
    ids = torch.randint(0, rows, (n,), device="cuda", generator=gen)
    outside = torch.rand(n, device="cuda", generator=gen) < 0.2
    outside[[0, n - 1]] = True  # at both ends
    bad = torch.tensor(BAD_IDS[kind], device="cuda")
    ids = torch.where(outside, bad[torch.arange(n, device="cuda") % len(bad)], ids).to(kind)
    table = _normal(gen, (rows, hidden), dtype).requires_grad_()
    y = embedding(ids, table, 2.0, 4)
    assert bool(torch.isnan(y[outside]).all())
    assert torch.equal(y[~outside], 2 * table[ids[~outside].long()])
    dy = _normal(gen, (n, hidden), dtype)
    for worst in (None, float("nan"), float("inf")):
        if worst is not None:
            dy[outside | (ids == 4)] = worst
        (grad,) = torch.autograd.grad(y, table, dy, retain_graph=True)
        ref.check(grad, ref.embedding_gradient(ids[~outside], dy[~outside], rows, 2.0, 4), "table")
        assert not grad[4].any()
    (none,) = torch.autograd.grad(embedding(bad.to(kind).repeat(n)[:n], table), table, dy)
    assert torch.equal(none, torch.zeros_like(none))


def _off(t):
    """The same values, contiguous, one element behind a 16-byte boundary."""

    store = torch.empty(t.numel() + 1, device="cuda", dtype=t.dtype)
    made = store[1:].view(t.shape).copy_(t)
    assert made.is_contiguous() and made.data_ptr() % 16 == t.element_size()
    return made


@pytest.mark.parametrize("rows", [20, 96, 2100])
@pytest.mark.parametrize("dtype", KINDS[:3], ids=str)
@pytest.mark.parametrize("which", ["rows", "weights", "all"])
def test_norm_gradients_off_the_boundaries(dtype, rows, which):
    """x, residual and dy, or the weights, behind a 16-byte boundary, at a width of whole chunks."""

    from disentangled_flash.training import layer_norm

    gen = _gen(rows)
    x, dy = (_normal(gen, (rows, 256), dtype) for _ in range(2))
    r = _normal(gen, (rows, 256), dtype, 1.3, 0.25)
    w, b = _normal(gen, (256,), dtype, 0.1, 1.0), _normal(gen, (256,), dtype, 0.1)
    want = ref.layer_norm(x, w, b, 1e-5, r, ref.factor((rows, 256), 0.2, _rng(), SITE), dy)
    if which != "weights":
        x, r, dy = _off(x), _off(r), _off(dy)
    if which != "rows":
        w, b = _off(w), _off(b)
    leaves = [t.requires_grad_() for t in (x, w, b, r)]
    y = layer_norm(x, w, b, 1e-5, r, 0.2, _rng(), SITE)
    ref.check(y.detach(), want["y"], "y")
    grads = torch.autograd.grad(y, leaves, dy)
    for name, grad in zip(("dx", "dweight", "dbias", "dresidual"), grads):
        ref.check(grad, want[name], name)


@pytest.mark.parametrize("n", [200, 700, 9000, 40000])
@pytest.mark.parametrize("dtype", KINDS[:3], ids=str)
def test_embedding_gradients_off_the_boundaries(dtype, n):
    from disentangled_flash.training import embedding

    gen = _gen(n)
    table = _off(_normal(gen, (50, 64), dtype)).requires_grad_()
    ids = torch.randint(0, 50, (n,), device="cuda", generator=gen)
    dy = _off(_normal(gen, (n, 64), dtype))
    y = embedding(ids, table, 0.5)
    (grad,) = torch.autograd.grad(y, table, dy)
    assert torch.equal(y, (table[ids].float() * 0.5).to(dtype))
    ref.check(grad, ref.embedding_gradient(ids, dy, 50, 0.5), "table")


def test_captured_and_eager_steps_in_turn():
    """Replays advance on the device; eager steps between them, of another state and of torch's own
    dropout, move torch's generator, which the graph uses too."""

    from disentangled_flash import training

    state, other = training.DropoutState(5, "cuda"), training.DropoutState(6, "cuda")
    x = torch.randn(64, 72, device="cuda")
    leaf = x.clone().requires_grad_()
    own = nn.Dropout(0.5)

    def step(state):
        state.advance()
        y = training.dropout(leaf, 0.5, state.rng, 3)
        return y.detach(), own(x), *torch.autograd.grad(y, leaf, x)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(state)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outputs = step(state)
    torch.cuda.current_stream().wait_stream(side)
    state.counter[1] = 10
    torchs = []
    for i in range(4):
        graph.replay()
        y, drawn, dx = (t.clone() for t in outputs)
        mult = ref.factor((64, 72), 0.5, torch.tensor([5, 11 + i], device="cuda"), 3).float()
        assert torch.equal(y, x * mult) and torch.equal(dx, x * mult)
        y, also, dx = step(other)
        mult = ref.factor((64, 72), 0.5, torch.tensor([6, 1 + i], device="cuda"), 3).float()
        assert torch.equal(y, x * mult) and torch.equal(dx, x * mult)
        torch.cuda.synchronize()
        torchs += [drawn, also]
    for i in range(8):  # torch's masks differ from one another
        assert all(not torch.equal(torchs[i], torchs[j]) for j in range(i))
