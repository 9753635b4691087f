"""``training.attention`` and ``training.orthogonalize`` as a program uses them: layouts, streams, graphs,
memory, the modules and a training step with all of them."""

from __future__ import annotations

import math

import pytest
import torch

import attention_reference as ref  # noqa: E402 (tests/ is on the path)
import training_reference as common
from test_gpu_attention_train import DTYPES, SITE, _case, _check, _gradients, _rng

pytestmark = pytest.mark.gpu


@pytest.fixture(params=list(DTYPES))
def dtype(request):
    return DTYPES[request.param]


def _run(args, dout, p=0.1, site=SITE):
    from disentangled_flash.training import attention

    y = attention(*args, p=p, rng=_rng(), site=site)
    return {"out": y.detach(), **_gradients(y, args[:5], dout)}


def _same(a, b):
    assert set(a) == set(b)
    for name in a:
        assert torch.equal(a[name], b[name]), name


def test_calls_are_repeatable(dtype):
    args, dout = _case(1, 3, 150, 2, 64, dtype)
    _same(_run(args, dout), _run(args, dout))


def test_layouts(dtype):
    """Slices of a fused projection, transposed and expanded tensors, rows off 16-byte boundaries."""

    (q, k, v, pk, pq, lut, scale, mask), dout = _case(2, 2, 70, 3, 32, dtype)
    want = _run([q, k, v, pk, pq, lut, scale, mask], dout)

    def given(tensors):
        leaves = [t.detach().requires_grad_() for t in tensors]
        assert [t.stride() for t in leaves] == [t.stride() for t in tensors]
        return [*leaves, lut, scale, mask]

    joined = torch.cat([t.detach().flatten(2) for t in (q, k, v)], -1)
    views = [x.view(2, 70, 3, 32) for x in joined.split(96, -1)]
    rows = [t.detach().transpose(0, 1).contiguous().transpose(0, 1) for t in (pk, pq)]
    _same(_run(given([*views, *rows]), dout), want)
    turned = [t.detach().permute(3, 1, 0, 2).contiguous().permute(2, 1, 3, 0) for t in (q, k, v)]
    _same(_run(given([*turned, pk, pq]), dout), want)
    heads = [t.detach().transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    _same(_run(given([*heads, pk, pq]), dout.transpose(1, 2).contiguous().transpose(1, 2)), want)
    shifted = []
    for t in (q, k, v, pk, pq):
        store = torch.empty(t.numel() + 1, dtype=dtype, device="cuda")[1:]
        shifted.append(store.copy_(t.detach().flatten()).view(t.shape))
    _same(_run(given(shifted), dout), want)
    one = q.detach()[:1].expand(2, -1, -1, -1)
    whole = one.contiguous()
    _same(_run(given([one, k, v, pk, pq]), dout), _run(given([whole, k, v, pk, pq]), dout))
    _same(_run([q, k, v, pk, pq, lut, scale, mask.to(torch.uint8) * 7], dout), want)


def test_broadcast_inputs_collect_their_gradient():
    args, dout = _case(3, 3, 40, 2, 64, torch.float32)
    leaf = args[1].detach()[:1].clone().requires_grad_()
    args[1] = leaf.expand(3, -1, -1, -1)
    y = _forward(args)
    (got,) = torch.autograd.grad(y, leaf, dout)
    whole = args[1].detach().requires_grad_()
    args[1] = whole
    (parts,) = torch.autograd.grad(_forward(args), whole, dout)
    assert torch.allclose(got, parts.sum(0, keepdim=True), rtol=1e-6, atol=1e-6)


def _forward(args, p=0.1):
    from disentangled_flash.training import attention

    return attention(*args, p=p, rng=_rng(), site=SITE)


def test_same_tensor_as_query_key_and_value():
    args, dout = _case(4, 2, 40, 2, 64, torch.float32)
    x = args[0]
    y = _forward([x, x, x, *args[3:]])
    (got,) = torch.autograd.grad(y, x, dout)
    parts = [x.detach().clone().requires_grad_() for _ in range(3)]
    grads = torch.autograd.grad(_forward([*parts, *args[3:]]), parts, dout)
    assert torch.allclose(got, sum(grads), rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("wanted", ["q", "k", "v", "pk", "pq", "qv", "k pk", "none"])
def test_gradients_one_by_one(wanted):
    args, dout = _case(5, 2, 50, 2, 64, torch.bfloat16)
    want = _run(args, dout)
    names = dict(zip(("q", "k", "v", "pk", "pq"), range(5)))
    chosen = [] if wanted == "none" else [n for n in names if n in wanted.split() or wanted == "qv"
                                          and n in "qv"]
    for name, at in names.items():
        args[at] = args[at].detach().requires_grad_(name in chosen)
    y = _forward(args)
    assert torch.equal(y, want["out"]) and y.requires_grad == bool(chosen)
    if chosen:
        got = _gradients(y, args[:5], dout)
        assert len(got) == len(chosen)
        for name, value in got.items():
            assert torch.equal(value, want[name]), name


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_padded_places_may_hold_anything(dtype, bad):
    """Kept rows and all gradients but dV's share of padded queries see nothing of it."""

    args, dout = _case(6, 3, 100, 2, 64, dtype, mask="holes")
    mask = args[7]
    dout[~mask] = 0
    want = _run(args, dout)
    with torch.no_grad():
        for t in args[:3]:
            t[~mask] = bad
    got = _run(args, dout)
    assert torch.equal(got["out"][mask], want["out"][mask])
    assert bool(torch.isfinite(got["out"]).all())
    for name in ("dq", "dk", "dv"):
        assert torch.equal(got[name][mask], want[name][mask]), name
        assert bool(torch.isfinite(got[name]).all()), name
    for name in ("dpos_key", "dpos_query"):
        assert torch.equal(got[name], want[name]), name


def test_sequences_stay_apart(dtype):
    args, dout = _case(7, 3, 90, 2, 32, dtype)
    want = _run(args, dout, p=0.0)
    with torch.no_grad():
        for t in args[:3]:
            t[1] = float("nan")
    got = _run(args, dout, p=0.0)
    for n in (0, 2):
        for name in ("out", "dq", "dk", "dv"):
            assert torch.equal(got[name][n], want[name][n]), name
    assert bool(torch.isnan(got["out"][1][args[7][1]]).all())


def test_of_nothing(dtype):
    from disentangled_flash.training import attention

    for shape in ((0, 5, 2, 64), (2, 0, 2, 64)):
        q, k, v = (torch.randn(shape, device="cuda", dtype=dtype).requires_grad_()
                   for _ in range(3))
        pk = torch.randn(2, 3, 64, device="cuda", dtype=dtype).requires_grad_()
        lut = torch.zeros(max(0, 2 * shape[1] - 1), dtype=torch.int32, device="cuda")
        y = attention(q, k, v, pk, None, lut, 0.1, p=0.1, rng=_rng())
        assert y.shape == shape
        grads = torch.autograd.grad(y.sum(), (q, k, v, pk))
        assert [g.shape for g in grads] == [q.shape] * 3 + [pk.shape]
        assert bool((grads[3] == 0).all())


def test_extreme_scores(dtype):
    """Scores of some hundreds: probabilities of 0 and 1, nothing that is not finite."""

    args, dout = _case(8, 2, 70, 2, 64, dtype)
    with torch.no_grad():
        args[0].mul_(30)
        args[3].mul_(4)
    _check((args, dout), p=0.0)


def test_large_batches_are_taken_in_parts():
    """More scores than the backward pass takes at a time (2 GiB): each sequence is what it is alone,
    and the tables' gradients are the sum."""

    b, length, h, d = 3, 4096, 24, 32
    args, dout = _case(9, b, length, h, d, torch.bfloat16, mask="ragged")
    whole = _run(args, dout, p=0.0)
    sums = {"dpos_key": 0, "dpos_query": 0}
    for n in range(b):
        one = [t.detach()[n:n + 1].requires_grad_() for t in args[:3]] + args[3:7] \
            + [args[7][n:n + 1]]
        part = _run(one, dout[n:n + 1], p=0.0)
        for name in ("out", "dq", "dk", "dv"):
            assert torch.equal(whole[name][n], part[name][0]), name
        for name in sums:
            sums[name] = sums[name] + part[name].double()
    for name, value in sums.items():
        # Each is rounded to bf16: half a step of each of the three parts and of the sum.
        size = value.abs().max()
        assert float((whole[name].double() - value).abs().max()) < 4 * 2 ** -8 * float(size), name


def test_long_sequences_are_taken_by_heads():
    """One pair of a sequence of 16384 takes 512 MiB: four heads at a time."""

    b, length, h, d = 1, 16384, 6, 32
    args, dout = _case(10, b, length, h, d, torch.bfloat16, mask="none")
    whole = _run(args, dout, p=0.0)
    for n in (0, 3, 4, 5):
        one = [t.detach()[:, :, n:n + 1].requires_grad_() for t in args[:3]] \
            + [t.detach()[n:n + 1].requires_grad_() for t in args[3:5]] + args[5:]
        part = _run(one, dout[:, :, n:n + 1], p=0.0)
        for name in ("out", "dq", "dk", "dv"):
            assert torch.equal(whole[name][:, :, n], part[name][:, :, 0]), name
        for name in ("dpos_key", "dpos_query"):
            assert torch.equal(whole[name][n], part[name][0]), name


def test_memory_stays_near_one_score_tensor():
    """Forward and what is kept: outputs, statistics, one bit a probability.  Backward: G in the dtype
    and the partial sums."""

    args, dout = _case(11, 8, 1024, 8, 64, torch.bfloat16, mask="none")
    pairs = 8 * 8 * 1024 * 1024
    _run(args, dout)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    y = _forward(args)
    kept = torch.cuda.memory_allocated() - before
    # The output, what its 16 bits left off, a bit a probability and a statistic a row.
    assert kept < 2 * y.nbytes + pairs / 8 + (1 << 20) + 8 * 8 * 1024 * 4
    grads = _gradients(y, args[:5], dout)
    peak = torch.cuda.max_memory_allocated() - before - kept
    assert peak < 2 * pairs + 4 * y.nbytes + (160 << 20)
    assert grads


def test_streams_and_current_device():
    args, dout = _case(12, 2, 130, 2, 64, torch.bfloat16)
    want = _run(args, dout)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        junk = torch.full((1 << 26,), 1.0, device="cuda")
        for _ in range(10):
            junk.mul_(1.0001)
        late = [t.detach().clone().requires_grad_() for t in args[:5]] + args[5:]
        got = _run(late, dout)
    torch.cuda.current_stream().wait_stream(side)
    _same(got, want)


def test_captured_step_equals_the_eager_one():
    """Forward, backward and an update, captured: every replay draws other masks and equals the
    eager call with its step."""

    from disentangled_flash.training import attention, orthogonalize

    args, dout = _case(13, 2, 100, 2, 64, torch.bfloat16)
    leaves = [t.detach().clone().requires_grad_() for t in args[:5]]
    rng = _rng()

    def step():
        y = attention(*leaves, *args[5:], p=0.2, rng=rng, site=SITE)
        grads = torch.autograd.grad(y, leaves, dout)
        return [y.detach(), *grads, orthogonalize(grads[0].flatten(2))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
        rng[1:] += 1
    seen = []
    for n in range(4):
        rng.copy_(_rng(step=20 + n))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        rng.copy_(_rng(step=20 + n))
        other = _case(20 + n, 1, 64, 2, 64, torch.bfloat16)
        _run(*other)  # eager work of the program's own between the replays
        for a, b in zip(got, step()):
            assert torch.equal(a, b)
        seen.append(got[0])
    assert not torch.equal(seen[0], seen[1])


def test_two_graphs_have_workspaces_of_their_own():
    args, dout = _case(14, 2, 200, 2, 64, torch.bfloat16)
    other, other_dout = _case(15, 2, 140, 2, 64, torch.bfloat16)
    want = [_run(args, dout), _run(other, other_dout)]
    graphs, outs = [], []
    for a, g in ((args, dout), (other, other_dout)):
        leaves = [t.detach().clone().requires_grad_() for t in a[:5]] + a[5:]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_run_captured(leaves, g))
        graphs.append(graph)
    for _ in range(3):
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for got, expected in zip(outs, want):
            _same(got, expected)


_FIXED = {}


def _run_captured(args, dout):
    from disentangled_flash.training import attention

    rng = _FIXED.setdefault("rng", None)
    y = attention(*args, p=0.1, rng=rng, site=SITE)
    return {"out": y.detach(), **_gradients(y, args[:5], dout)}


@pytest.fixture(autouse=True)
def _fixed_rng():
    _FIXED["rng"] = _rng()  # (made outside the capture)
    yield


def test_second_derivatives_raise():
    args, dout = _case(16, 1, 20, 1, 32, torch.float32)
    y = _forward(args)
    (dq,) = torch.autograd.grad(y, args[0], dout, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        dq.sum().backward()


def test_operators_called_by_name_refuse_what_does_not_fit():
    from disentangled_flash import training

    args, dout = _case(17, 2, 20, 2, 64, torch.bfloat16)
    args = [t.detach() if isinstance(t, torch.Tensor) else t for t in args]
    q, k, v, pk, pq, lut, scale, mask = args
    training._load()
    op = torch.ops.disentangled_flash
    good = [q, k, v, pk, pq, lut, mask, None, scale, 0.0, 0]
    want = op.attention(*good)
    assert want.shape == q.shape
    for at, value in ((0, q.flatten(2)), (1, k[:, 1:]), (2, v.float()), (3, pk[:1]), (3, pk.float()),
                      (4, pq[:, 1:]), (5, lut[1:]), (5, lut.long()), (5, lut[::2]), (6, mask[:1]),
                      (6, mask.float()), (6, mask.t().contiguous().t()), (1, k.cpu()), (5, lut.cpu()),
                      (6, mask.cpu()), (9, 0.5), (10, -1)):
        bad = list(good)
        bad[at] = value
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            op.attention(*bad)
    out, low, lse, bits = op.attention_train(*good[:7], _rng(), scale, 0.5, 0)
    back = [dout, out, low, lse, bits, q, k, v, pk, pq, lut, mask, scale, 0.5, True, True]
    op.attention_backward(*back)
    for at, value in ((0, dout[:1]), (0, dout.transpose(1, 2)), (1, out.float()), (2, low[:1]),
                      (2, low.float()), (3, lse[:1]), (4, bits[1:]), (11, mask[:1])):
        bad = list(back)
        bad[at] = value
        with pytest.raises((ValueError, RuntimeError)):
            op.attention_backward(*bad)
    for bad in (torch.zeros(3, device="cuda"), torch.zeros(2, 3, 4, device="cuda").mT,
                torch.zeros(2, 0, 4, device="cuda")):
        with pytest.raises(ValueError):
            op.orthogonalize(bad, 5, 1.0, 1.0, 1.0, 0.0)
    with pytest.raises(ValueError):
        op.orthogonalize(torch.zeros(2, 3, 4, device="cuda"), 0, 1.0, 1.0, 1.0, 0.0)
    assert torch.equal(op.attention(*good), want)


# ---- a backbone -----------------------------------------------------------------------


transformers = pytest.importorskip("transformers")


def _model(dtype=torch.float32, attention="hip", dropout=0.0, layers=2, **changed):
    from disentangled_flash import enable_deberta_training

    torch.manual_seed(0)
    settings = dict(vocab_size=100, hidden_size=128, num_hidden_layers=layers,
                    num_attention_heads=2, intermediate_size=192, relative_attention=True,
                    position_buckets=32, max_position_embeddings=128, max_relative_positions=-1,
                    type_vocab_size=0, pos_att_type=["c2p", "p2c"], share_att_key=True,
                    norm_rel_ebd="layer_norm", position_biased_input=False, conv_kernel_size=3,
                    hidden_dropout_prob=dropout, attention_probs_dropout_prob=dropout,
                    conv_act="gelu")
    config = transformers.DebertaV2Config(**{**settings, **changed})
    model = transformers.DebertaV2Model(config).cuda().to(dtype).train()
    return enable_deberta_training(model, seed=3, attention=attention)


def _batch(b=3, length=90):
    gen = torch.Generator().manual_seed(1)
    ids = torch.randint(0, 100, (b, length), generator=gen).cuda()
    kept = torch.tensor([length, 47, 1])[:b, None]
    return ids, (torch.arange(length)[None] < kept).long().cuda()


def _grads(model, ids, mask):
    model.zero_grad()
    hidden = model(ids, attention_mask=mask).last_hidden_state
    # A fixed direction, over the kept tokens: what a loss sees.  (The sum of squares would not do:
    # a LayerNorm's output has the same one whatever its input, so its gradient is rounding alone.)
    gen = torch.Generator(device="cuda").manual_seed(5)
    direction = torch.randn(hidden.shape, device="cuda", generator=gen)
    (hidden.float() * mask[..., None] * direction).sum().backward()
    return hidden.detach(), {n: p.grad for n, p in model.named_parameters() if p.grad is not None}


@pytest.mark.parametrize("dropout", [0.0, 0.1])
@pytest.mark.parametrize("changed", [{}, {"share_att_key": False, "pos_att_type": ["p2c", "c2p"]},
                                     {"pos_att_type": ["c2p"]}], ids=str)
def test_backbone_is_torchs_in_fp32(dropout, changed):
    """Outputs and every parameter's gradient, against the same model with torch's attention (and
    the same dropped places): both in fp32, so 1e-4 of the largest."""

    ids, mask = _batch()
    want, want_grads = _grads(_model(attention="torch", dropout=dropout, **changed), ids, mask)
    got, grads = _grads(_model(dropout=dropout, **changed), ids, mask)
    kept = mask.bool()
    assert float((got - want)[kept].abs().max()) < 1e-4 * float(want.abs().max())
    assert set(grads) == set(want_grads)
    for name, g in grads.items():
        w = want_grads[name]
        assert float((g - w).abs().max()) <= 1e-4 * float(w.abs().max()) + 1e-6, name


@pytest.mark.parametrize("how", ["reentrant", "other", "compiled", "autocast"])
def test_backbone_checkpointed_compiled_and_under_autocast(how):
    ids, mask = _batch()
    plain = _model(dropout=0.1)
    if how == "autocast":
        with torch.autocast("cuda", dtype=torch.bfloat16):
            hidden = plain(ids, attention_mask=mask).last_hidden_state
            hidden.float().pow(3).sum().backward()
        assert all(p.grad is not None and bool(torch.isfinite(p.grad).all())
                   for n, p in plain.named_parameters())
        return
    # (Reentrant checkpoints of layers want position rows without a graph of their own, whatever the
    # attention: each layer would free that graph for the next.)
    changed = {"norm_rel_ebd": "none"} if how == "reentrant" else {}
    if changed:
        plain = _model(dropout=0.1, **changed)
    want, want_grads = _grads(plain, ids, mask)
    model = _model(dropout=0.1, **changed)
    if how == "compiled":
        model.compile(backend="eager")
    else:
        model.gradient_checkpointing_enable({"use_reentrant": how == "reentrant"})
    got, grads = _grads(model, ids, mask)
    # (Torch's convolution and products of this model differ by 1e-6 from run to run; other
    # masks would differ by whole values.)
    assert float((got - want).abs().max()) < 1e-5 * float(want.abs().max())
    for name, g in grads.items():
        w = want_grads[name]
        assert float((g - w).abs().max()) <= 1e-4 * float(w.abs().max()) + 1e-6, name


def test_training_steps_with_muon():
    """The operators of a step together: two micro-batches, gradients that add up, Muon for the
    projections beside SGD for the rest, against the same step from its parts."""

    from disentangled_flash.training import NEWTON_SCHULZ, Muon, orthogonalize, split_parameters

    model = _model(torch.bfloat16, dropout=0.1)
    matrices, rest = split_parameters(model)
    names = {id(p): n for n, p in model.named_parameters()}
    muon = Muon(matrices, lr=0.02, weight_decay=0.1, adjust_lr_fn="match_rms_adamw")
    sgd = torch.optim.SGD(rest, lr=1e-3)
    ids, mask = _batch()
    buffers = {}
    for step in range(3):
        model.zero_grad()
        for half in (slice(0, 2), slice(2, 3)):
            hidden = model(ids[half], attention_mask=mask[half]).last_hidden_state
            (hidden * mask[half][..., None]).float().pow(3).mean().backward()
        want = {}
        by_shape = {}
        for p in matrices:
            if p.grad is not None:
                by_shape.setdefault(p.shape, []).append(p)
        for shape, params in by_shape.items():
            updates = []
            for p in params:
                b = buffers.setdefault(id(p), torch.zeros_like(p, requires_grad=False))
                b.mul_(0.95).add_(p.grad)
                updates.append(torch.add(p.grad, b, alpha=0.95))
            turned = orthogonalize(torch.stack(updates), 5, NEWTON_SCHULZ, 1e-7)
            for p, o in zip(params, turned):
                lr = 0.02 * 0.2 * math.sqrt(max(shape))
                want[id(p)] = p.detach().double() * (1 - 0.02 * 0.1) - lr * o.double()
        muon.step()
        sgd.step()
        for p in matrices:
            if id(p) in want:
                w = want[id(p)]
                # Half a step of the decayed weight and of the result (a quarter more for w in
                # place of either).
                off = (p.detach().double() - w).abs().max()
                assert float(off) < 2.5 * 2 ** -8 * float(w.abs().max()), names[id(p)]
        assert all(bool(torch.isfinite(p).all()) for p in model.parameters())


def test_trained_model_goes_on_to_inference():
    from disentangled_flash import optimize_deberta

    ids, mask = _batch()
    model = _model()
    _grads(model, ids, mask)
    model.eval()
    with torch.no_grad():
        want = model(ids, attention_mask=mask).last_hidden_state
        optimize_deberta(model, sequence_lengths=[90])
        model.encoder.activate_shape(90)
        got = model(ids, attention_mask=mask).last_hidden_state
    kept = mask.bool()
    assert float((got - want)[kept].abs().max()) < 1e-4 * float(want.abs().max())


def test_transforms():
    """vmap over calls, with an rng for every sample; no transforms that differentiate."""

    from disentangled_flash.training import attention

    args, dout = _case(31, 4, 33, 2, 32, torch.bfloat16, mask="none")
    q, k, v, pk, pq = [t.detach() for t in args[:5]]
    lut, scale = args[5:7]
    rngs = torch.stack([_rng() + i for i in range(4)])

    def one(q, k, v, r):
        return attention(q[None], k[None], v[None], pk, pq, lut, scale, p=0.3, rng=r, site=SITE)[0]

    got = torch.func.vmap(one)(q, k, v, rngs)
    for i in range(4):
        assert torch.equal(got[i], one(q[i], k[i], v[i], rngs[i]))
    with pytest.raises(ValueError, match="rng"):
        torch.func.vmap(lambda t: one(t, k[0], v[0], rngs[0]))(q)

    def loss(q, pk):
        return (attention(q, k, v, pk, pq, lut, scale) * dout).float().sum()

    with pytest.raises(RuntimeError):
        torch.func.grad(loss, argnums=(0, 1))(q, pk)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: attention(t, k, v, pk, pq, lut, scale), (q,), (q,))
    with torch.inference_mode():
        assert torch.equal(attention(q, k, v, pk, pq, lut, scale),
                           attention(q.clone().requires_grad_(), k, v, pk, pq, lut, scale))


def test_muon_takes_a_rate_that_is_a_tensor():
    from disentangled_flash import training

    values = torch.randn(24, 40, device="cuda")
    found = []
    for lr in (0.1, torch.tensor(0.1)):
        p = torch.nn.Parameter(values.clone())
        p.grad = torch.ones_like(p).cumsum(0).cumsum(1)
        training.Muon([p], lr=lr).step()
        found.append(p.detach())
    assert torch.allclose(found[0], found[1], rtol=1e-6, atol=1e-7)  # 0.1 in 32 bits
    assert not torch.equal(found[0], values)
