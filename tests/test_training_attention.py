"""CPU tests of the fused attention's place in a Hugging Face backbone and of Muon: what runs without
a GPU must be torch's own, bit for bit, and the host logic is tested with the operator replaced."""

from __future__ import annotations

import copy
import io
import math

import pytest
import torch
from torch import nn

transformers = pytest.importorskip("transformers")

from disentangled_flash import enable_deberta_training, training  # noqa: E402


def _model(**changed):
    torch.manual_seed(0)
    settings = dict(vocab_size=60, hidden_size=64, num_hidden_layers=2, num_attention_heads=2,
                    intermediate_size=96, relative_attention=True, position_buckets=8,
                    max_position_embeddings=40, max_relative_positions=-1, type_vocab_size=0,
                    pos_att_type=["c2p", "p2c"], share_att_key=True, norm_rel_ebd="layer_norm",
                    position_biased_input=False, conv_kernel_size=3, conv_act="gelu")
    config = transformers.DebertaV2Config(**{**settings, **changed})
    return transformers.DebertaV2Model(config)


def _inputs(b=3, length=11):
    gen = torch.Generator().manual_seed(1)
    ids = torch.randint(0, 60, (b, length), generator=gen)
    mask = (torch.arange(length)[None] < torch.tensor([[length], [6], [1]])[:b]).long()
    return ids, mask


@pytest.mark.parametrize("mask", ["padding", "none"])
@pytest.mark.parametrize("attentions", [False, True])
def test_on_the_cpu_it_is_torchs(mask, attentions):
    model = _model().eval()
    ids, padding = _inputs()
    given = {"padding": padding, "none": None}[mask]
    want = model(ids, attention_mask=given, output_attentions=attentions)
    keys = list(model.state_dict())
    fused = enable_deberta_training(model, attention="hip").eval()
    assert list(fused.state_dict()) == keys
    got = fused(ids, attention_mask=given, output_attentions=attentions)
    assert torch.equal(got.last_hidden_state, want.last_hidden_state)
    if attentions:
        assert all(map(torch.equal, got.attentions, want.attentions))


def _pairs(mask):
    """A mask of pairs, which only the encoder itself takes (and not its convolution)."""

    return (mask[:, None, :] * mask[:, :, None]).tril()


def test_masks_of_pairs_are_torchs():
    model = _model(conv_kernel_size=0).eval()
    _, mask = _inputs()
    hidden = torch.randn(3, 11, 64, generator=torch.Generator().manual_seed(2))
    want = model.encoder(hidden, _pairs(mask)).last_hidden_state
    enable_deberta_training(model, attention="hip").eval()
    assert torch.equal(model.encoder(hidden, _pairs(mask)).last_hidden_state, want)


def test_default_leaves_the_attention():
    model = enable_deberta_training(_model())
    for layer in model.encoder.layer:
        assert type(layer.attention.self).__module__.startswith("transformers.")
    assert "get_attention_mask" not in model.encoder.__dict__
    with pytest.raises(ValueError):
        enable_deberta_training(_model(), attention="cuda")


def test_copies_and_pickles():
    model = enable_deberta_training(_model(), attention="hip").eval()
    ids, mask = _inputs()
    want = model(ids, attention_mask=mask).last_hidden_state
    store = io.BytesIO()
    torch.save(model, store)
    store.seek(0)
    for other in (copy.deepcopy(model), torch.load(store, weights_only=False)):
        assert other.encoder.__dict__["get_attention_mask"].encoder is other.encoder
        assert torch.equal(other(ids, attention_mask=mask).last_hidden_state, want)


def test_hooks_and_other_classes_are_refused():
    model = _model()
    model.encoder.layer[1].attention.self.register_forward_hook(lambda *a: None)
    with pytest.raises(TypeError, match="attention"):
        enable_deberta_training(model, attention="hip")
    assert not hasattr(model, "dropout_state")  # and nothing was changed
    assert type(model.encoder.layer[0].attention.self).__module__.startswith("transformers.")


@pytest.fixture
def calls(monkeypatch):
    """The fused path on the CPU, with the operator's definition in torch in the operator's place."""

    seen = []

    def attention(query, key, value, pos_key, pos_query, places, scale, mask=None, p=0.0, rng=None,
                  site=0):
        seen.append(dict(p=p, site=site, rng=rng, mask=mask))
        assert p == 0.0 or rng is not None
        q, k, v = (t.transpose(1, 2) for t in (query, key, value))
        length = q.shape[2]
        at = torch.arange(length)
        slot = places.long()[at[:, None] - at[None] + length - 1]
        s = q @ k.mT
        if pos_key is not None:
            s = s + (q @ pos_key.mT).gather(3, slot.expand_as(s))
        if pos_query is not None:
            s = s + (k @ pos_query.mT).gather(3, slot.t().expand_as(s)).mT
        pair = mask[:, None, :, None] & mask[:, None, None, :]
        s = (s * scale).masked_fill(~pair, torch.finfo(s.dtype).min)
        return (torch.softmax(s, -1) @ v).transpose(1, 2).contiguous()

    monkeypatch.setattr(training, "attention", attention)
    monkeypatch.setattr(training, "_on_gpu", lambda x: x.dim() == 3)
    monkeypatch.setattr(training, "layer_norm", lambda x, w, b, eps, residual=None, p=0.0, rng=None,
                        site=0: nn.functional.layer_norm(
                            x if residual is None else x + residual, w.shape, w, b, eps))
    monkeypatch.setattr(training, "dropout", lambda x, p, rng, site=0: x)
    return seen


@pytest.mark.parametrize("changed", [
    {}, {"share_att_key": False}, {"pos_att_type": ["c2p"]}, {"pos_att_type": ["p2c"]},
    {"pos_att_type": []}, {"relative_attention": False}, {"position_buckets": -1},
    {"hidden_size": 128, "num_attention_heads": 1}], ids=str)
def test_fused_forward_is_the_module(calls, changed):
    """Slots, terms, projections and scale, against the module itself."""

    model = _model(**changed).eval()
    ids, mask = _inputs()
    want = model(ids, attention_mask=mask).last_hidden_state
    fused = enable_deberta_training(model, attention="hip").eval()
    got = fused(ids, attention_mask=mask).last_hidden_state
    assert len(calls) == 2 and all(c["p"] == 0.0 for c in calls)
    assert all(torch.equal(c["mask"], mask.bool()) for c in calls)
    kept = mask.bool()
    assert torch.allclose(got[kept], want[kept], atol=2e-6)


def test_fused_dropout_is_the_modules(calls):
    model = enable_deberta_training(_model(), attention="hip").train()
    ids, mask = _inputs()
    model(ids, attention_mask=mask)
    sites = [layer.attention.self.dropout.site for layer in model.encoder.layer]
    assert [c["site"] for c in calls] == sites and len(set(sites)) == 2
    assert all(c["p"] == 0.1 and c["rng"].tolist() == [0, 1] for c in calls)


def test_what_the_fused_forward_lacks_goes_to_torch(calls):
    ids, mask = _inputs()
    model = enable_deberta_training(_model(conv_kernel_size=0), attention="hip").eval()
    model(ids, attention_mask=mask, output_attentions=True)
    hidden = torch.randn(3, 11, 64)
    model.encoder(hidden, _pairs(mask))
    model.encoder(hidden, mask, relative_pos=model.encoder.layer[0].attention.self.pos_ebd_size
                  * torch.ones(1, 11, 11, dtype=torch.long))
    assert not calls
    attention = model.encoder.layer[0].attention.self
    attention.dropout.register_forward_hook(lambda *a: None)
    model(ids, attention_mask=mask)
    assert len(calls) == 1  # the other layer
    attention.dropout = nn.Dropout(0.1)
    model(ids, attention_mask=mask)
    assert len(calls) == 2
    small = enable_deberta_training(_model(hidden_size=32, num_attention_heads=2),
                                    attention="hip").eval()
    small(ids, attention_mask=mask)  # heads of 16
    assert len(calls) == 2


# ---- Muon ------------------------------------------------------------------------------


def _exact(update, steps=5, coefficients=training.NEWTON_SCHULZ, eps=1e-7):
    a, b, c = coefficients
    x = update.double()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    for _ in range(steps):
        s = x @ x.mT
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.mT if tall else x


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("adjust", [None, "original", "match_rms_adamw"])
def test_muon_steps(monkeypatch, nesterov, adjust):
    shapes = []

    def orthogonalize(update, steps, coefficients, eps):
        shapes.append(tuple(update.shape))
        return _exact(update, steps, coefficients, eps)

    monkeypatch.setattr(training, "orthogonalize", orthogonalize)
    monkeypatch.setattr(training, "_check_floating", lambda *a: None)  # on the CPU, in 64 bits
    gen = torch.Generator().manual_seed(0)

    def normal(*shape):
        return torch.randn(shape, generator=gen, dtype=torch.float64)

    params = [nn.Parameter(normal(*s)) for s in ((6, 4), (3, 7), (6, 4), (5, 5))]
    want = [p.detach().clone() for p in params]
    buffers = [torch.zeros_like(p) for p in want]
    optimizer = training.Muon(params, lr=0.1, weight_decay=0.2, momentum=0.9, nesterov=nesterov,
                              adjust_lr_fn=adjust)
    for step in range(3):
        grads = [normal(*p.shape) for p in params]
        for n, (p, g) in enumerate(zip(params, grads)):
            p.grad = None if step == 1 and n == 3 else g
        shapes.clear()
        optimizer.step()
        assert sorted(shapes) == ([(1, 3, 7), (1, 5, 5), (2, 6, 4)] if step != 1
                                  else [(1, 3, 7), (2, 6, 4)])
        for n, g in enumerate(grads):
            if step == 1 and n == 3:
                continue
            buffers[n] = 0.9 * buffers[n] + g
            update = g + 0.9 * buffers[n] if nesterov else buffers[n]
            m, k = g.shape
            ratio = 0.2 * math.sqrt(max(m, k)) if adjust == "match_rms_adamw" \
                else math.sqrt(max(1, m / k))
            want[n] = want[n] * (1 - 0.1 * 0.2) - 0.1 * ratio * _exact(update)
        for p, w in zip(params, want):
            assert torch.allclose(p, w, rtol=1e-12, atol=1e-12)
    state = optimizer.state_dict()
    other = training.Muon(params, lr=0.3)
    other.load_state_dict(state)
    assert other.param_groups[0]["lr"] == 0.1
    assert torch.equal(other.state[params[0]]["momentum_buffer"], buffers[0])


def test_muon_refusals():
    matrix = nn.Parameter(torch.zeros(3, 4))
    for settings in ({"lr": -1.0}, {"momentum": 1.0}, {"momentum": -0.1}, {"weight_decay": -1.0},
                     {"adjust_lr_fn": "other"}):
        with pytest.raises(ValueError):
            training.Muon([matrix], **settings)
    with pytest.raises(ValueError, match="matrices"):
        training.Muon([nn.Parameter(torch.zeros(3))])
    optimizer = training.Muon([matrix])
    for bad in (torch.zeros(3), torch.zeros(2, 3, 4), torch.zeros(0, 4)):
        with pytest.raises(ValueError, match="matrices"):
            optimizer.add_param_group({"params": [nn.Parameter(bad)]})
    assert len(optimizer.param_groups) == 1
    matrix.grad = torch.ones(3, 4)
    with pytest.raises(RuntimeError, match="GPU"):
        optimizer.step()
    assert not optimizer.state and torch.equal(matrix, torch.zeros(3, 4))


def test_split_parameters():
    model = _model(share_att_key=False)
    matrices, rest = training.split_parameters(model)
    assert len(matrices) == 2 * 8 and all(m.dim() == 2 for m in matrices)
    every = {id(p) for p in model.parameters()}
    assert {id(p) for p in matrices} | {id(p) for p in rest} == every
    assert len(matrices) + len(rest) == len(every)
    model.encoder.layer[0].attention.self.query_proj.weight.requires_grad_(False)
    assert len(training.split_parameters(model)[0]) == 15


def test_orthogonalize_refusals():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with pytest.raises(RuntimeError, match="GPU"):
        training.orthogonalize(torch.zeros(3, 4))
    with FakeTensorMode():
        def t(*shape, dtype=torch.float32):
            return torch.empty(shape, dtype=dtype, device="cuda")

        out = training.orthogonalize(t(2, 3, 5, 7))
        assert out.shape == (2, 3, 5, 7) and out.dtype == torch.bfloat16
        for error, args in ((TypeError, (t(3, 4, dtype=torch.float64),)), (ValueError, (t(4),)),
                            (ValueError, (t(0, 4),)), (ValueError, (t(4, 0),)),
                            (ValueError, (t(3, 4), 0)),
                            (ValueError, (t(3, 4), 5, training.NEWTON_SCHULZ, -1.0)),
                            (ValueError, (t(3, 4), 5, training.NEWTON_SCHULZ, float("nan")))):
            with pytest.raises(error):
                training.orthogonalize(*args)


def test_c_orthogonalize_refusals():
    from disentangled_flash import _lib

    lib, at = _lib.load(), 1 << 20
    null, shape, dtype, align, large, workspace = -1, -2, -4, -5, -6, -7
    size = lib.dflash_orthogonalize_workspace_bytes(2, 5, 7)
    assert size > 0
    good = [at, at, 2, 5, 7, 5, 3.0, -4.0, 2.0, 1e-7, 0, at, size, None]
    for code, changed in (
        (null, {0: None}), (null, {1: None}), (null, {11: None}), (shape, {2: -1}), (shape, {3: 0}),
        (shape, {4: 0}), (shape, {5: 0}), (shape, {9: -1.0}), (shape, {9: float("nan")}),
        (dtype, {10: 3}), (align, {0: at + 1}), (align, {1: at + 8}), (align, {11: at + 8}),
        (large, {3: 1 << 21}), (large, {2: 65536}), (large, {3: 1 << 20, 4: 1 << 20}),
        (workspace, {12: size - 1}),
    ):
        args = list(good)
        for n, value in changed.items():
            args[n] = value
        assert lib.dflash_orthogonalize(*args) == code, changed
    args = list(good)
    args[2] = 0
    assert lib.dflash_orthogonalize(*args) == 0
    assert lib.dflash_orthogonalize_workspace_bytes(0, 5, 7) == 0
    assert lib.dflash_orthogonalize_workspace_bytes(1, 1 << 21, 7) == 0
