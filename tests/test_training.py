"""CPU tests of the training operators: the generator's definition, refusals of the Python and
the C interface, and the modules that ``enable_deberta_training`` puts in."""

from __future__ import annotations

import copy
import ctypes

import pytest
import torch
from torch import nn
from torch._subclasses.fake_tensor import FakeTensorMode

import training_reference as ref  # noqa: E402 (tests/ is on the path)


def test_generator_gives_the_published_words():
    """Known answers of Philox4x32 with 7 and 10 rounds (the paper's test vectors)."""

    def words(counter, key, rounds):
        return [int(w) for w in ref.philox(counter, key, rounds)]

    assert words([0] * 4, (0, 0), 7) == [0x5F6FB709, 0x0D893F64, 0x4F121F81, 0x4F730A48]
    assert words([0] * 4, (0, 0), 10) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = 0xFFFFFFFF
    assert words([ones] * 4, (ones, ones), 10) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


def test_generator_keeps_the_share_it_is_asked_for():
    """The kept share of 2^20 elements lies within 5 deviations, neighbours and sites are
    uncorrelated within 5, and p is a multiple of 2^-16."""

    n = 1 << 20
    rng = torch.tensor([1234567890123456789, 42])
    for p in (0.1, 0.5, 1 / 65536):
        share = ref.limit_of(p) / 65536
        deviation = (share * (1 - share) / n) ** 0.5
        a = (~ref.kept((n,), p, rng, 3)).double() - share
        assert abs(a.mean().item()) < 5 * deviation
        other = (~ref.kept((n,), p, rng, 4)).double() - share
        for b in (a.roll(1), a.roll(8), other):
            assert abs((a * b).mean().item()) < 5 * share * (1 - share) / n ** 0.5
    assert ref.limit_of(1e-9) == 1 and ref.limit_of(1 - 1e-9) == 65535
    assert ref.limit_of(0) == 0 and ref.limit_of(1) == 65536


def test_reference_gradients_are_differences():
    """The float64 formulas the GPU tests compare with, against central differences."""

    gen = torch.Generator().manual_seed(0)
    x, r, dy = (torch.randn(5, 24, generator=gen, dtype=torch.float64) for _ in range(3))
    w, b = (torch.randn(24, generator=gen, dtype=torch.float64) for _ in range(2))
    mult = ref.factor((5, 24), 0.3, torch.tensor([7, 1]), 2)
    out = ref.layer_norm(x, w, b, 1e-5, r, mult, dy)
    inputs = {"dx": x, "dresidual": r, "dweight": w, "dbias": b}
    for name, tensor in inputs.items():
        direction = torch.randn(tensor.shape, generator=gen, dtype=torch.float64)
        step = 1e-5
        values = []
        for sign in (1, -1):
            args = {n: t + sign * step * direction if t is tensor else t
                    for n, t in inputs.items()}
            y = ref.layer_norm(args["dx"], args["dweight"], args["dbias"], 1e-5,
                               args["dresidual"], mult)["y"][0]
            values.append((y * dy).sum())
        difference = (values[0] - values[1]) / (2 * step)
        analytic = (out[name][0] * direction).sum()
        # The difference is off by step^2 / 6 of the third derivative and 1e-16 / step of y.
        assert abs(difference - analytic) < 1e-7 * (1 + abs(analytic)), name


# ---- refusals ------------------------------------------------------------------------


def test_operators_want_gpu_tensors():
    from disentangled_flash import training

    x = torch.zeros(2, 8)
    with pytest.raises(RuntimeError, match="GPU"):
        training.dropout(x, 0.1, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="GPU"):
        training.layer_norm(x, torch.ones(8), torch.ones(8), 1e-5)
    with pytest.raises(RuntimeError, match="GPU"):
        training.embedding(torch.zeros(2, dtype=torch.int64), x)


def test_layer_norm_refusals():
    from disentangled_flash.training import layer_norm

    with FakeTensorMode():
        def t(*shape, dtype=torch.float16, device="cuda"):
            return torch.empty(shape, dtype=dtype, device=device)

        x, w = t(4, 64), t(64)
        rng = t(2, dtype=torch.int64)
        assert layer_norm(x, w, w, 1e-5).shape == x.shape
        assert layer_norm(x, w.float(), w.float(), 1e-5, x, 0.1, rng).dtype == torch.float16
        for error, match, args in (
            (TypeError, "not fp16", (x.double(), w, w, 1e-5)),
            (ValueError, r"\[\.\.\., H\]", (t(), w, w, 1e-5)),
            (ValueError, r"\[\.\.\., H\]", (t(4, 0), t(0), t(0), 1e-5)),
            (ValueError, r"\[\.\.\., H\]", (t(4, 8193), t(8193), t(8193), 1e-5)),
            (ValueError, "weight must be", (x, t(63), w, 1e-5)),
            (ValueError, "bias must be", (x, w, t(1, 64), 1e-5)),
            (TypeError, "weight dtype", (x, w.bfloat16(), w.bfloat16(), 1e-5)),
            (TypeError, "bias dtype", (x, w, w.float(), 1e-5)),
            (ValueError, "weight is on", (x, t(64, device="cpu"), w, 1e-5)),
            (ValueError, "residual must match", (x, w, w, 1e-5, t(4, 63))),
            (ValueError, "residual must match", (x, w, w, 1e-5, x.float())),
            (ValueError, "residual must match", (x, w, w, 1e-5, t(4, 64, device="cpu"))),
            (ValueError, "probability", (x, w, w, 1e-5, None, -0.1, rng)),
            (ValueError, "probability", (x, w, w, 1e-5, None, float("nan"), rng)),
            (ValueError, "needs rng", (x, w, w, 1e-5, None, 0.1)),
            (ValueError, "int64", (x, w, w, 1e-5, None, 0.1, rng.int())),
            (ValueError, "int64", (x, w, w, 1e-5, None, 0.1, t(3, dtype=torch.int64))),
            (ValueError, "rng is on", (x, w, w, 1e-5, None, 0.1,
                                       t(2, dtype=torch.int64, device="cpu"))),
            (ValueError, "site", (x, w, w, 1e-5, None, 0.1, rng, -1)),
            (ValueError, "site", (x, w, w, 1e-5, None, 0.1, rng, 1 << 32)),
        ):
            with pytest.raises(error, match=match):
                layer_norm(*args)


def test_dropout_refusals():
    from disentangled_flash.training import dropout

    with FakeTensorMode():
        x = torch.empty(4, 64, device="cuda")
        rng = torch.empty(2, dtype=torch.int64, device="cuda")
        assert dropout(x, 0.0, rng) is x
        assert dropout(x, 1.0, rng).shape == x.shape
        for error, match, args in (
            (TypeError, "not fp16", (x.long(), 0.1, rng)),
            (ValueError, "probability", (x, 1.1, rng)),
            (ValueError, "needs rng", (x, 0.1, None)),
            (ValueError, "int64", (x, 0.1, rng[:1])),
            (ValueError, "int64", (x, 0.1, torch.empty(4, dtype=torch.int64, device="cuda")[::2])),
            (ValueError, "site", (x, 0.1, rng, -5)),
        ):
            with pytest.raises(error, match=match):
                dropout(*args)


def test_embedding_refusals():
    from disentangled_flash.training import embedding

    with FakeTensorMode():
        table = torch.empty(10, 16, device="cuda")
        ids = torch.empty(3, 5, dtype=torch.int64, device="cuda")
        assert embedding(ids, table).shape == (3, 5, 16)
        assert embedding(ids[0, 0], table).shape == (16,)
        for error, match, args in (
            (TypeError, "not fp16", (ids, table.double())),
            (ValueError, "weight must be", (ids, table[0])),
            (ValueError, "weight must be", (ids, table[:0])),
            (ValueError, "contiguous", (ids, table.t())),
            (TypeError, "int32 or int64", (ids.float(), table)),
            (TypeError, "int32 or int64", (ids.short(), table)),
            (ValueError, "input_ids are on", (torch.empty(3, dtype=torch.int64), table)),
            (ValueError, "padding_idx", (ids, table, 1.0, 10)),
            (ValueError, "padding_idx", (ids, table, 1.0, -11)),
        ):
            with pytest.raises(error, match=match):
                embedding(*args)


def test_missing_torch_library_is_named(monkeypatch, tmp_path, lib):
    from disentangled_flash import _lib

    monkeypatch.setattr(_lib, "_torch_ops_loaded", False)
    monkeypatch.setattr(_lib, "library_path", lambda: tmp_path / _lib.LIBRARY_NAME)
    with pytest.raises(RuntimeError, match="libdflash_torch.so is missing: build"):
        _lib.load_torch_ops()
    (tmp_path / _lib.TORCH_LIBRARY_NAME).write_bytes(b"not a library")
    with pytest.raises(RuntimeError, match="cannot load"):
        _lib.load_torch_ops()


@pytest.fixture(scope="module")
def lib():
    from disentangled_flash import _lib

    if not _lib.library_path().exists():
        pytest.skip("libdflash.so not built (run python __graft_entry__.py)")
    return _lib.load()


NULL, SHAPE, DTYPE, ALIGN, LARGE, WORKSPACE = -1, -2, -4, -5, -6, -7
A = 4096  # stands for an address: every call below is refused before anything is launched


def test_c_dropout_refusals(lib):
    def call(x=A, y=A, n=8, p=0.1, rng=A, site=0, dtype=0):
        return lib.dflash_dropout(x, y, n, p, rng, site, dtype, None)

    assert call(n=0) == 0 and call(n=0, x=None, y=None, rng=None) == 0
    assert call(n=-1) == SHAPE
    assert call(p=-0.1) == SHAPE and call(p=1.5) == SHAPE and call(p=float("nan")) == SHAPE
    assert call(dtype=3) == DTYPE and call(dtype=-1) == DTYPE
    assert call(x=None) == NULL and call(y=None) == NULL and call(rng=None) == NULL
    assert call(x=A + 1) == ALIGN and call(y=A + 2, dtype=2) == ALIGN and call(rng=A + 4) == ALIGN
    assert call(n=1 << 40) == LARGE


def test_c_layernorm_refusals(lib):
    def fwd(x=A, r=A, g=A, b=A, y=A, mean=A, rstd=A, rows=4, hidden=64, p=0.1, rng=A, dtype=1,
            wdtype=1):
        return lib.dflash_dropout_layernorm_fwd(x, r, g, b, y, mean, rstd, rows, hidden, 1e-7, p,
                                                rng, 0, dtype, wdtype, None)

    assert fwd(rows=0) == 0
    for over in ({"rows": -1}, {"hidden": 0}, {"hidden": 8193}, {"p": 2.0}, {"rows": 1 << 60}):
        assert fwd(**over) == SHAPE, over
    for over in ({"dtype": 3}, {"wdtype": 0}, {"dtype": 2}, {"dtype": 0}, {"wdtype": -1}):
        assert fwd(**over) == DTYPE, over
    for over in ({"x": None}, {"g": None}, {"b": None}, {"y": None}, {"mean": None},
                 {"rstd": None}, {"rng": None}):
        assert fwd(**over) == NULL, over
    for over in ({"x": A + 1}, {"r": A + 1}, {"y": A + 1}, {"g": A + 1}, {"mean": A + 2},
                 {"rng": A + 4}, {"g": A + 2, "wdtype": 2}, {"x": A + 8}, {"r": A + 4}):
        assert fwd(**over) == ALIGN, over
    size = lib.dflash_dropout_layernorm_bwd_workspace_bytes(40, 64)
    assert size == 40 * 2 * 64 * 4
    assert lib.dflash_dropout_layernorm_bwd_workspace_bytes(32, 64) == 0  # one workgroup's rows
    assert lib.dflash_dropout_layernorm_bwd_workspace_bytes(32, 63) == 32 * 2 * 63 * 4
    assert lib.dflash_dropout_layernorm_bwd_workspace_bytes(1 << 40, 64) == 512 * 2 * 64 * 4
    assert lib.dflash_dropout_layernorm_bwd_workspace_bytes(-1, 64) == 0
    assert lib.dflash_dropout_layernorm_bwd_workspace_bytes(4, 9000) == 0

    def bwd(dy=A, x=A, r=A, g=A, mean=A, rstd=A, dx=A, dr=A, dg=A, db=A, rows=40, hidden=64, p=0.1,
            rng=A, dtype=1, wdtype=1, ws=A, size=size):
        return lib.dflash_dropout_layernorm_bwd(dy, x, r, g, mean, rstd, dx, dr, dg, db, rows,
                                                hidden, p, rng, 0, dtype, wdtype, ws, size, None)

    assert bwd(dx=None, dr=None, dg=None, db=None) == 0  # nothing wanted
    for over in ({"rows": -1}, {"hidden": 0}, {"hidden": 8193}, {"p": -1.0}):
        assert bwd(**over) == SHAPE, over
    for over in ({"dtype": 3}, {"wdtype": 0}, {"dtype": 2}):
        assert bwd(**over) == DTYPE, over
    for over in ({"dy": None}, {"x": None}, {"g": None}, {"mean": None}, {"rstd": None},
                 {"rng": None}, {"dg": None}, {"db": None}, {"ws": None}):
        assert bwd(**over) == NULL, over
    for over in ({"dy": A + 1}, {"dx": A + 1}, {"dr": A + 1}, {"dg": A + 1}, {"ws": A + 2}):
        assert bwd(**over) == ALIGN, over
    assert bwd(size=size - 1) == WORKSPACE


def test_c_embedding_refusals(lib):
    def fwd(ids=A, table=A, out=A, n=4, rows=10, hidden=64, bytes_=8, dtype=1):
        return lib.dflash_embedding_fwd(ids, table, out, n, rows, hidden, 1.0, bytes_, dtype, None)

    assert fwd(n=0) == 0
    for over in ({"n": -1}, {"n": (1 << 26) + 1}, {"rows": 0}, {"hidden": 0},
                 {"hidden": (1 << 20) + 1}, {"rows": 2 ** 31 - 1}):
        assert fwd(**over) == SHAPE, over
    assert fwd(bytes_=2) == DTYPE and fwd(dtype=3) == DTYPE
    for over in ({"ids": None}, {"table": None}, {"out": None}):
        assert fwd(**over) == NULL, over
    for over in ({"ids": A + 4}, {"table": A + 1}, {"out": A + 1}):
        assert fwd(**over) == ALIGN, over

    size = lib.dflash_embedding_bwd_workspace_bytes(400, 64)
    assert size > 0 and lib.dflash_embedding_bwd_workspace_bytes(-1, 64) == 0

    def bwd(ids=A, dout=A, dtable=A, n=400, rows=10, hidden=64, bytes_=8, dtype=1, ws=A, size=size):
        return lib.dflash_embedding_bwd(ids, dout, dtable, n, rows, hidden, 1.0, -1, bytes_, dtype,
                                        ws, size, None)

    for over in ({"n": -1}, {"rows": 0}, {"hidden": 0}):
        assert bwd(**over) == SHAPE, over
    assert bwd(bytes_=1) == DTYPE and bwd(dtype=7) == DTYPE
    for over in ({"ids": None}, {"dout": None}, {"dtable": None}, {"ws": None}):
        assert bwd(**over) == NULL, over
    for over in ({"ids": A + 4}, {"dout": A + 1}, {"dtable": A + 8}, {"ws": A + 4}):
        assert bwd(**over) == ALIGN, over
    assert bwd(size=size - 1) == WORKSPACE


# ---- modules -------------------------------------------------------------------------


def _backbone(**over):
    from transformers import DebertaV2Config, DebertaV2Model

    fields = dict(vocab_size=100, hidden_size=64, num_hidden_layers=2, num_attention_heads=2,
                  intermediate_size=128, hidden_act="gelu", type_vocab_size=2,
                  max_position_embeddings=64, relative_attention=True, position_buckets=16,
                  pos_att_type=["p2c", "c2p"], norm_rel_ebd="layer_norm", share_att_key=True,
                  conv_kernel_size=3, conv_act="gelu", position_biased_input=True)
    fields.update(over)
    torch.manual_seed(5)
    return DebertaV2Model(DebertaV2Config(**fields))


def test_enable_training_keeps_parameters_and_keys():
    from disentangled_flash import enable_deberta_training, training

    model = _backbone()
    keys = list(model.state_dict())
    before = {name: p for name, p in model.named_parameters()}
    assert enable_deberta_training(model, seed=9) is model
    assert list(model.state_dict()) == keys
    after = dict(model.named_parameters())
    assert after.keys() == before.keys() and all(after[n] is before[n] for n in before)
    kinds = [type(m) for m in model.modules()]
    assert nn.Dropout not in kinds and nn.Embedding not in kinds
    assert kinds.count(training.OutputBlock) == 4 and kinds.count(training.Embedding) == 4
    # (The norms inside the output blocks stay: the block calls the operator itself.)
    assert kinds.count(training.LayerNorm) == 3
    drops = [m for m in model.modules() if isinstance(m, training.Dropout)]
    assert len({d.site for d in drops}) == len(drops)
    assert all(d.state is model.dropout_state for d in drops)
    with pytest.raises(TypeError, match="already"):
        enable_deberta_training(model)
    with pytest.raises(TypeError, match="backbone"):
        enable_deberta_training(nn.Linear(2, 2))


def test_enabled_model_on_the_cpu_is_the_same_in_eval_mode():
    from disentangled_flash import enable_deberta_training

    model = _backbone().eval()
    ids, mask = torch.arange(20).reshape(2, 10), torch.ones(2, 10, dtype=torch.long)
    with torch.no_grad():
        want = model(ids, attention_mask=mask).last_hidden_state
        enable_deberta_training(model)
        got = model(ids, attention_mask=mask).last_hidden_state
    assert torch.equal(got, want)
    model.train()
    with pytest.raises(RuntimeError, match="GPU"):
        model(ids, attention_mask=mask)


def test_enable_training_leaves_what_it_does_not_compute():
    from disentangled_flash import enable_deberta_inference, enable_deberta_training, training

    model = _backbone()
    model.embeddings.word_embeddings = nn.Embedding(100, 64, sparse=True)
    model.embeddings.position_embeddings.register_forward_hook(lambda *a: None)
    model.encoder.layer[0].output.register_forward_hook(lambda *a: None)
    model.encoder.layer[1].output.LayerNorm = nn.LayerNorm(64, elementwise_affine=False)
    enable_deberta_training(model)
    assert type(model.embeddings.word_embeddings) is nn.Embedding
    assert type(model.embeddings.position_embeddings) is nn.Embedding
    assert type(model.encoder.layer[0].output).__name__ == "DebertaV2Output"
    assert type(model.encoder.layer[1].output).__name__ == "DebertaV2Output"
    assert type(model.encoder.layer[1].attention.output) is training.OutputBlock
    inference = enable_deberta_inference(_backbone().eval(), backend="torch", sequence_lengths=[4])
    with pytest.raises(TypeError, match="inference-only"):
        enable_deberta_training(inference)


def test_dropout_state_steps_and_copies():
    from disentangled_flash import enable_deberta_training, training

    state = training.DropoutState(-3)
    assert state.rng.tolist() == [-3, 0] and not state.state_dict()
    first = state.rng
    state.advance()
    assert first.tolist() == [-3, 0] and state.rng.tolist() == [-3, 1]
    with pytest.raises(ValueError, match="64 bits"):
        training.DropoutState(1 << 63)
    model = enable_deberta_training(_backbone(), seed=4)
    twin = copy.deepcopy(model)
    assert twin.dropout_state is not model.dropout_state
    assert twin.embeddings.dropout.state is twin.dropout_state
    assert model.half().dropout_state.counter.dtype == torch.int64
    with pytest.raises(ValueError, match="probability"):
        training.Dropout(1.5, state, 0)


def test_inference_encoder_takes_a_trained_model():
    """``enable_deberta_inference`` after ``enable_deberta_training``, on the torch backend."""

    from disentangled_flash import enable_deberta_inference, enable_deberta_training
    from disentangled_flash.layers import fusable_output_block

    model = _backbone().eval()
    ids, mask = torch.arange(20).reshape(2, 10), torch.ones(2, 10, dtype=torch.long)
    with torch.no_grad():
        want = model(ids, attention_mask=mask).last_hidden_state
        enable_deberta_training(model)
        assert fusable_output_block(model.encoder.layer[0].output)
        enable_deberta_inference(model, backend="torch", sequence_lengths=[10])
        got = model(ids, attention_mask=mask).last_hidden_state
    torch.testing.assert_close(got, want, atol=1e-5, rtol=1e-5)


def test_library_signature_of_the_probability(lib):
    """p crosses the ABI as a double: 1 - 2^-17 must not become 1."""

    assert lib.dflash_dropout.argtypes[3] is ctypes.c_double
