"""CPU tests of the training operators in programs: transforms, compilers, checkpoints and modules
that change after ``enable_deberta_training``.  Kernels do not run here: operators meet fake GPU
tensors, or are recorded."""

from __future__ import annotations

import contextlib
import copy
import functools
import pickle
import subprocess
import sys

import pytest
import torch
from torch import nn
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad
from torch.utils.checkpoint import checkpoint


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


def test_one_mask_for_every_sample_is_refused():
    """Under vmap: the samples' masks come from their own rng, or the call raises."""

    from disentangled_flash import training

    vmap = torch.func.vmap
    with FakeTensorMode():
        x = torch.empty(4, 3, 16, device="cuda")
        w = torch.empty(16, device="cuda")
        rng = torch.empty(2, dtype=torch.int64, device="cuda")
        rngs = torch.empty(4, 2, dtype=torch.int64, device="cuda")

        def drop(t, r):
            return training.dropout(t, 0.5, r)

        def tail(t, residual, r, p=0.5):
            return training.layer_norm(t, w, w, 1e-5, residual, p, r)

        for call in (
            lambda: vmap(drop, (0, None))(x, rng),
            lambda: vmap(tail, (0, 0, None))(x, x, rng),
            lambda: vmap(tail, (0, None, None))(x, x[0], rng),
            lambda: vmap(tail, (None, 0, None))(x[0], x, rng),
            lambda: vmap(vmap(drop, (0, None)), (0, 0))(x, rngs),  # the inner samples share one
            lambda: vmap(vmap(drop, (0, 0)), (0, None))(x, rngs[:3]),  # the outer ones
        ):
            with pytest.raises(ValueError, match="vmap"):
                call()
        assert vmap(drop)(x, rngs).shape == x.shape
        assert vmap(tail)(x, x, rngs).shape == x.shape
        assert vmap(lambda t: tail(t, None, None, 0.0))(x).shape == x.shape
        assert vmap(lambda t: training.dropout(t, 0.0, rng))(x).shape == x.shape


_FIRST_USE = """
import sys
import torch
sys.path.insert(0, {package!r})
from disentangled_flash import training

training._check_floating = lambda name, tensor: None  # (CPU tensors: nothing is run)
graphs = []

def backend(graph, inputs):
    graphs.append(graph)
    return lambda *args: (torch.zeros(3, 16),)

x, w, rng = torch.zeros(3, 16), torch.zeros(16), torch.zeros(2, dtype=torch.int64)
table, ids = torch.zeros(9, 16), torch.zeros(3, dtype=torch.int64)
call = {call}
torch.compile(call, backend=backend, fullgraph=True)()
names = [str(node.target) for graph in graphs for node in graph.graph.nodes]
assert any("disentangled_flash." in name for name in names), names
"""


@pytest.mark.parametrize("call", ["lambda: training.dropout(x, 0.5, rng)",
                                  "lambda: training.layer_norm(x, w, w, 1e-5, x, 0.5, rng)",
                                  "lambda: training.embedding(ids, table)"])
def test_first_use_may_be_traced(call):
    """A process whose first call of an operator is inside torch.compile, as one graph."""

    from disentangled_flash import _lib

    program = _FIRST_USE.format(package=str(_lib.library_path().parents[1]), call=call)
    done = subprocess.run([sys.executable, "-c", program], capture_output=True, text=True,
                          timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def _backbone(**over):
    from transformers import DebertaV2Config, DebertaV2Model

    fields = dict(vocab_size=100, hidden_size=64, num_hidden_layers=2, num_attention_heads=2,
                  intermediate_size=128, hidden_act="gelu", type_vocab_size=2,
                  max_position_embeddings=64, relative_attention=True, position_buckets=16,
                  pos_att_type=["p2c", "c2p"], norm_rel_ebd="layer_norm", share_att_key=True)
    fields.update(over)
    torch.manual_seed(5)
    return DebertaV2Model(DebertaV2Config(**fields))


@pytest.fixture
def drops(monkeypatch):
    """The (site, seed, step) of every element-wise dropout, which returns its input."""

    from disentangled_flash import training

    seen = []

    def dropout(x, p, rng, site=0):
        seen.append((site, *rng.tolist()))
        return x

    monkeypatch.setattr(training, "dropout", dropout)
    return seen


def _forward(model):
    return model(torch.arange(20).reshape(2, 10)).last_hidden_state


def _steps(drops):
    """The steps met since the last call, and forgets them."""

    steps = {step for _, _, step in drops}
    drops.clear()
    return steps


@pytest.mark.parametrize("found_by", ["class name", "type", "layer"])
def test_dropout_of_a_backbone_in_eval_mode_draws_new_masks(drops, found_by):
    """Monte Carlo dropout, and a layer in training in a backbone that is not."""

    from disentangled_flash import enable_deberta_training

    model = enable_deberta_training(_backbone(), seed=3).eval()
    with torch.no_grad():
        _forward(model)
    assert not drops and model.dropout_state.counter.tolist() == [3, 0]
    if found_by == "layer":
        model.encoder.layer[1].train()
    else:
        for module in model.modules():
            if isinstance(module, nn.Dropout) if found_by == "type" \
                    else type(module).__name__.startswith("Dropout"):
                module.train()
    with torch.no_grad():
        for step in (1, 2, 3):
            _forward(model)
            assert _steps(drops) == {step}
    model.eval()
    with torch.no_grad():
        _forward(model)
    assert not drops
    model.train()
    _forward(model)
    assert _steps(drops) == {4}


def test_backward_pass_after_a_forward_in_eval_mode(drops):
    """A forward in eval mode between a forward and its backward pass, whose checkpointed layer
    recomputes what it computed; a head that drops behind a backbone in eval mode draws new masks."""

    from disentangled_flash import enable_deberta_training, training

    model = enable_deberta_training(_backbone(), seed=3).train()
    for layer in model.encoder.layer:
        layer.forward = functools.partial(checkpoint, layer.forward, use_reentrant=False)
    out = _forward(model)
    with torch.no_grad():
        _forward(model.eval())
    model.train()
    assert _steps(drops) == {1}
    out.sum().backward()
    assert _steps(drops) == {1}
    head = training.Dropout(0.5, model.dropout_state, 1000)
    model.eval()
    for step in (2, 3):
        head(_forward(model)).sum().backward()
        assert _steps(drops) == {step}


def test_dropout_made_in_place_is_torchs(drops):
    from disentangled_flash import training

    drop = training.Dropout(1.0, training.DropoutState(0), 0)
    drop.inplace = True
    x = torch.ones(4)
    assert drop(x) is x and not x.any() and not drops


class _Generator:
    """torch's generator of a GPU, as far as the state reads it."""

    offset = 0

    def initial_seed(self):
        return 1234

    def get_offset(self):
        return self.offset

    def set_offset(self, offset):
        self.offset = offset

    @contextlib.contextmanager
    def back_at(self, offset):
        self.offset, now = offset, self.offset
        yield
        self.offset = now


@pytest.fixture
def generator(monkeypatch):
    from disentangled_flash import training

    made = _Generator()
    monkeypatch.setattr(training, "_generator", lambda counter: made)
    return made


def _checkpointed(model, generator, use_reentrant):
    """torch.utils.checkpoint around the backbone, which puts ``generator`` back."""

    start = generator.offset
    weight = torch.ones(1, requires_grad=True)  # (what a reentrant one has to differentiate)

    def call(weight):
        with generator.back_at(start) if torch._C._current_graph_task_id() != -1 \
                else contextlib.nullcontext():
            return _forward(model) * weight

    return checkpoint(call, weight, use_reentrant=use_reentrant)


@pytest.mark.parametrize("use_reentrant", [False, True])
@pytest.mark.parametrize("mode", ["train", "eval"])
def test_checkpointed_backbone_recomputes_its_own_masks(drops, generator, use_reentrant, mode):
    """Two forwards before their backward passes, in either order."""

    from disentangled_flash import enable_deberta_training

    model = enable_deberta_training(_backbone(), seed=3).train()
    if mode == "eval":
        model.eval().encoder.layer[1].train()
    for order in ((0, 1), (1, 0)):
        steps, outs = [], []
        for _ in range(2):
            outs.append(_checkpointed(model, generator, use_reentrant))
            steps.append(_steps(drops))
            assert len(steps[-1]) == 1
        assert steps[0] != steps[1]
        counter = model.dropout_state.counter.tolist()
        for i in order:
            outs[i].sum().backward()
            assert _steps(drops) == steps[i]
        assert model.dropout_state.counter.tolist() == counter
    _forward(model)
    assert _steps(drops) == {counter[1] + 1}


def test_recomputation_without_its_generator_raises(drops, generator):
    from disentangled_flash import enable_deberta_training

    model = enable_deberta_training(_backbone(), seed=3).train()
    out = checkpoint(lambda: _forward(model), use_reentrant=False)
    with pytest.raises(RuntimeError, match="generator"):
        out.sum().backward()
    drops.clear()
    _forward(model).sum().backward()  # the state goes on
    assert _steps(drops) == {2}
    # Where nothing is dropped nothing is wrong.
    model = enable_deberta_training(
        _backbone(hidden_dropout_prob=0.0, attention_probs_dropout_prob=0.0)).train()
    checkpoint(lambda: _forward(model), use_reentrant=False).sum().backward()
    assert not drops


def test_copies_of_a_model_have_steps_of_their_own(drops, generator):
    from disentangled_flash import enable_deberta_training

    model = enable_deberta_training(_backbone(), seed=3).train()
    twin = copy.deepcopy(model)
    twin.dropout_state.counter[1] = 10
    start = generator.offset
    first = _checkpointed(model, generator, False)
    generator.offset = start  # (the same position)
    second = _checkpointed(twin, generator, False)
    assert _steps(drops) == {1, 11}
    first.sum().backward()
    assert _steps(drops) == {1}
    second.sum().backward()
    assert _steps(drops) == {11}


def test_steps_remembered_are_bounded(drops, generator, monkeypatch):
    from disentangled_flash import training

    monkeypatch.setattr(training, "_DRAWN_KEPT", 3)
    training._drawn.clear()
    state = training.DropoutState(1)
    for _ in range(5):
        state.advance()
    assert [rng.tolist() for rng in training._drawn.values()] == [[1, 3], [1, 4], [1, 5]]


# ---- output blocks whose children change ---------------------------------------------


@pytest.fixture
def block(monkeypatch):
    """An output block that takes CPU tensors for a GPU's, and records what it computes itself."""

    from disentangled_flash import enable_deberta_training, training

    made = enable_deberta_training(_backbone()).encoder.layer[0].output.train()
    assert type(made) is training.OutputBlock
    made.calls = calls = []

    def layer_norm(x, weight, bias, eps, residual=None, p=0.0, rng=None, site=0):
        calls.append("layer_norm")
        return nn.functional.layer_norm(x + residual, (64,), weight, bias, eps)

    monkeypatch.setattr(training, "layer_norm", layer_norm)
    monkeypatch.setattr(training, "dropout", lambda x, p, rng, site=0: calls.append("dropout") or x)
    monkeypatch.setattr(training, "_on_gpu", lambda x: True)
    return made


def _call(block):
    block.calls.clear()
    return block(torch.ones(2, 128), torch.linspace(-1, 1, 128).view(2, 64))


def test_output_block_is_one_call(block):
    want = _call(block)
    assert block.calls == ["layer_norm"]
    assert torch.equal(_call(block.eval()), want) and block.calls == ["layer_norm"]


@pytest.mark.parametrize("child", ["LayerNorm", "dropout"])
@pytest.mark.parametrize("kind", ["forward", "forward_pre", "full_backward", "full_backward_pre"])
def test_hooks_put_on_later_run(block, child, kind):
    seen = []
    module = getattr(block, child)
    handle = getattr(module, f"register_{kind}_hook")(lambda *a: seen.append(child) and None)
    _call(block).sum().backward()
    assert seen == [child] and block.calls == ["dropout"]
    handle.remove()
    _call(block)
    assert seen == [child] and block.calls == ["layer_norm"]


@pytest.mark.parametrize("kind", ["forward", "forward_pre", "full_backward", "full_backward_pre"])
def test_hooks_of_all_modules_run(block, kind):
    seen = []
    register = getattr(torch.nn.modules.module, f"register_module_{kind}_hook")
    handle = register(lambda module, *a: seen.append(type(module).__name__) and None)
    try:
        _call(block).sum().backward()
    finally:
        handle.remove()
    assert "LayerNorm" in seen and "Dropout" in seen


def test_forward_set_on_a_child_is_called(block):
    block.LayerNorm.forward = lambda x: x * 0 + 5
    assert bool((_call(block) == 5).all())


def test_replaced_children_are_called(block):
    class Scaled(nn.LayerNorm):
        def forward(self, x):
            return 3 * super().forward(x)

    want = _call(block)
    plain = block.LayerNorm
    block.LayerNorm = Scaled(64, plain.eps)
    assert torch.equal(_call(block), 3 * want)
    block.LayerNorm = nn.RMSNorm(64)
    assert not torch.equal(_call(block), want) and block.calls == ["dropout"]
    block.LayerNorm = nn.LayerNorm(64, elementwise_affine=False)
    _call(block)
    block.LayerNorm = nn.Identity()
    _call(block)
    block.LayerNorm = plain
    for drop in (nn.Dropout(0.0), nn.Identity()):
        block.dropout = drop
        assert torch.equal(_call(block), want) and block.calls == []
    block.dropout = nn.Dropout(1.0)
    assert torch.equal(_call(block)[0], _call(block)[0]) and block.calls == []


# ---- which modules are replaced ------------------------------------------------------


def test_blocks_are_recognised_by_more_than_their_name():
    """A class of the same name elsewhere, and a subclass of the norm, keep their own forward."""

    from transformers.models.deberta_v2 import modeling_deberta_v2 as hf

    from disentangled_flash import enable_deberta_training, training

    class DebertaV2Output(nn.Module):
        def __init__(self, block):
            super().__init__()
            self.dense, self.LayerNorm, self.dropout = block.dense, block.LayerNorm, block.dropout

        def forward(self, hidden_states, input_tensor):
            return self.dropout(self.LayerNorm(self.dense(hidden_states))) + input_tensor

    class Scaled(nn.LayerNorm):
        def forward(self, x):
            return 3 * super().forward(x)

    model = _backbone().eval()
    first, second = model.encoder.layer
    first.output = DebertaV2Output(first.output)
    second.output.LayerNorm = Scaled(64)
    want = _forward(model)
    enable_deberta_training(model)
    assert type(first.output) is DebertaV2Output and type(second.output) is hf.DebertaV2Output
    assert type(first.output.dropout) is training.Dropout  # (its children are replaced)
    assert type(second.output.LayerNorm) is Scaled
    assert type(first.attention.output) is training.OutputBlock
    assert torch.equal(_forward(model), want)


def test_a_patched_block_class_keeps_its_forward(monkeypatch):
    from transformers.models.deberta_v2 import modeling_deberta_v2 as hf

    from disentangled_flash import enable_deberta_training, training

    monkeypatch.setattr(hf.DebertaV2Output, "forward", lambda self, h, x: self.dense(h) + x)
    model = enable_deberta_training(_backbone())
    assert type(model.encoder.layer[0].output) is hf.DebertaV2Output
    assert type(model.encoder.layer[0].attention.output) is training.OutputBlock


# ---- settings that the operators lack ------------------------------------------------


def test_settings_changed_later_are_honoured(monkeypatch):
    """torch's own module computes what the operator does not."""

    from disentangled_flash import training

    calls = []
    monkeypatch.setattr(training, "_on_gpu", lambda x: True)
    monkeypatch.setattr(training, "embedding",
                        lambda ids, weight, padding_idx=None: calls.append("embedding") or
                        nn.functional.embedding(ids, weight, padding_idx))
    monkeypatch.setattr(training, "layer_norm",
                        lambda x, w, b, eps: calls.append("layer_norm") or
                        nn.functional.layer_norm(x, x.shape[-1:], w, b, eps))
    ids = torch.tensor([1, 1, 2])
    made = training.Embedding(5, 8)
    made(ids)
    assert calls == ["embedding"]
    for name, value in (("max_norm", 0.5), ("sparse", True), ("scale_grad_by_freq", True)):
        calls.clear()
        made = training.Embedding(5, 8)
        setattr(made, name, value)
        out = made(ids)
        out.sum().backward()
        assert not calls
        if name == "max_norm":
            assert out.norm(dim=-1).max() <= 0.5 * (1 + 1e-5)
        assert made.weight.grad.is_sparse == (name == "sparse")
        if name == "scale_grad_by_freq":
            assert torch.equal(made.weight.grad[1], torch.ones(8))
    made = training.Embedding(5, 8)
    made.weight = nn.Parameter(torch.randn(8, 5).t())
    assert torch.equal(made(ids), made.weight[ids]) and not calls

    x = torch.randn(2, 3, 8)
    assert training.LayerNorm(8)(x).shape == x.shape and calls == ["layer_norm"]
    calls.clear()
    for norm, plain in ((training.LayerNorm(8, elementwise_affine=False),
                         nn.LayerNorm(8, elementwise_affine=False)),
                        (training.LayerNorm(8, bias=False), nn.LayerNorm(8, bias=False)),
                        (training.LayerNorm((3, 8)), nn.LayerNorm((3, 8)))):
        assert torch.equal(norm(x), plain(x)) and not calls
    wide = training.MAX_HIDDEN + 1
    assert training.LayerNorm(wide)(torch.ones(wide)).shape == (wide,) and not calls


def test_state_is_pickled_with_its_step(drops, generator):
    from disentangled_flash import training

    state = training.DropoutState(7)
    state.advance()
    state.begin()
    back = pickle.loads(pickle.dumps(state))
    assert back.rng.tolist() == [7, 1] and back._token != state._token
    assert state.rng.tolist() == [7, 2]  # (begun)
