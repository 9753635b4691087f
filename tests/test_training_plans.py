"""CPU tests of what calls share: the tables of relative distances, the steps of a dropout state."""

from __future__ import annotations

import io

import pytest
import torch

from disentangled_flash import enable_deberta_training, training
from disentangled_flash.position import SharedPositionPlanCache

transformers = pytest.importorskip("transformers")

from test_training_attention import _inputs, _model, calls  # noqa: E402, F401 (tests/ is on the path)


def _cache():
    return SharedPositionPlanCache(position_buckets=8, max_relative_positions=40,
                                   position_embedding_size=8)


class _Saves(torch.autograd.Function):
    """Saves a table for its backward pass, as the attention's node does."""

    @staticmethod
    def forward(ctx, x, table):
        ctx.save_for_backward(table)
        return x * 1

    @staticmethod
    def backward(ctx, grad):
        assert ctx.saved_tensors[0] is not None
        return grad, None


def test_tables_made_in_inference_mode_serve_a_backward_pass():
    cache = _cache()
    with torch.inference_mode():
        dense = cache.dense(9, "cpu")
        compact = cache.compact(11, "cpu")
    x = torch.ones(3, requires_grad=True)
    for table in (dense.pair_to_local, dense.active_slots, dense.compact.delta_to_local,
                  compact.active_slots, compact.delta_to_local):
        assert not table.is_inference()
        _Saves.apply(x, table).sum().backward()
    assert cache.compact(9, "cpu") is dense.compact


def test_training_after_a_validation_in_inference_mode(calls, monkeypatch):  # noqa: F811
    """The first forward of a length runs in inference mode, the next one trains."""

    stand_in = training.attention

    def attention(query, key, value, pos_key, pos_query, places, *args, **settings):
        out = stand_in(query, key, value, pos_key, pos_query, places, *args, **settings)
        return _Saves.apply(out, places) if out.requires_grad else out

    monkeypatch.setattr(training, "attention", attention)
    model = enable_deberta_training(_model(), attention="hip")
    ids, mask = _inputs()
    model.eval()
    with torch.inference_mode():
        model(ids, attention_mask=mask)
    model.train()
    model(ids, attention_mask=mask).last_hidden_state.sum().backward()
    assert len(calls) == 4
    assert model.encoder.rel_embeddings.weight.grad is not None


@pytest.mark.parametrize("how", ["first read", "advance", "begin"])
def test_a_step_drawn_in_inference_mode_serves_a_backward_pass(how):
    state = training.DropoutState(5)
    with torch.inference_mode():
        if how == "advance":
            state.advance()
        elif how == "begin":
            state.begin()
        state.rng  # noqa: B018
        state.end()
    assert not state.rng.is_inference() and not state.counter.is_inference()
    assert state.rng.tolist() == [5, 0 if how == "first read" else 1]
    x = torch.ones(3, requires_grad=True)
    _Saves.apply(x, state.rng).sum().backward()
    state.advance()
    assert state.rng.tolist() == [5, 1 if how == "first read" else 2]


def test_tables_of_a_cache_that_was_moved_are_made_again():
    """Loading to another device moves the tables, not the names under which they are kept."""

    cache = _cache()
    want = cache.dense(9, "cpu"), cache.compact(11, "cpu")
    store = io.BytesIO()
    torch.save(cache, store)
    store.seek(0)
    moved = torch.load(store, weights_only=False, map_location="meta")
    got = moved.dense(9, "cpu"), moved.compact(11, "cpu")
    assert torch.equal(got[0].pair_to_local, want[0].pair_to_local)
    for a, b in ((got[0].compact, want[0].compact), (got[1], want[1])):
        assert torch.equal(a.active_slots, b.active_slots)
        assert torch.equal(a.delta_to_local, b.delta_to_local)
    assert moved.dense(9, "cpu") is got[0] and moved.compact(11, "cpu") is got[1]
    assert cache.compact(11, torch.device("cpu", 0)).delta_to_local.device.type == "cpu"
    named = cache.compact(11, torch.device("cpu", 0))
    assert cache.compact(11, torch.device("cpu", 0)) is named


def test_a_backbone_that_was_saved_on_another_device(calls):  # noqa: F811
    model = enable_deberta_training(_model(), attention="hip").eval()
    ids, mask = _inputs()
    want = model(ids, attention_mask=mask).last_hidden_state
    plans = model.encoder.layer[0].attention.self._plans
    store = io.BytesIO()
    torch.save(plans, store)
    store.seek(0)
    moved = torch.load(store, weights_only=False, map_location="meta")
    for layer in model.encoder.layer:
        layer.attention.self.__dict__["_plans"] = moved
    assert torch.equal(model(ids, attention_mask=mask).last_hidden_state, want)
