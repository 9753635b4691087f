"""Operators of a DeBERTa training step around its matrix products, and the modules that call them.

The operators, on a GPU in fp16, bf16 and fp32, with their gradients:

* :func:`layer_norm` - ``LayerNorm(dropout(x) + residual)``, the tail of every output block
  (``DebertaV2SelfOutput`` / ``DebertaV2Output``, reference ``_reference.py:101-112`` and
  ``474-485``, which in training drops elements between its dense layer and its residual);
  without residual and dropout a plain LayerNorm.
* :func:`dropout` - dropout whose mask comes from a counter-based generator and is drawn
  again in the backward pass instead of being stored.
* :func:`attention` - disentangled attention with learned rows for the log buckets of the relative
  distance and with dropout on its probabilities, without an ``[L, L]`` tensor of scores.
* :func:`embedding` - the table lookup with a scale, and the dense gradient of the table,
  summed in an order that depends on the ids alone (the same bits on every call).

* :func:`orthogonalize` - the Newton-Schulz iterations of the Muon optimiser for a batch of matrices;
  :class:`Muon` is that optimiser.

:func:`enable_deberta_training` puts them into a Hugging Face DeBERTa-v2/v3 backbone;
``optimize_deberta`` takes the same model afterwards for inference.

**Random numbers** are an input: ``rng`` is an int64 tensor ``[seed, step]`` on the GPU, read
by the kernels, so that a captured step that advances it drops other elements on every
replay; ``site`` numbers the places of a model that drop elements.  An element is dropped by
its index in the flattened tensor, ``rng`` and ``site`` alone, whatever the dtype.  ``p`` is
rounded to a multiple of 2^-16 (to 0 and 1 only where it is 0 or 1), and kept elements are
divided by the rounded probability of being kept.  A dropped element is 0 whatever it held.
Under ``torch.func.vmap`` each sample needs an ``rng`` of its own.

Small steps are bound by the host, and most of that is torch's hand-over of the backward pass
to a thread of its own: under ``torch.autograd.set_multithreading_enabled(False)`` the
gradients of a norm tail took 28 us of host time instead of 61.

Work is launched on torch's current stream of the inputs' device.  Second derivatives raise,
but for dropout's, and forward-mode derivatives do.  Inputs that are not contiguous are copied first, and in :func:`layer_norm`
those that do not start on a 16-byte boundary.
"""

from __future__ import annotations

import itertools
import math
import threading
from collections import OrderedDict
from collections.abc import Iterable, Mapping
from typing import Any

import torch
from torch import nn
from torch.nn.modules import module as torch_module

from . import _lib
from .position import SharedPositionPlanCache

MAX_HIDDEN = 8192  # widest row of layer_norm
ATTENTION_WIDTHS = (32, 64, 128)  # head widths of attention
MAX_LENGTH = 16384  # longest sequence of attention


class _Ops:
    """The torch operators (``csrc/torch_ops.cpp``), loaded at the first call."""

    names = ("dropout", "dropout_layernorm", "embedding_lookup", "attention",
             "orthogonalize")

    def __getattr__(self, name: str) -> Any:
        if name not in self.names:
            raise AttributeError(name)
        _load()
        return getattr(torch.ops.disentangled_flash, name).default


_ops = _Ops()
_loading = threading.Lock()


@torch.compiler.assume_constant_result  # (a first use may be traced: this runs, and is not)
def _load() -> bool:
    with _loading:
        if _Ops.names[0] not in _ops.__dict__:
            _lib.load_torch_ops()
            _register_fakes()
            for op in reversed(_Ops.names):
                setattr(_ops, op, getattr(torch.ops.disentangled_flash, op).default)
    return True


def _register_fakes() -> None:
    """Shapes for tracing (torch.compile, export, FakeTensorMode)."""

    fake = torch.library.register_fake

    @fake("disentangled_flash::dropout")
    def _(x, rng, p, site):
        return torch.empty_like(x)

    @fake("disentangled_flash::dropout_layernorm")
    def _(x, residual, weight, bias, rng, eps, p, site):
        return torch.empty_like(x)

    @fake("disentangled_flash::dropout_layernorm_train")
    def _(x, residual, weight, bias, rng, eps, p, site):
        return (torch.empty_like(x),
                x.new_empty((2, x.numel() // x.shape[-1]), dtype=torch.float32))

    @fake("disentangled_flash::dropout_layernorm_backward")
    def _(dy, x, residual, weight, statistics, rng, p, site, want_x, want_residual, want_weights):
        hidden = x.shape[-1] if want_weights else 0
        return (torch.empty_like(x) if want_x else x.new_empty(0),
                torch.empty_like(x) if want_residual else x.new_empty(0),
                weight.new_empty(hidden), weight.new_empty(hidden))

    @fake("disentangled_flash::embedding_lookup")
    def _(ids, table, scale, padding):
        return table.new_empty(ids.shape + (table.shape[1],))

    @fake("disentangled_flash::embedding_gradient")
    def _(dy, ids, rows, scale, padding):
        return dy.new_empty((rows, dy.shape[-1]))

    @fake("disentangled_flash::orthogonalize")
    def _(update, steps, a, b, c, eps):
        return update.new_empty(update.shape, dtype=torch.bfloat16)

    def contiguous(t):  # the outputs are, whatever the inputs' strides
        return t.new_empty(t.shape)

    @fake("disentangled_flash::attention")
    def _(query, key, value, pos_key, pos_query, delta_to_slot, mask, rng, scale, p, site):
        return contiguous(query)

    @fake("disentangled_flash::attention_train")
    def _(query, key, value, pos_key, pos_query, delta_to_slot, mask, rng, scale, p, site):
        batch, length, heads, _ = query.shape
        row = (length + 63) // 64 * 8
        bits = batch * heads * length * row if p > 0 else 0
        low = query.new_empty(0) if query.dtype == torch.float32 else contiguous(query)
        return (contiguous(query), low,
                query.new_empty((batch, heads, length), dtype=torch.float32),
                query.new_empty(bits, dtype=torch.uint8))

    @fake("disentangled_flash::attention_backward")
    def _(dout, out, low, lse, bits, query, key, value, pos_key, pos_query, delta_to_slot, mask,
          scale, p, want_pos_key, want_pos_query):
        def table(t, wanted):
            if t is None or not wanted:
                return query.new_empty(0)
            return t.new_empty((t.shape[1], t.shape[0], t.shape[2]))

        return (contiguous(query), contiguous(key), contiguous(value),
                table(pos_key, want_pos_key), table(pos_query, want_pos_query))


# ---- operators -----------------------------------------------------------------------


def _check_floating(name: str, tensor: torch.Tensor) -> None:
    if not tensor.is_cuda:
        raise RuntimeError(f"{name} must be on a GPU, is on {tensor.device}")
    if tensor.dtype not in _lib.DTYPE_CODES:
        raise TypeError(f"{name} dtype {tensor.dtype} is not fp16, bf16 or fp32")


_is_batched = torch._C._functorch.is_batchedtensor


def _vmap_levels(tensor: torch.Tensor) -> set[int]:
    """The vmaps, by their levels, over which ``tensor`` holds a value for each sample."""

    levels = set()
    while _is_batched(tensor):
        levels.add(torch._C._functorch.maybe_get_level(tensor))
        tensor = torch._C._functorch.get_unwrapped(tensor)
    return levels


def _check_dropout(p: float, rng: torch.Tensor | None, site: int, like: torch.Tensor) -> None:
    if not 0.0 <= p <= 1.0:  # (NaN too)
        raise ValueError(f"dropout probability must be in [0, 1], got {p}")
    if not 0 <= site < 1 << 32:
        raise ValueError(f"site must be in [0, 2^32), got {site}")
    if p == 0.0:
        return
    if rng is None:
        raise ValueError("dropout needs rng, an int64 tensor [seed, step]")
    if rng.dtype != torch.int64 or rng.shape != (2,) or not rng.is_contiguous():
        raise ValueError(f"rng must be a contiguous int64 tensor [seed, step], got {rng.dtype} "
                         f"{tuple(rng.shape)}")
    if rng.get_device() != like.get_device():
        raise ValueError(f"rng is on {rng.device}, the input on {like.device}")
    if _is_batched(like) and not _vmap_levels(like) <= _vmap_levels(rng):
        raise ValueError("under vmap every sample would drop the same elements: map over rng too, "
                         "[seed, step] of each sample")


def dropout(x: torch.Tensor, p: float, rng: torch.Tensor, site: int = 0) -> torch.Tensor:
    """Drops elements of ``x`` with probability ``p`` and divides the others by ``1 - p``.

    ``rng`` and ``site`` choose the elements (see the module's text).  ``rng`` must keep its
    values until the backward pass has run.  ``p == 0`` returns ``x`` itself.
    """

    p, site = float(p), int(site)
    _check_floating("x", x)
    _check_dropout(p, rng, site, x)
    if p == 0.0:
        return x
    return _ops.dropout(x.contiguous(), rng, p, site)


def layer_norm(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor,
    eps: float,
    residual: torch.Tensor | None = None,
    p: float = 0.0,
    rng: torch.Tensor | None = None,
    site: int = 0,
) -> torch.Tensor:
    """``LayerNorm(dropout(x) + residual)`` over the last dimension, of at most 8192 elements.

    ``weight`` and ``bias`` are of ``x``'s dtype or fp32; the output and the gradients of ``x``
    and ``residual`` are of ``x``'s dtype, those of the weights of theirs.  Everything between
    is fp32 and each result is rounded once (``layers.add_layernorm`` also rounds the
    sum).  ``p``, ``rng`` and ``site`` as in :func:`dropout`.
    """

    p, site, eps = float(p), int(site), float(eps)
    _check_floating("x", x)
    shape, dtype, device = x.shape, x.dtype, x.get_device()
    if not shape or not 1 <= shape[-1] <= MAX_HIDDEN:
        raise ValueError(f"x must be [..., H] with H in [1, {MAX_HIDDEN}], got {tuple(shape)}")
    width, kind = shape[-1:], weight.dtype
    for name, tensor in (("weight", weight), ("bias", bias)):
        if tensor.shape != width:
            raise ValueError(f"{name} must be [H={shape[-1]}], got {tuple(tensor.shape)}")
        if tensor.dtype != kind or (kind != dtype and kind != torch.float32):
            raise TypeError(f"{name} dtype {tensor.dtype}: weight and bias must both have the "
                            f"dtype of x ({dtype}) or both be fp32")
        if tensor.get_device() != device:
            raise ValueError(f"{name} is on {tensor.device}, x on {x.device}")
    if residual is not None:
        if residual.shape != shape or residual.dtype != dtype or residual.get_device() != device:
            raise ValueError(f"residual must match x: {tuple(shape)} {dtype} on {x.device}, got "
                             f"{tuple(residual.shape)} {residual.dtype} on {residual.device}")
        residual = residual.contiguous()
    _check_dropout(p, rng, site, x)
    if p == 0.0:
        rng = None
    elif residual is not None and _is_batched(residual):
        _check_dropout(p, rng, site, residual)
    return _ops.dropout_layernorm(x.contiguous(), residual, weight.contiguous(),
                                  bias.contiguous(), rng, eps, p, site)


def embedding(
    input_ids: torch.Tensor,
    weight: torch.Tensor,
    scale: float = 1.0,
    padding_idx: int | None = None,
) -> torch.Tensor:
    """``scale * weight[input_ids]``, ``[..., H]`` for int32 or int64 ids ``[...]``.

    The gradient of ``weight`` is dense, of its dtype, summed in fp32 and rounded once; the row
    ``padding_idx`` takes none.  An id outside ``[0, V)`` gives a row of NaN and adds to no
    gradient (the ids are on the GPU, so the host cannot refuse them without waiting for it).
    """

    scale = float(scale)
    _check_floating("weight", weight)
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"weight must be [V, H], got {tuple(weight.shape)}")
    if not weight.is_contiguous():
        raise ValueError("weight must be contiguous")
    if input_ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"input_ids dtype {input_ids.dtype} is not int32 or int64")
    if input_ids.get_device() != weight.get_device():
        raise ValueError(f"input_ids are on {input_ids.device}, weight on {weight.device}")
    rows = weight.shape[0]
    padding = -1
    if padding_idx is not None:
        if not -rows <= padding_idx < rows:
            raise ValueError(f"padding_idx {padding_idx} is outside the table of {rows} rows")
        padding = int(padding_idx) % rows
    return _ops.embedding_lookup(input_ids.contiguous(), weight, scale, padding)


def attention(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    pos_key: torch.Tensor | None,
    pos_query: torch.Tensor | None,
    delta_to_slot: torch.Tensor,
    scale: float,
    mask: torch.Tensor | None = None,
    p: float = 0.0,
    rng: torch.Tensor | None = None,
    site: int = 0,
) -> torch.Tensor:
    """Disentangled attention with dropout on its probabilities, ``[B, L, H, d]``.

    The score of query ``i`` and key ``j`` is ``scale * (q_i.k_j + q_i.pos_key[t] +
    k_j.pos_query[t])`` with the learned row ``t = delta_to_slot[i - j + L - 1]`` of the relative
    distance (``position.SharedPositionPlanCache.compact`` has that table, an int32 ``[2L - 1]``).
    An entry outside the tables stands for a row of zeros.

    ``query``, ``key`` and ``value`` are ``[B, L, H, d]`` with ``d`` 32, 64 or 128 and at most
    16384 tokens, ``pos_key`` and ``pos_query`` ``[H, S, d]`` (``None``: no such term), all of one
    dtype; views whose rows of ``d`` start on 16-byte boundaries and, of one head, lie within 2 GiB (the
    projections' outputs do) are read where they lie, others are copied.
    ``mask`` is a bool or uint8 ``[B, L]``, nonzero for tokens that are kept.  A kept query has
    the softmax over the kept keys, whatever the padded places hold; a padded query has ``1 / L``
    for every key, as in Hugging Face's attention (where a padded key's value is not finite it
    counts as 0; a kept key's makes the rows that see it NaN).  ``p``, ``rng`` and ``site`` as in
    :func:`dropout`, on the probabilities ``[B, H, L, L]``.

    Scores, softmax and sums are fp32, the same in both passes.  The output is that of unrounded
    probabilities, rounded once; the backward pass
    rounds probabilities and the scores' gradients to the dtype where they are multiplied.
    Kept for it are the inputs, the output, in 16 bits also what its rounding left off, a
    statistic for each row and with dropout one bit for each probability.  It takes memory for the
    scores' gradients, ``[B, H, L, L]`` of the dtype in parts of up to 2 GiB, and for the sums of the tables'
    gradients by distance, up to ``16 d`` MiB in 16 bits and half of that in fp32.

    ``B H`` is at most 2^20, ``H`` 65535 and ``H S`` below 2^22.
    """

    p, site, scale = float(p), int(site), float(scale)
    _check_floating("query", query)
    shape, dtype, device = query.shape, query.dtype, query.get_device()
    if len(shape) != 4 or shape[3] not in ATTENTION_WIDTHS or shape[2] < 1:
        raise ValueError(f"query must be [B, L, H, d] with d in {ATTENTION_WIDTHS}, "
                         f"got {tuple(shape)}")
    if shape[1] > MAX_LENGTH:
        raise ValueError(f"at most {MAX_LENGTH} tokens, got {shape[1]}")
    for name, tensor in (("key", key), ("value", value)):
        if tensor.shape != shape or tensor.dtype != dtype or tensor.get_device() != device:
            raise ValueError(f"{name} must match query: {tuple(shape)} {dtype} on {query.device}, "
                             f"got {tuple(tensor.shape)} {tensor.dtype} on {tensor.device}")
    if not 0.0 < scale < float("inf"):
        raise ValueError(f"scale must be positive and finite, got {scale}")
    slots = None
    for name, tensor in (("pos_key", pos_key), ("pos_query", pos_query)):
        if tensor is None:
            continue
        if tensor.dim() != 3 or tensor.shape[0] != shape[2] or tensor.shape[2] != shape[3] \
                or tensor.shape[1] < 1:
            raise ValueError(f"{name} must be [H={shape[2]}, S, d={shape[3]}], got "
                             f"{tuple(tensor.shape)}")
        if tensor.dtype != dtype:
            raise TypeError(f"{name} dtype {tensor.dtype} is not that of query ({dtype})")
        if tensor.get_device() != device:
            raise ValueError(f"{name} is on {tensor.device}, query on {query.device}")
        if slots is not None and tensor.shape[1] != slots:
            raise ValueError(f"pos_key has {slots} slots, pos_query {tensor.shape[1]}")
        slots = tensor.shape[1]
    if delta_to_slot.dtype != torch.int32 or delta_to_slot.dim() != 1:
        raise TypeError("delta_to_slot must be a 1-D int32 tensor")
    if shape[1] > 0 and delta_to_slot.shape[0] != 2 * shape[1] - 1:
        raise ValueError(f"delta_to_slot has {delta_to_slot.shape[0]} entries, expected 2L-1 = "
                         f"{2 * shape[1] - 1}")
    if delta_to_slot.get_device() != device:
        raise ValueError(f"delta_to_slot is on {delta_to_slot.device}, query on {query.device}")
    if mask is not None:
        if mask.shape != shape[:2] or mask.dtype not in (torch.bool, torch.uint8):
            raise ValueError(f"mask must be bool or uint8 {tuple(shape[:2])}, got {mask.dtype} "
                             f"{tuple(mask.shape)}")
        if mask.get_device() != device:
            raise ValueError(f"mask is on {mask.device}, query on {query.device}")
        mask = mask.contiguous()
    _check_dropout(p, rng, site, query)
    if p == 0.0:
        rng = None
    else:
        for tensor in (key, value, pos_key, pos_query, mask):
            if tensor is not None and _is_batched(tensor):
                _check_dropout(p, rng, site, tensor)
    return _ops.attention(query, key, value, pos_key, pos_query, delta_to_slot.contiguous(), mask,
                          rng, scale, p, site)


NEWTON_SCHULZ = (3.4445, -4.775, 2.0315)  # the quintic's coefficients that are in common use
_TILE = 128  # of orthogonalize's products


def _check_iterations(batch: int, m: int, n: int, steps: int, eps: float) -> None:
    if steps < 1:
        raise ValueError(f"steps must be at least 1, got {steps}")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    if batch > 65535 or max(m, n) > 1 << 20 or batch * -(-m // _TILE) * -(-n // _TILE) > 1 << 22:
        raise ValueError(f"at most 65535 matrices of at most 2^20 rows and columns and 2^22 tiles of "
                         f"{_TILE} x {_TILE} in all, got {batch} of {m} x {n}")


def orthogonalize(
    update: torch.Tensor,
    steps: int = 5,
    coefficients: tuple[float, float, float] = NEWTON_SCHULZ,
    eps: float = 1e-7,
) -> torch.Tensor:
    """The matrices ``update`` ``[..., m, n]`` with their singular values brought near 1, bf16.

    ``X = update / (|update|_F + eps)``, then ``steps`` times ``X <- a X + (b A + c A A) X`` with
    ``A = X X^T`` (transposed where ``m > n``), as the Muon optimiser takes it: with the usual
    coefficients and five steps, singular values above 1e-3 of the norm come to lie between 0.7 and 1.2.  All matrices
    of a call go through the same launches: at most 65535, of at most 2^20 rows and columns, 2^22 tiles of
    128 x 128 in all.  The products take fp16 operands and fp32
    sums (2e-3 from the formula's result, which bf16 rounds by as much); at every step each singular value
    ``s`` of ``X`` must be below 255 and ``|b s^2 + c s^4|`` below 65504 (with the usual coefficients, which keep
    ``s`` near 1, below 13.4), or the result is not finite.  Not differentiable: the result has no gradient.
    """

    steps, eps = int(steps), float(eps)
    a, b, c = (float(x) for x in coefficients)
    _check_floating("update", update)
    if update.dim() < 2 or update.shape[-1] < 1 or update.shape[-2] < 1:
        raise ValueError(f"update must be [..., m, n], got {tuple(update.shape)}")
    shape = update.shape
    _check_iterations(update.numel() // (shape[-2] * shape[-1]), shape[-2], shape[-1], steps, eps)
    rows = update.detach().reshape(-1, shape[-2], shape[-1]).contiguous()
    return _ops.orthogonalize(rows, steps, a, b, c, eps).view(shape)


# ---- modules ---------------------------------------------------------------------------


# Where torch's generator stood when a state drew a step: (the state's token, device, seed,
# offset) -> that step's rng.  torch.utils.checkpoint puts the generator back for its
# recomputations, so one of a whole backbone finds the step of its forward here.
_drawn: OrderedDict[tuple[int, ...], torch.Tensor] = OrderedDict()
_DRAWN_KEPT = 1 << 12  # forwards whose backward pass is still to come; 512 bytes each on the GPU
_tokens = itertools.count()


def _generator(counter: torch.Tensor) -> Any:
    """torch's generator of the counter's GPU, where its position can be read."""

    if not _lib.runs_directly(counter) or torch.cuda.is_current_stream_capturing():
        return None
    return torch.cuda.default_generators[counter.get_device()]


def _leave_position(counter: torch.Tensor) -> None:
    """Moves torch's generator on, as a dropout of its own would: positions are met once."""

    generator = _generator(counter)
    if generator is not None:
        generator.set_offset(generator.get_offset() + 4)


def _position(counter: torch.Tensor, token: int) -> tuple[int, ...] | None:
    generator = _generator(counter)
    if generator is None:
        return None
    return (token, counter.get_device(), generator.initial_seed(), generator.get_offset())


def _in_backward_pass() -> bool:
    return torch._C._current_graph_task_id() != -1


_UNKNOWN_STEP = (
    "a forward that draws dropout masks ran inside a backward pass, and none began where torch's "
    "generator stands: its masks would not be those of the forward that it recomputes "
    "(torch.utils.checkpoint puts the generator back with preserve_rng_state=True and the input "
    "ids as positional arguments, outside graph capture)")


def _remember(place: tuple[int, ...] | None, rng: torch.Tensor) -> None:
    if place is not None:
        _drawn[place] = rng
        _drawn.move_to_end(place)
        if len(_drawn) > _DRAWN_KEPT:
            _drawn.popitem(last=False)


@torch.library.custom_op("disentangled_flash::next_step", mutates_args=())
def _next_step(counter: torch.Tensor, token: int) -> tuple[torch.Tensor, torch.Tensor]:
    """:meth:`DropoutState.advance` for a traced graph: the counter's new value, and rng."""

    place = _position(counter, token)
    _leave_position(counter)
    if _in_backward_pass():
        if place not in _drawn:
            raise RuntimeError(_UNKNOWN_STEP)
        return counter.clone(), _drawn[place].clone()
    advanced = counter.clone()
    advanced[1:].add_(1)
    _remember(place, advanced.clone())
    return advanced, advanced.clone()


@_next_step.register_fake
def _(counter, token):
    return torch.empty_like(counter), torch.empty_like(counter)


class _Phase:
    """Where a state stands (apart from it: an nn.Module's attributes are slow to set)."""

    begun = False  # the next place that asks for rng advances
    inside = False  # a forward in eval mode runs
    unknown = False  # the forward that is recomputed was not found


class DropoutState(nn.Module):
    """Seed and step of a model's dropout: one buffer that its :class:`Dropout` modules share.

    :meth:`advance` starts the next step.  It adds to the buffer in place (so a captured step
    goes on at every replay) and takes a copy as this step's ``rng``: a forward whose backward
    pass is still to come keeps its own.  The buffer is not saved with the model.
    Between :meth:`begin` and :meth:`end` the first place that asks for ``rng`` advances.

    In a backward pass ``advance`` belongs to a recomputation (``torch.utils.checkpoint`` around
    the backbone): ``rng`` is that of the forward which drew where torch's generator of the GPU
    stands again.  Where there is none (the generator was not put back) asking for it raises.
    Advancing moves that generator on, as ``nn.Dropout`` does.

    :meth:`keep_for` ties a step to a forward's outputs: when their backward pass begins, the
    step's ``rng`` is the current one again, so that layers recomputed in it (checkpointing)
    drop what they dropped, also when another forward ran in between.
    """

    def __init__(self, seed: int, device: torch.device | str | None = None) -> None:
        super().__init__()
        if not -(1 << 63) <= int(seed) < 1 << 63:
            raise ValueError(f"seed must fit 64 bits, got {seed}")
        self.register_buffer("counter", torch.tensor([int(seed), 0], dtype=torch.int64,
                                                     device=device), persistent=False)
        self._rng: torch.Tensor | None = None
        self._phase = _Phase()
        self._token = next(_tokens)

    def __setstate__(self, state: dict[str, Any]) -> None:
        super().__setstate__(state)
        self._phase, self._token = _Phase(), next(_tokens)  # (a copy draws steps of its own)

    @property
    def rng(self) -> torch.Tensor:
        if self._phase.begun:
            # (The place that asks may lie in a checkpointed layer, whose recomputation does not
            # come here: inside a forward torch's generator stays where it is until the end.)
            self._advance(moves=not self._phase.inside)
        if self._phase.unknown:
            raise RuntimeError(_UNKNOWN_STEP)
        if self._rng is None or self._rng.device != self.counter.device:
            self._rng = self._copy()
        return self._rng

    def _copy(self) -> torch.Tensor:
        """The counter's values; not an inference tensor, since a training forward may come to it."""

        with torch.inference_mode(False):
            return self.counter.clone()

    def begin(self) -> None:
        self._phase.begun = self._phase.inside = True

    def end(self) -> bool:
        """Whether rng was asked for since :meth:`begin`."""

        self._phase.inside = False
        if not self._phase.begun:
            _leave_position(self.counter)
        return not self._phase.begun

    def advance(self) -> None:
        self._advance(moves=True)

    @torch.no_grad()
    def _advance(self, moves: bool) -> None:
        phase = self._phase
        phase.begun = phase.unknown = False
        if torch.compiler.is_compiling():
            advanced, self._rng = _next_step(self.counter, self._token)
            self.counter.copy_(advanced)
            return
        place = _position(self.counter, self._token)
        if moves:
            _leave_position(self.counter)
        if _in_backward_pass():
            self._rng = _drawn.get(place)
            phase.unknown = self._rng is None  # (an error where masks are drawn)
            return
        self.counter[1:].add_(1)
        self._rng = self._copy()
        _remember(place, self._rng)

    def keep_for(self, outputs: Any) -> None:
        if self._phase.unknown:
            return
        rng = self.rng

        def restore(_: torch.Tensor) -> None:
            self._rng = rng
            self._phase.begun = self._phase.unknown = False

        pending = [outputs]
        while pending:
            item = pending.pop()
            if isinstance(item, torch.Tensor):
                if item.requires_grad:
                    item.register_hook(restore)
            elif isinstance(item, Mapping):
                pending.extend(item.values())
            elif isinstance(item, (tuple, list)):
                pending.extend(item)


class Dropout(nn.Dropout):
    """``nn.Dropout`` on :func:`dropout`: the identity in eval mode, torch's for float64.

    Called again before the next :meth:`DropoutState.advance` it drops the same elements, which
    is what recomputing a checkpointed layer needs.
    """

    def __init__(self, p: float, state: DropoutState, site: int) -> None:
        _check_dropout(p, state.counter, site, state.counter)
        super().__init__(p)
        self.site = site
        self.__dict__["state"] = state  # the model's, registered there once

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if not self.training or self.p == 0:
            return x
        if self.inplace or (_on_gpu(x) and x.dtype not in _lib.DTYPE_CODES):
            return super().forward(x)
        return dropout(x, self.p, self.state.rng, self.site)

    def extra_repr(self) -> str:
        return f"p={self.p}, site={self.site}"


def _on_gpu(x: torch.Tensor) -> bool:
    return x.device.type == "cuda"


def _single(*tensors: torch.Tensor) -> tuple[torch.Tensor, ...]:
    """As ``torch.autocast`` gives them to torch's own LayerNorm: 16 bits become fp32."""

    return tuple(t.float() if t.dtype in (torch.float16, torch.bfloat16) else t for t in tensors)


def _types_fit(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor) -> bool:
    """Whether :func:`layer_norm` takes these types."""

    kind = weight.dtype
    return (x.dtype in _lib.DTYPE_CODES and kind == bias.dtype
            and (kind == x.dtype or kind == torch.float32))


def _norm_is_affine(norm: nn.LayerNorm) -> bool:
    """Over the last dimension, with weight and bias, and as wide as :func:`layer_norm` takes."""

    return (norm.weight is not None and norm.bias is not None and len(norm.normalized_shape) == 1
            and norm.normalized_shape[0] <= MAX_HIDDEN)


class LayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` on :func:`layer_norm`; torch's on the CPU and for types and settings that
    the operator lacks.  Under ``torch.autocast`` in fp32, as torch's."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if not _on_gpu(x) or not _norm_is_affine(self):
            return super().forward(x)
        rows, weight, bias = x, self.weight, self.bias
        if torch.is_autocast_enabled("cuda"):
            rows, weight, bias = _single(rows, weight, bias)
        if not _types_fit(rows, weight, bias):
            return super().forward(x)
        return layer_norm(rows, weight, bias, self.eps)


def _settings_fit(module: nn.Embedding) -> bool:
    """Whether :func:`embedding` and its dense gradient are what the module asks for."""

    return module.max_norm is None and not module.sparse and not module.scale_grad_by_freq


class Embedding(nn.Embedding):
    """``nn.Embedding`` on :func:`embedding`; torch's on the CPU and for types, settings and
    strides that the operator lacks."""

    def forward(self, input_ids: torch.Tensor) -> torch.Tensor:
        weight = self.weight
        if not _on_gpu(input_ids) or not _settings_fit(self) \
                or weight.dtype not in _lib.DTYPE_CODES or not weight.is_contiguous():
            return super().forward(input_ids)
        return embedding(input_ids, weight, padding_idx=self.padding_idx)


class OutputBlock(nn.Module):
    """``LayerNorm(dropout(dense(x)) + input)`` with the sub-modules of a Hugging Face
    ``DebertaV2SelfOutput`` / ``DebertaV2Output`` under their names.

    Dropout, sum and norm are one call while ``LayerNorm`` and ``dropout`` are what they were:
    where one is replaced or has hooks, they are called themselves.
    """

    def __init__(self, dense: nn.Module, norm: nn.LayerNorm, drop: Dropout) -> None:
        super().__init__()
        self.dense = dense
        self.LayerNorm = norm
        self.dropout = drop

    def forward(self, hidden_states: torch.Tensor, input_tensor: torch.Tensor) -> torch.Tensor:
        x = self.dense(hidden_states)
        norm, drop = self.LayerNorm, self.dropout
        if not (_on_gpu(x) and _norm_fits(norm) and _dropout_fits(drop)) \
                or _hooks_on_all_modules():
            return norm(drop(x) + input_tensor)
        rows, residual, weight, bias = x, input_tensor, norm.weight, norm.bias
        if torch.is_autocast_enabled("cuda"):  # (the norm's part of it; 16-bit sums are not rounded)
            rows, residual, weight, bias = _single(rows, residual, weight, bias)
        if rows.dtype != residual.dtype:  # as their sum promotes them
            dtype = torch.promote_types(rows.dtype, residual.dtype)
            rows, residual = rows.to(dtype), residual.to(dtype)
        if not _types_fit(rows, weight, bias):
            return norm(drop(x) + input_tensor)
        dropping = drop.training and drop.p > 0
        return layer_norm(rows, weight, bias, norm.eps, residual=residual,
                          p=drop.p if dropping else 0.0, rng=drop.state.rng if dropping else None,
                          site=drop.site)


class _PositionPlans:
    """Slots and places of relative distances for each length, and whether the slots in use are
    successive rows of the table (then they are a view of it)."""

    def __init__(self, attention: nn.Module) -> None:
        self.cache = SharedPositionPlanCache(
            position_buckets=attention.position_buckets,
            max_relative_positions=attention.max_relative_positions,
            position_embedding_size=attention.pos_ebd_size)
        self.ranges: dict[int, tuple[int, int] | None] = {}

    def of(self, length: int, device: torch.device) -> tuple[Any, tuple[int, int] | None]:
        if length not in self.ranges:
            slots = self.cache.compact(length, "cpu").active_slots
            first, last = int(slots[0]), int(slots[-1])
            self.ranges[length] = (first, last + 1) if last - first + 1 == len(slots) else None
        return self.cache.compact(length, device), self.ranges[length]


def _is_factorized(mask: Any) -> bool:
    """The form in which :class:`_EncoderParts` hands a padding mask on: ``[B, 1, L, 1, 1]``, of a
    dimension more than any mask that an attention takes."""

    return isinstance(mask, torch.Tensor) and mask.dim() == 5


class _Attention:
    """The forward of a Hugging Face ``DisentangledSelfAttention`` on :func:`attention`.

    Its projections and its dropouts stay the modules that they are.  What the operator lacks (the
    CPU, other dtypes and head widths, attention probabilities as an output, masks of pairs, relative
    positions given by the caller) and children that were replaced or have hooks go to the
    original's forward.
    """

    def forward(self, hidden_states, attention_mask, output_attentions=False, query_states=None,
                relative_pos=None, rel_embeddings=None):
        if _is_factorized(attention_mask):
            mask = attention_mask[:, 0, :, 0, 0]
            if relative_pos is None and not output_attentions:
                out = self._fused(hidden_states, mask,
                                  hidden_states if query_states is None else query_states,
                                  rel_embeddings)
                if out is not None:
                    return out, None
            attention_mask = mask[:, None, None, :] * mask[:, None, :, None]
        return super().forward(hidden_states, attention_mask, output_attentions,
                               query_states=query_states, relative_pos=relative_pos,
                               rel_embeddings=rel_embeddings)

    def _fused(self, hidden_states, mask, query_states, rel_embeddings):
        drop = self.dropout
        terms = [m for m in ("c2p", "p2c") if m in self.pos_att_type]  # (the scale counts them)
        modes = terms if self.relative_attention else []
        if not (_on_gpu(hidden_states) and self.attention_head_size in ATTENTION_WIDTHS
                and 1 <= hidden_states.shape[1] <= MAX_LENGTH
                and query_states.shape == hidden_states.shape
                and all(n in (1, m) for n, m in zip(mask.shape, hidden_states.shape))
                and _dropout_fits(drop) and not _hooks_on_all_modules()
                and (not modes or (rel_embeddings is not None
                                   and rel_embeddings.shape[0] >= 2 * self.pos_ebd_size))):
            return None
        batch, length = hidden_states.shape[:2]
        shape = (batch, length, self.num_attention_heads, self.attention_head_size)
        query, key, value = (projection(x).view(shape) for projection, x in (
            (self.query_proj, query_states), (self.key_proj, hidden_states),
            (self.value_proj, hidden_states)))
        pos_key = pos_query = None
        if modes:
            plan, rows = self._plans.of(length, hidden_states.device)
            used = self.pos_dropout(rel_embeddings)
            used = used[rows[0]:rows[1]] if rows else used.index_select(0, plan.active_slots)
            shared = self.share_att_key

            def table(projection):
                return projection(used).view(-1, *shape[2:]).transpose(0, 1)

            if "c2p" in modes:
                pos_key = table(self.key_proj if shared else self.pos_key_proj)
            if "p2c" in modes:
                pos_query = table(self.query_proj if shared else self.pos_query_proj)
            places = plan.delta_to_local
        else:
            places = self._no_places(length, hidden_states.device)
        tensors = [t for t in (query, key, value, pos_key, pos_query) if t is not None]
        dtype = query.dtype
        if dtype not in _lib.DTYPE_CODES or any(t.dtype != dtype for t in tensors):
            return None
        dropping = drop.training and drop.p > 0
        out = attention(query, key, value, pos_key, pos_query, places,
                        1 / math.sqrt(self.attention_head_size * (1 + len(terms))),
                        mask=mask.bool().expand(batch, length), p=drop.p if dropping else 0.0,
                        rng=drop.state.rng if dropping else None, site=drop.site)
        return out.view(batch, length, -1)

    @staticmethod
    def _no_places(length, device):
        return torch.zeros(2 * length - 1, dtype=torch.int32, device=device)


class _EncoderParts:
    """Stands for ``get_attention_mask`` or ``get_rel_pos`` of a Hugging Face encoder whose
    attention is :class:`_Attention`: a padding mask stays ``[B, L]`` values, and the
    relative positions are left to the attention.  Anything else is the encoder's own."""

    def __init__(self, encoder: nn.Module, name: str) -> None:
        self.encoder, self.name = encoder, name

    def __call__(self, *args: Any, **kwargs: Any) -> Any:
        encoder = self.encoder
        own = getattr(type(encoder), self.name)
        if not all(isinstance(layer.attention.self, _Attention) for layer in encoder.layer):
            return own(encoder, *args, **kwargs)
        if self.name == "get_attention_mask":
            mask = args[0] if args else kwargs.get("attention_mask")
            if isinstance(mask, torch.Tensor) and mask.dim() == 2:
                return mask[:, None, :, None, None]
        elif (args[2] if len(args) > 2 else kwargs.get("relative_pos")) is None:
            return None
        return own(encoder, *args, **kwargs)


_attention_class: type | None = None


def __getattr__(name: str) -> Any:
    """``DisentangledSelfAttention``: Hugging Face's with the forward of :class:`_Attention` (made when
    first asked for: this module does without transformers)."""

    global _attention_class
    if name != "DisentangledSelfAttention":
        raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
    if _attention_class is None:
        from transformers.models.deberta_v2.modeling_deberta_v2 import DisentangledSelfAttention

        _attention_class = type("DisentangledSelfAttention", (_Attention, DisentangledSelfAttention),
                                {"__module__": __name__, "__doc__": _Attention.__doc__})
    return _attention_class


def _is_attention(module: nn.Module) -> bool:
    kind = type(module)
    return (kind.__name__ == "DisentangledSelfAttention" and kind.__module__ == _OUTPUT_BLOCKS_FROM
            and kind.forward.__module__ == _OUTPUT_BLOCKS_FROM)


def _fuse_attention(encoder: nn.Module) -> None:
    """Gives every attention of the encoder the fused forward, in place; none of them where one
    is not Hugging Face's own, or has hooks."""

    modules = [layer.attention.self for layer in encoder.layer]
    if not modules or not all(_is_attention(m) and not _has_hooks(m) for m in modules):
        raise TypeError("the encoder's attention is not transformers' DisentangledSelfAttention")
    if type(encoder).__module__ != _OUTPUT_BLOCKS_FROM:
        raise TypeError("the encoder is not transformers' DebertaV2Encoder")
    plans = None
    for module in modules:
        if module.relative_attention and plans is None:
            plans = _PositionPlans(module)
        module.__class__ = __getattr__("DisentangledSelfAttention")
        module.__dict__["_plans"] = plans
    for name in ("get_attention_mask", "get_rel_pos"):
        encoder.__dict__[name] = _EncoderParts(encoder, name)


_OUTPUT_BLOCKS = ("DebertaV2SelfOutput", "DebertaV2Output")
_OUTPUT_BLOCKS_FROM = "transformers.models.deberta_v2.modeling_deberta_v2"


def _is_output_block(module: nn.Module) -> bool:
    kind = type(module)
    return (kind.__name__ in _OUTPUT_BLOCKS and kind.__module__ == _OUTPUT_BLOCKS_FROM
            and kind.forward.__module__ == _OUTPUT_BLOCKS_FROM)


def _has_hooks(module: nn.Module) -> bool:
    return bool(module._forward_hooks or module._forward_pre_hooks or module._backward_hooks
                or module._backward_pre_hooks or "forward" in module.__dict__)


def _hooks_on_all_modules() -> bool:
    return bool(torch_module._global_forward_hooks or torch_module._global_forward_pre_hooks
                or torch_module._global_backward_hooks or torch_module._global_backward_pre_hooks)


def _norm_fits(module: Any) -> bool:
    """Whether calling ``module`` is :func:`layer_norm` of its weights and nothing else."""

    return ((type(module) is nn.LayerNorm or type(module) is LayerNorm)
            and _norm_is_affine(module) and not _has_hooks(module))


def _dropout_fits(module: Any) -> bool:
    return type(module) is Dropout and not module.inplace and not _has_hooks(module)


def _adopt(made: nn.Module, module: nn.Module) -> nn.Module:
    """``made`` (built empty) with the parameters and the mode of ``module``."""

    made._parameters.update(module._parameters)
    return made.train(module.training)


def _training_form(module: nn.Module, state: DropoutState, sites: Any) -> nn.Module:
    """The module that takes ``module``'s place; itself where nothing here computes it."""

    if _has_hooks(module):
        return module
    if type(module) is nn.Dropout and not module.inplace:
        return Dropout(module.p, state, next(sites)).train(module.training)
    if type(module) is nn.LayerNorm and _norm_fits(module):
        made = LayerNorm(module.normalized_shape, module.eps, device="meta")
        return _adopt(made, module)
    if type(module) is nn.Embedding and _settings_fit(module):
        made = Embedding(module.num_embeddings, module.embedding_dim, module.padding_idx,
                         device="meta")
        return _adopt(made, module)
    if _is_output_block(module):
        children = dict(module.named_children())
        drop = children.get("dropout")
        if set(children) == {"dense", "LayerNorm", "dropout"} and type(drop) is nn.Dropout \
                and _norm_fits(children["LayerNorm"]) and not _has_hooks(drop):
            made = OutputBlock(children["dense"], children["LayerNorm"],
                               Dropout(drop.p, state, next(sites)).train(drop.training))
            made.training = module.training
            return made
    return module


def _advance_state(model: nn.Module, args: Any) -> None:
    if model.training:
        model.dropout_state.advance()
    else:  # parts of it may be in training mode
        model.dropout_state.begin()


def _keep_state(model: nn.Module, args: Any, outputs: Any) -> None:
    state = model.dropout_state
    if model.training or state.end():
        state.keep_for(outputs)


def enable_deberta_training(
    model: nn.Module, *, seed: int = 0, attention: str = "torch"
) -> nn.Module:
    """Put the training operators into a HF DeBERTa-v2/v3 backbone, in place.

    ``model`` is the Hugging Face backbone (the module with ``embeddings`` and ``encoder``), as
    for ``optimize_deberta``.  Its ``nn.Embedding``, ``nn.LayerNorm`` and ``nn.Dropout`` modules
    and its output blocks are replaced; parameters stay the same objects under the same names,
    so checkpoints, tied weights and an optimizer made before are not affected.  Modules with
    hooks and settings that the operators lack (a sparse or renormalised embedding, a norm
    without weights) stay as they are.

    Every training forward of the backbone starts with ``model.dropout_state.advance()``, and
    its backward pass has the same step again, so what is checkpointed (a layer, or the whole
    backbone) recomputes what it computed.  A forward of a backbone in eval mode advances where a
    dropout in training mode first drops (Monte Carlo dropout, a few layers in training).

    ``attention="hip"`` runs the backbone's attention on :func:`attention` too (its projections stay
    torch's products): no ``[L, L]`` tensor of scores or probabilities is made, and the same
    probabilities are dropped as with ``"torch"``, which leaves the attention as it is.
    """

    from .deberta import DebertaV2InferenceEncoder, resolve_backend

    if not (hasattr(model, "encoder") and hasattr(model, "embeddings")):
        raise TypeError("model must be a Hugging Face DeBERTa-v2/v3 backbone")
    if isinstance(model.encoder, DebertaV2InferenceEncoder):
        raise TypeError("the model's encoder is inference-only (DebertaV2InferenceEncoder)")
    if hasattr(model, "dropout_state"):
        raise TypeError("the model already uses the training operators")
    if resolve_backend(attention) == "hip":
        _fuse_attention(model.encoder)
    state = DropoutState(seed, next(model.parameters()).device)
    sites = iter(range(1 << 32))
    places: list[nn.Module] = [model]
    for parent in places:
        for name, child in list(parent.named_children()):
            made = _training_form(child, state, sites)
            if made is not child:
                setattr(parent, name, made)
            elif child not in places:
                places.append(child)
    model.dropout_state = state
    model.register_forward_pre_hook(_advance_state)
    model.register_forward_hook(_keep_state)
    return model


# ---- optimiser ---------------------------------------------------------------------------


def split_parameters(model: nn.Module) -> tuple[list[nn.Parameter], list[nn.Parameter]]:
    """(the weights of the encoder's ``nn.Linear`` layers, all other parameters), those that require a
    gradient: the former for :class:`Muon`, the latter for another optimiser."""

    encoder = getattr(model, "encoder", model)
    matrices = {id(m.weight): m.weight for m in encoder.modules()
                if isinstance(m, nn.Linear) and m.weight.requires_grad}
    rest = [p for p in model.parameters() if p.requires_grad and id(p) not in matrices]
    return list(matrices.values()), rest


class Muon(torch.optim.Optimizer):
    """Muon on :func:`orthogonalize`, for matrices: ``B <- momentum B + g``; the update is
    ``g + momentum B`` (``B`` without ``nesterov``), orthogonalised;
    ``p <- (1 - lr weight_decay) p - lr r update``.

    ``adjust_lr_fn`` chooses ``r`` for
    ``[m, n]``: ``"original"`` (the default) ``sqrt(max(1, m / n))``, ``"match_rms_adamw"``
    ``0.2 sqrt(max(m, n))``.  Parameters of one shape, dtype and device are orthogonalised by one call.  They must be on
    a GPU, in fp16, bf16 or fp32; the momentum is kept in the parameter's dtype.

    Names and defaults are those of ``torch.optim.Muon``, whose ``momentum_buffer`` however is an average:
    ``B <- momentum B + (1 - momentum) g``, and the update ``(1 - momentum) g + momentum B``.
    ``average=True`` takes that rule.  While ``momentum`` stays what it is both rules take the same steps, but for
    ``eps``, since an update's length does not count; where it changes they differ.  States are interchangeable
    with torch's under ``average=True`` alone: one that does not say which of the two it holds is
    refused.  A sum of steady gradients is ``1 / (1 - momentum)`` times as large as they are, which in fp16 may
    pass 65504; an average never does.  Unlike torch's, ``momentum`` must be below 1, and ``eps`` is added
    to an update's norm.
    """

    def __init__(self, params: Iterable[Any], lr: float = 1e-3, weight_decay: float = 0.1,
                 momentum: float = 0.95, nesterov: bool = True,
                 ns_coefficients: tuple[float, float, float] = NEWTON_SCHULZ, eps: float = 1e-7,
                 ns_steps: int = 5, adjust_lr_fn: str | None = None,
                 average: bool = False) -> None:
        if not lr >= 0.0:
            raise ValueError(f"lr must not be negative, got {lr}")
        if not 0.0 <= momentum < 1.0:
            raise ValueError(f"momentum must be in [0, 1), got {momentum}")
        if not weight_decay >= 0.0:
            raise ValueError(f"weight_decay must not be negative, got {weight_decay}")
        if adjust_lr_fn not in (None, "original", "match_rms_adamw"):
            raise ValueError(f"adjust_lr_fn must be 'original' or 'match_rms_adamw', got "
                             f"{adjust_lr_fn!r}")
        super().__init__(params, dict(lr=lr, weight_decay=weight_decay, momentum=momentum,
                                      nesterov=nesterov, ns_coefficients=ns_coefficients, eps=eps,
                                      ns_steps=ns_steps, adjust_lr_fn=adjust_lr_fn,
                                      average=bool(average)))

    def __setstate__(self, state: dict[str, Any]) -> None:
        super().__setstate__(state)
        for group in self.param_groups:
            group.setdefault("average", False)

    def load_state_dict(self, state_dict: dict[str, Any]) -> None:
        for group in state_dict["param_groups"]:
            if "average" not in group:
                raise ValueError(
                    "the state does not say what its momentum_buffer holds: set 'average' in each of its "
                    "param_groups, to True for a state of torch.optim.Muon and to False for a sum of gradients")
        super().load_state_dict(state_dict)

    def add_param_group(self, param_group: dict[str, Any]) -> None:
        super().add_param_group(param_group)
        for p in self.param_groups[-1]["params"]:
            if p.dim() != 2 or p.numel() == 0:
                del self.param_groups[-1]
                raise ValueError(f"parameters must be matrices, got {tuple(p.shape)}")

    @torch.no_grad()
    def step(self, closure: Any = None) -> Any:
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        alike: dict[Any, list[nn.Parameter]] = {}
        for n, group in enumerate(self.param_groups):
            for p in group["params"]:
                if p.grad is not None:
                    if p.grad.is_sparse:
                        raise RuntimeError("sparse gradients are not supported")
                    _check_floating("parameters", p)
                    alike.setdefault((n, p.shape, p.dtype, p.device), []).append(p)
        for (n, shape, *_), params in alike.items():
            group = self.param_groups[n]
            _check_iterations(len(params), *shape, int(group["ns_steps"]), float(group["eps"]))
        # (What is refused is refused before any group's momentum or weights change.)
        for (n, shape, dtype, _), params in alike.items():
            self._update(self.param_groups[n], shape, dtype, params)
        return loss

    def _update(self, group: dict[str, Any], shape: torch.Size, dtype: torch.dtype,
                params: list[nn.Parameter]) -> None:
        grads = [p.grad for p in params]
        for p in params:
            if "momentum_buffer" not in self.state[p]:
                self.state[p]["momentum_buffer"] = torch.zeros_like(p)
        buffers = [self.state[p]["momentum_buffer"] for p in params]
        momentum, updates = float(group["momentum"]), buffers
        if group["average"]:
            torch._foreach_lerp_(buffers, grads, 1.0 - momentum)
            if group["nesterov"]:
                updates = torch._foreach_lerp(grads, buffers, momentum)
        else:
            torch._foreach_mul_(buffers, momentum)
            torch._foreach_add_(buffers, grads)
            if group["nesterov"]:
                updates = torch._foreach_add(grads, buffers, alpha=momentum)
        rows, columns, lr = *shape, float(group["lr"])
        if group["adjust_lr_fn"] == "match_rms_adamw":
            ratio = 0.2 * math.sqrt(max(rows, columns))
        else:
            ratio = math.sqrt(max(1.0, rows / columns))
        turned = orthogonalize(torch.stack(updates), group["ns_steps"], group["ns_coefficients"],
                               group["eps"]).to(dtype)
        torch._foreach_mul_(params, 1.0 - lr * group["weight_decay"])
        torch._foreach_add_(params, list(turned.unbind()), alpha=-lr * ratio)


__all__ = [
    "Dropout",
    "DropoutState",
    "Embedding",
    "LayerNorm",
    "Muon",
    "OutputBlock",
    "attention",
    "dropout",
    "embedding",
    "enable_deberta_training",
    "layer_norm",
    "orthogonalize",
    "split_parameters",
]
