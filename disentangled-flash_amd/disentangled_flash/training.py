"""Operators of a DeBERTa training step around its matrix products, and the modules that call them.

The operators, on a GPU in fp16, bf16 and fp32, with their gradients:

* :func:`layer_norm` - ``LayerNorm(dropout(x) + residual)``, the tail of every output block
  (``DebertaV2SelfOutput`` / ``DebertaV2Output``, reference ``_reference.py:101-112`` and
  ``474-485``, which in training drops elements between its dense layer and its residual);
  without residual and dropout a plain LayerNorm.
* :func:`dropout` - dropout whose mask comes from a counter-based generator and is drawn
  again in the backward pass instead of being stored.
* :func:`embedding` - the table lookup with a scale, and the dense gradient of the table,
  summed in an order that depends on the ids alone (the same bits on every call).

:func:`enable_deberta_training` puts them into a Hugging Face DeBERTa-v2/v3 backbone;
``optimize_deberta`` takes the same model afterwards for inference.

**Random numbers** are an input: ``rng`` is an int64 tensor ``[seed, step]`` on the GPU, read
by the kernels, so that a captured step that advances it drops other elements on every
replay; ``site`` numbers the places of a model that drop elements.  An element is dropped by
its index in the flattened tensor, ``rng`` and ``site`` alone, whatever the dtype.  ``p`` is
rounded to a multiple of 2^-16 (to 0 and 1 only where it is 0 or 1), and kept elements are
divided by the rounded probability of being kept.  A dropped element is 0 whatever it held.

Work is launched on torch's current stream of the inputs' device.  Second derivatives are not
implemented (they raise).  Inputs that are not contiguous are copied first.
"""

from __future__ import annotations

import contextlib
from typing import Any

import torch
from torch import nn
from torch.autograd.function import once_differentiable
from torch.nn import functional as F

from . import _lib

MAX_HIDDEN = 8192  # widest row of layer_norm


def _device_of(tensor: torch.Tensor):
    """Makes ``tensor``'s device the current one (the library launches on the current device)."""

    if tensor.device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(tensor.device)


def _pointer(tensor: torch.Tensor | None) -> int | None:
    return None if tensor is None else tensor.data_ptr()


# ---- ops: one library call each ----------------------------------------------------


@_lib.hip_op("disentangled_flash::dropout")
def dropout_op(x: torch.Tensor, rng: torch.Tensor, p: float, site: int) -> torch.Tensor:
    """``x`` with the elements of ``(rng, site)`` dropped; ``x`` contiguous."""

    lib = _lib.load()
    out = torch.empty_like(x)
    with _device_of(x):
        code = lib.dflash_dropout(x.data_ptr(), out.data_ptr(), x.numel(), p, rng.data_ptr(), site,
                                  _lib.DTYPE_CODES[x.dtype], _lib.current_stream_handle(x.device))
    _lib.check(code, "dflash_dropout")
    return out


@dropout_op.register_fake
def _dropout_fake(x, rng, p, site):
    return torch.empty_like(x)


@_lib.hip_op("disentangled_flash::dropout_layernorm")
def dropout_layernorm_op(
    x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, bias: torch.Tensor,
    rng: torch.Tensor | None, eps: float, p: float, site: int, statistics: bool
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(y, mean, rstd)``; the statistics are empty unless asked for."""

    lib = _lib.load()
    hidden = x.shape[-1]
    rows = x.numel() // hidden
    y = torch.empty_like(x)
    kept = torch.empty((2, rows if statistics else 0), device=x.device, dtype=torch.float32)
    mean, rstd = kept[0], kept[1]
    with _device_of(x):
        code = lib.dflash_dropout_layernorm_fwd(
            x.data_ptr(), _pointer(residual), weight.data_ptr(), bias.data_ptr(), y.data_ptr(),
            mean.data_ptr() if statistics else None, rstd.data_ptr() if statistics else None,
            rows, hidden, eps, p, _pointer(rng), site, _lib.DTYPE_CODES[x.dtype],
            _lib.DTYPE_CODES[weight.dtype], _lib.current_stream_handle(x.device))
    _lib.check(code, "dflash_dropout_layernorm_fwd")
    return y, mean, rstd


@dropout_layernorm_op.register_fake
def _dropout_layernorm_fake(x, residual, weight, bias, rng, eps, p, site, statistics):
    rows = x.numel() // x.shape[-1] if statistics else 0
    mean, rstd = (x.new_empty(rows, dtype=torch.float32) for _ in range(2))
    return torch.empty_like(x), mean, rstd


@_lib.hip_op("disentangled_flash::dropout_layernorm_backward")
def dropout_layernorm_backward_op(
    dy: torch.Tensor, x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor,
    mean: torch.Tensor, rstd: torch.Tensor, rng: torch.Tensor | None, p: float, site: int,
    want_x: bool, want_residual: bool, want_weights: bool
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(dx, dresidual, dweight, dbias)``; those not wanted are empty."""

    lib = _lib.load()
    hidden = x.shape[-1]
    rows = x.numel() // hidden
    dx = torch.empty_like(x) if want_x else x.new_empty(0)
    dresidual = torch.empty_like(x) if want_residual else x.new_empty(0)
    dweight = weight.new_empty(hidden if want_weights else 0)
    dbias = weight.new_empty(hidden if want_weights else 0)
    size = lib.dflash_dropout_layernorm_bwd_workspace_bytes(rows, hidden) if want_weights else 0
    workspace = torch.empty(size, device=x.device, dtype=torch.uint8)
    with _device_of(x):
        code = lib.dflash_dropout_layernorm_bwd(
            dy.data_ptr(), x.data_ptr(), _pointer(residual), weight.data_ptr(), mean.data_ptr(),
            rstd.data_ptr(), dx.data_ptr() if want_x else None,
            dresidual.data_ptr() if want_residual else None,
            dweight.data_ptr() if want_weights else None,
            dbias.data_ptr() if want_weights else None, rows, hidden, p, _pointer(rng), site,
            _lib.DTYPE_CODES[x.dtype], _lib.DTYPE_CODES[weight.dtype], workspace.data_ptr(), size,
            _lib.current_stream_handle(x.device))
    _lib.check(code, "dflash_dropout_layernorm_bwd")
    return dx, dresidual, dweight, dbias


@dropout_layernorm_backward_op.register_fake
def _dropout_layernorm_backward_fake(dy, x, residual, weight, mean, rstd, rng, p, site, want_x,
                                     want_residual, want_weights):
    hidden = x.shape[-1] if want_weights else 0
    return (torch.empty_like(x) if want_x else x.new_empty(0),
            torch.empty_like(x) if want_residual else x.new_empty(0),
            weight.new_empty(hidden), weight.new_empty(hidden))


@_lib.hip_op("disentangled_flash::embedding_lookup")
def embedding_op(input_ids: torch.Tensor, weight: torch.Tensor, scale: float) -> torch.Tensor:
    """``scale * weight[input_ids]``; both contiguous."""

    lib = _lib.load()
    rows, hidden = weight.shape
    out = weight.new_empty(*input_ids.shape, hidden)
    with _device_of(weight):
        code = lib.dflash_embedding_fwd(
            input_ids.data_ptr(), weight.data_ptr(), out.data_ptr(), input_ids.numel(), rows,
            hidden, scale, input_ids.element_size(), _lib.DTYPE_CODES[weight.dtype],
            _lib.current_stream_handle(weight.device))
    _lib.check(code, "dflash_embedding_fwd")
    return out


@embedding_op.register_fake
def _embedding_fake(input_ids, weight, scale):
    return weight.new_empty(*input_ids.shape, weight.shape[1])


@_lib.hip_op("disentangled_flash::embedding_gradient")
def embedding_gradient_op(dy: torch.Tensor, input_ids: torch.Tensor, rows: int, scale: float,
                          padding_idx: int) -> torch.Tensor:
    """The table's dense gradient ``[rows, H]``; ``padding_idx`` -1: none."""

    lib = _lib.load()
    hidden = dy.shape[-1]
    tokens = input_ids.numel()
    out = dy.new_empty(rows, hidden)
    size = lib.dflash_embedding_bwd_workspace_bytes(tokens, hidden)
    workspace = torch.empty(size, device=dy.device, dtype=torch.uint8)
    with _device_of(dy):
        code = lib.dflash_embedding_bwd(
            input_ids.data_ptr(), dy.data_ptr(), out.data_ptr(), tokens, rows, hidden, scale,
            padding_idx, input_ids.element_size(), _lib.DTYPE_CODES[dy.dtype],
            workspace.data_ptr(), size, _lib.current_stream_handle(dy.device))
    _lib.check(code, "dflash_embedding_bwd")
    return out


@embedding_gradient_op.register_fake
def _embedding_gradient_fake(dy, input_ids, rows, scale, padding_idx):
    return dy.new_empty(rows, dy.shape[-1])


# ---- operators -----------------------------------------------------------------------


def _check_floating(name: str, tensor: torch.Tensor) -> None:
    if tensor.device.type != "cuda":
        raise RuntimeError(f"{name} must be on a GPU, is on {tensor.device}")
    if tensor.dtype not in _lib.DTYPE_CODES:
        raise TypeError(f"{name} dtype {tensor.dtype} is not fp16, bf16 or fp32")


def _check_dropout(p: float, rng: torch.Tensor | None, site: int, device: torch.device) -> None:
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
    if rng.device != device:
        raise ValueError(f"rng is on {rng.device}, the input on {device}")


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, rng, p, site):
        ctx.save_for_backward(rng)
        ctx.p, ctx.site = p, site
        return dropout_op(x, rng, p, site)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        (rng,) = ctx.saved_tensors
        return dropout_op(dy.contiguous(), rng, ctx.p, ctx.site), None, None, None


def dropout(x: torch.Tensor, p: float, rng: torch.Tensor, site: int = 0) -> torch.Tensor:
    """Drops elements of ``x`` with probability ``p`` and divides the others by ``1 - p``.

    ``rng`` and ``site`` choose the elements (see the module's text).  ``rng`` must keep its
    values until the backward pass has run.  ``p == 0`` returns ``x`` itself.
    """

    p, site = float(p), int(site)
    _check_floating("x", x)
    _check_dropout(p, rng, site, x.device)
    if p == 0.0:
        return x
    x = x.contiguous()
    if torch.is_grad_enabled() and x.requires_grad:
        return _Dropout.apply(x, rng, p, site)
    return dropout_op(x, rng, p, site)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, rng, eps, p, site):
        y, mean, rstd = dropout_layernorm_op(x, residual, weight, bias, rng, eps, p, site, True)
        ctx.save_for_backward(x, residual, weight, mean, rstd, rng)
        ctx.p, ctx.site = p, site
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, residual, weight, mean, rstd, rng = ctx.saved_tensors
        want_x, want_weight, want_bias, want_residual = ctx.needs_input_grad[:4]
        # Without dropout the gradients of x and of the residual are the same tensor.
        shared = ctx.p == 0.0 and want_residual
        dx, dresidual, dweight, dbias = dropout_layernorm_backward_op(
            dy.contiguous(), x, residual, weight, mean, rstd, rng, ctx.p, ctx.site,
            want_x or shared, want_residual and not shared, want_weight or want_bias)
        return (dx if want_x else None, dweight if want_weight else None,
                dbias if want_bias else None,
                (dx if shared else dresidual) if want_residual else None, None, None, None, None)


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
    if x.dim() == 0 or not 1 <= x.shape[-1] <= MAX_HIDDEN:
        raise ValueError(f"x must be [..., H] with H in [1, {MAX_HIDDEN}], got {tuple(x.shape)}")
    for name, tensor in (("weight", weight), ("bias", bias)):
        if tensor.shape != x.shape[-1:]:
            raise ValueError(f"{name} must be [H={x.shape[-1]}], got {tuple(tensor.shape)}")
        if tensor.dtype not in (x.dtype, torch.float32) or tensor.dtype != weight.dtype:
            raise TypeError(f"{name} dtype {tensor.dtype}: weight and bias must both have the "
                            f"dtype of x ({x.dtype}) or both be fp32")
        if tensor.device != x.device:
            raise ValueError(f"{name} is on {tensor.device}, x on {x.device}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype
                                 or residual.device != x.device):
        raise ValueError(f"residual must match x: {tuple(x.shape)} {x.dtype} on {x.device}, got "
                         f"{tuple(residual.shape)} {residual.dtype} on {residual.device}")
    _check_dropout(p, rng, site, x.device)
    if p == 0.0:
        rng = None
    x, weight, bias = x.contiguous(), weight.contiguous(), bias.contiguous()
    residual = None if residual is None else residual.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or bias.requires_grad
                                    or (residual is not None and residual.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, residual, rng, eps, p, site)
    return dropout_layernorm_op(x, residual, weight, bias, rng, eps, p, site, False)[0]


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, input_ids, weight, scale, padding_idx):
        ctx.save_for_backward(input_ids)
        ctx.rows, ctx.scale, ctx.padding_idx = weight.shape[0], scale, padding_idx
        return embedding_op(input_ids, weight, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        (input_ids,) = ctx.saved_tensors
        return None, embedding_gradient_op(dy.contiguous(), input_ids, ctx.rows, ctx.scale,
                                           ctx.padding_idx), None, None


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
    if input_ids.device != weight.device:
        raise ValueError(f"input_ids are on {input_ids.device}, weight on {weight.device}")
    rows = weight.shape[0]
    padding = -1
    if padding_idx is not None:
        if not -rows <= padding_idx < rows:
            raise ValueError(f"padding_idx {padding_idx} is outside the table of {rows} rows")
        padding = int(padding_idx) % rows
    input_ids = input_ids.contiguous()
    if torch.is_grad_enabled() and weight.requires_grad:
        return _Embedding.apply(input_ids, weight, scale, padding)
    return embedding_op(input_ids, weight, scale)


# ---- modules ---------------------------------------------------------------------------


class DropoutState(nn.Module):
    """Seed and step of a model's dropout: one buffer that its :class:`Dropout` modules share.

    :meth:`advance` starts the next step.  It adds to the buffer in place (so a captured step
    goes on at every replay) and takes a copy as this step's ``rng``: a forward whose backward
    pass is still to come keeps its own.  The buffer is not saved with the model.
    """

    def __init__(self, seed: int, device: torch.device | str | None = None) -> None:
        super().__init__()
        if not -(1 << 63) <= int(seed) < 1 << 63:
            raise ValueError(f"seed must fit 64 bits, got {seed}")
        self.register_buffer("counter", torch.tensor([int(seed), 0], dtype=torch.int64,
                                                     device=device), persistent=False)
        self._rng: torch.Tensor | None = None

    @property
    def rng(self) -> torch.Tensor:
        if self._rng is None or self._rng.device != self.counter.device:
            self._rng = self.counter.clone()
        return self._rng

    @torch.no_grad()
    def advance(self) -> None:
        self.counter[1:].add_(1)
        self._rng = self.counter.clone()


class Dropout(nn.Module):
    """``nn.Dropout`` on :func:`dropout`: the identity in eval mode.

    Called again before the next :meth:`DropoutState.advance` it drops the same elements, which
    is what recomputing a checkpointed layer needs.
    """

    def __init__(self, p: float, state: DropoutState, site: int) -> None:
        super().__init__()
        _check_dropout(0.0 if p == 0 else p, state.counter, site, state.counter.device)
        self.p = p
        self.site = site
        self.__dict__["state"] = state  # the model's, registered there once

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if not self.training or self.p == 0:
            return x
        return dropout(x, self.p, self.state.rng, self.site)

    def extra_repr(self) -> str:
        return f"p={self.p}, site={self.site}"


class LayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` over the last dimension on :func:`layer_norm`; torch's on the CPU."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.device.type != "cuda":
            return super().forward(x)
        return layer_norm(x, self.weight, self.bias, self.eps)


class Embedding(nn.Embedding):
    """``nn.Embedding`` on :func:`embedding`; torch's on the CPU."""

    def forward(self, input_ids: torch.Tensor) -> torch.Tensor:
        if input_ids.device.type != "cuda":
            return super().forward(input_ids)
        return embedding(input_ids, self.weight, padding_idx=self.padding_idx)


class OutputBlock(nn.Module):
    """``LayerNorm(dropout(dense(x)) + input)`` with the sub-modules of a Hugging Face
    ``DebertaV2SelfOutput`` / ``DebertaV2Output`` under their names."""

    def __init__(self, dense: nn.Module, norm: nn.LayerNorm, drop: Dropout) -> None:
        super().__init__()
        self.dense = dense
        self.LayerNorm = norm
        self.dropout = drop

    def forward(self, hidden_states: torch.Tensor, input_tensor: torch.Tensor) -> torch.Tensor:
        x = self.dense(hidden_states)
        norm, drop = self.LayerNorm, self.dropout
        if x.device.type != "cuda":
            return norm(drop(x) + input_tensor)
        if x.dtype != input_tensor.dtype:  # (under autocast: as the sum would promote them)
            dtype = torch.promote_types(x.dtype, input_tensor.dtype)
            x, input_tensor = x.to(dtype), input_tensor.to(dtype)
        dropping = drop.training and drop.p > 0
        return layer_norm(x, norm.weight, norm.bias, norm.eps, residual=input_tensor,
                          p=drop.p if dropping else 0.0, rng=drop.state.rng if dropping else None,
                          site=drop.site)


_OUTPUT_BLOCKS = ("DebertaV2SelfOutput", "DebertaV2Output")


def _has_hooks(module: nn.Module) -> bool:
    return bool(module._forward_hooks or module._forward_pre_hooks or module._backward_hooks
                or module._backward_pre_hooks or "forward" in module.__dict__)


def _norm_fits(module: Any) -> bool:
    return (isinstance(module, nn.LayerNorm) and module.weight is not None
            and module.bias is not None and len(module.normalized_shape) == 1
            and module.normalized_shape[0] <= MAX_HIDDEN and not _has_hooks(module))


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
    if type(module) is nn.Embedding and module.max_norm is None and not module.sparse \
            and not module.scale_grad_by_freq:
        made = Embedding(module.num_embeddings, module.embedding_dim, module.padding_idx,
                         device="meta")
        return _adopt(made, module)
    if type(module).__name__ in _OUTPUT_BLOCKS:
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


def enable_deberta_training(model: nn.Module, *, seed: int = 0) -> nn.Module:
    """Put the training operators into a HF DeBERTa-v2/v3 backbone, in place.

    ``model`` is the Hugging Face backbone (the module with ``embeddings`` and ``encoder``), as
    for ``optimize_deberta``.  Its ``nn.Embedding``, ``nn.LayerNorm`` and ``nn.Dropout`` modules
    and its output blocks are replaced; parameters stay the same objects under the same names,
    so checkpoints, tied weights and an optimizer made before are not affected.  Modules with
    hooks and settings that the operators lack (a sparse or renormalised embedding, a norm
    without weights) stay as they are.

    Every training forward of the backbone starts with ``model.dropout_state.advance()``.
    Checkpointing single layers is fine; recomputing the whole backbone would draw new masks.
    """

    from .deberta import DebertaV2InferenceEncoder

    if not (hasattr(model, "encoder") and hasattr(model, "embeddings")):
        raise TypeError("model must be a Hugging Face DeBERTa-v2/v3 backbone")
    if isinstance(model.encoder, DebertaV2InferenceEncoder):
        raise TypeError("the model's encoder is inference-only (DebertaV2InferenceEncoder)")
    if hasattr(model, "dropout_state"):
        raise TypeError("the model already uses the training operators")
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
    return model


__all__ = [
    "Dropout",
    "DropoutState",
    "Embedding",
    "LayerNorm",
    "OutputBlock",
    "dropout",
    "embedding",
    "enable_deberta_training",
    "layer_norm",
]
