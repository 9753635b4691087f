"""The training operators of the package as cases that can be timed.

Three operators of a DeBERTa training step, as a user calls them:

* ``norm`` - ``training.layer_norm``: LayerNorm of ``dropout(x) + residual`` (the tail of
  every output block) or of ``x`` alone, with its backward pass;
* ``dropout`` - ``training.dropout``: dropout whose mask comes from a counter-based
  generator and is never stored;
* ``embedding`` - ``training.embedding``: the scaled lookup and the dense gradient of its
  table.

With ``own`` true, :func:`run` calls the package; with ``own`` false it computes the same
values from elementary torch operations in 32 bits, rounded once at the end.

The generator's output is part of an operator's definition, so both forms drop the same
elements: Philox4x32 with 7 rounds (Salmon, Moraes, Dror and Shaw, SC'11), keyed by the
64-bit seed ``rng[0]``.  One call serves eight consecutive elements of the flattened tensor;
its counter is (index of the eight, low and high word; site; step ``rng[1]``).  Element e of
the eight takes 16 bits of word e / 2, the low half first, and is kept where they are at
least ``round(65536 * p)``; kept elements are divided by the probability of being kept.
"""

from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

_PACKAGE = os.path.abspath("disentangled-flash_amd")
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SITE = 5  # the number of the call's place in a model
VOCABULARY = 128100


def _norm(name, batch, length, hidden, dtype, residual, p, backward, weights="same"):
    case = {"op": "norm", "batch": batch, "length": length, "hidden": hidden, "dtype": dtype,
            "residual": residual, "p": p, "backward": backward, "weights": weights}
    return {"name": name, **case} if name else case


def _dropout(name, batch, length, hidden, dtype, p, backward):
    case = {"op": "dropout", "batch": batch, "length": length, "hidden": hidden, "dtype": dtype,
            "p": p, "backward": backward}
    return {"name": name, **case} if name else case


def _embedding(name, batch, length, rows, hidden, dtype, ids, scale, padding, backward):
    case = {"op": "embedding", "batch": batch, "length": length, "rows": rows, "hidden": hidden,
            "dtype": dtype, "ids": ids, "scale": scale, "padding": padding, "backward": backward}
    return {"name": name, **case} if name else case


def listed():
    return [
        # The tail of an output block in a training step of the 12-layer base model at the
        # benchmark's batch: the most frequent call of the three.
        _norm("norm_tail_base", 32, 512, 768, "bf16", True, 0.1, True),
        # The same tail for one short sequence: latency is everything.
        _norm("norm_tail_short", 1, 17, 768, "fp16", True, 0.1, True),
        # The widest model in full precision.
        _norm("norm_tail_xlarge_fp32", 32, 512, 1536, "fp32", True, 0.1, True),
        # The norm after the embeddings: no residual, no dropout before it, and weights kept
        # in fp32 beside half-precision activations.
        _norm("norm_embeddings", 32, 512, 1024, "fp16", False, 0.0, True, "fp32"),
        # A forward pass alone (a validation loss with dropout left on), a ragged batch
        # and a width that no vector load divides.
        _norm("norm_odd_forward", 7, 437, 1001, "bf16", True, 0.1, False),
        # Attention probabilities, 8 sequences of 512 tokens and 12 heads: the largest mask of
        # a training step.
        _dropout("dropout_probabilities", 8 * 12, 512, 512, "bf16", 0.1, True),
        # Hidden states in full precision, forward only.
        _dropout("dropout_hidden_fp32", 16, 384, 768, "fp32", 0.1, False),
        # One short sequence of an odd width.
        _dropout("dropout_odd", 1, 97, 769, "fp16", 0.5, True),
        # Word embeddings of the base model at the benchmark's batch: word-like frequencies and
        # padding that takes no gradient.
        _embedding("embedding_words", 32, 512, VOCABULARY, 768, "bf16", "zipf", 1.0, True, True),
        # The widest model's table: writing the dense gradient is most of the work.
        _embedding("embedding_words_xlarge", 32, 512, VOCABULARY, 1536, "fp16", "zipf", 1.0, True,
                   True),
        # One query of a server: a lookup of a few rows in a large table.
        _embedding("embedding_query", 1, 17, VOCABULARY, 768, "fp16", "zipf", 1.0, False, False),
        # Absolute positions: a small table, every row used by every sequence, scaled.
        _embedding("embedding_positions", 32, 512, 512, 1024, "fp32", "positions", 32.0, False,
                   True),
    ]


def _spread(rng, low, high):
    """A whole number from [low, high], even over its logarithm."""

    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _shape(rng, most):
    """Batch and length of at most ``most`` tokens, lengths up to 512."""

    length = _spread(rng, 1, 512)
    return _spread(rng, 1, max(1, min(32, most // length))), length


def _width(rng):
    """A model's width, a multiple of 8 near it, or any whole number."""

    kind = rng.random()
    if kind < 0.5:
        return rng.choice([64, 384, 512, 768, 1024, 1536])
    width = _spread(rng, 32, 1536)
    return max(32, width // 8 * 8) if kind < 0.75 else width


def draw(rng):
    op = rng.choice(["norm", "dropout", "embedding"])
    dtype = rng.choice(["fp16", "bf16", "fp32"])
    backward = rng.random() < 0.7
    batch, length = _shape(rng, 16384)
    if op == "norm":
        residual = rng.random() < 0.7
        p = rng.choice([0.0, 0.1, 0.1, round(rng.uniform(0.01, 0.6), 3)])
        return _norm(None, batch, length, _width(rng), dtype, residual, p, backward,
                     rng.choice(["same", "same", "fp32"]))
    if op == "dropout":
        p = rng.choice([0.1, 0.1, round(rng.uniform(0.01, 0.9), 3)])
        return _dropout(None, batch, length, _width(rng), dtype, p, backward)
    rows = _spread(rng, 2, VOCABULARY)
    width = _width(rng) if dtype != "fp32" else min(_width(rng), 768)
    ids = rng.choice(["zipf", "zipf", "uniform", "positions"])
    scale = rng.choice([1.0, 1.0, round(math.sqrt(width), 3)])
    return _embedding(None, batch, length, rows, width, dtype, ids, scale, rng.random() < 0.5,
                      backward)


def work(case):
    tokens, hidden = case["batch"] * case["length"], case["hidden"]
    size = 4 if case["dtype"] == "fp32" else 2
    n = tokens * hidden
    if case["op"] == "norm":
        wsize = 4 if case["weights"] == "fp32" else size
        inputs = 2 if case["residual"] else 1
        moved = n * size * (inputs + 1) + 2 * hidden * wsize
        flops = 8 * n
        if case["backward"]:
            # dy once more, and a gradient for every input; without dropout the residual's
            # and x's gradients are equal, and one write serves both.
            grads = 2 if case["residual"] and case["p"] > 0 else 1
            moved += n * size * (1 + grads) + 2 * hidden * wsize
            flops += 14 * n
        return {"bytes": moved, "flops": flops}
    if case["op"] == "dropout":
        passes = 2 if case["backward"] else 1
        return {"bytes": 2 * n * size * passes, "flops": n * passes}
    moved = tokens * 8 + min(tokens, case["rows"]) * hidden * size + n * size
    flops = n
    if case["backward"]:
        moved += n * size + case["rows"] * hidden * size
        flops += n
    return {"bytes": moved, "flops": flops}


# ---- inputs ------------------------------------------------------------------

def _ids(case, gen):
    batch, length, rows = case["batch"], case["length"], case["rows"]
    if case["ids"] == "positions":
        ids = (torch.arange(length, device="cuda") % rows).repeat(batch, 1)
    elif case["ids"] == "uniform":
        ids = torch.randint(0, rows, (batch, length), device="cuda", generator=gen)
    else:
        # P(id) ~ 1 / (id + 1), as a vocabulary sorted by frequency is used.
        u = torch.rand(batch, length, device="cuda", generator=gen, dtype=torch.float64)
        ids = (torch.exp(u * math.log(rows + 1)).long() - 1).clamp_(0, rows - 1)
    if case["padding"]:
        kept = torch.randint((length + 1) // 2, length + 1, (batch, 1), device="cuda",
                             generator=gen)
        ids = ids.masked_fill(torch.arange(length, device="cuda")[None] >= kept, 0)
    return ids


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]
    shape = (case["batch"], case["length"], case["hidden"])

    def normal(size, scale=1.0, at=0.0, kind=dtype):
        return (torch.randn(size, device="cuda", generator=gen) * scale + at).to(kind)

    state = {"case": case}
    backward = case["backward"]
    if case["op"] in ("norm", "dropout"):
        state["rng"] = torch.randint(0, 1 << 62, (2,), device="cuda", generator=gen)
        state["rng"][1] %= 100000
        state["x"] = normal(shape).requires_grad_(backward)
    if case["op"] == "norm":
        weights = torch.float32 if case["weights"] == "fp32" else dtype
        hidden = case["hidden"]
        state["weight"] = normal(hidden, 0.1, 1.0, weights).requires_grad_(backward)
        state["bias"] = normal(hidden, 0.1, 0.0, weights).requires_grad_(backward)
        state["eps"] = 1e-7
        if case["residual"]:
            state["residual"] = normal(shape, 1.3, 0.25).requires_grad_(backward)
    if case["op"] == "embedding":
        state["weight"] = normal((case["rows"], case["hidden"]), 0.02).requires_grad_(backward)
        state["ids"] = _ids(case, gen)
    if backward:
        state["dy"] = normal(shape)
    return state


# ---- the passes --------------------------------------------------------------

def run(state):
    case = state["case"]
    return _run_own(state, case) if own else _PLAIN[case["op"]](state, case)


def _run_own(state, case):
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    from disentangled_flash import training

    if case["op"] == "norm":
        residual = state.get("residual")
        y = training.layer_norm(state["x"], state["weight"], state["bias"], state["eps"],
                                residual=residual, p=case["p"], rng=state["rng"], site=SITE)
        leaves = [state["x"], state["weight"], state["bias"]]
        if residual is not None:
            leaves.append(residual)
    elif case["op"] == "dropout":
        y = training.dropout(state["x"], case["p"], state["rng"], site=SITE)
        leaves = [state["x"]]
    else:
        y = training.embedding(state["ids"], state["weight"], scale=case["scale"],
                               padding_idx=0 if case["padding"] else None)
        leaves = [state["weight"]]
    if not case["backward"]:
        return (y,)
    return (y.detach(), *torch.autograd.grad(y, leaves, state["dy"]))


def _plain_factor(shape, p, rng):
    """What an element is multiplied by: 0 or the inverse of the kept share, 32 bits."""

    n = math.prod(shape)
    blocks = (n + 7) // 8
    low = 0xFFFFFFFF
    index = torch.arange(blocks, device="cuda")
    seed = rng[0]
    k0, k1 = seed & low, (seed >> 32) & low
    c0, c1 = index & low, index >> 32
    c2 = torch.full_like(index, SITE)
    c3 = (rng[1] & low).expand(blocks)
    for _ in range(7):
        # (64-bit products wrap; the words cut out of them are the unsigned ones.)
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack([c0, c1, c2, c3], dim=1)
    halves = torch.stack([words & 0xFFFF, words >> 16], dim=2).reshape(-1)[:n].reshape(shape)
    limit = _limit(p)
    return (halves >= limit).float() * (65536.0 / (65536 - limit))


def _limit(p):
    return min(65535, max(1, round(65536 * p)))


def _plain_norm(state, case):
    x, w, b = state["x"].detach(), state["weight"].detach(), state["bias"].detach()
    dtype, p = x.dtype, case["p"]
    factor = _plain_factor(x.shape, p, state["rng"]) if p > 0 else None
    s = x.float() if factor is None else x.float() * factor
    if case["residual"]:
        s = s + state["residual"].detach().float()
    mean = s.mean(-1, keepdim=True)
    centred = s - mean
    rstd = (centred.square().mean(-1, keepdim=True) + state["eps"]).rsqrt()
    normal = centred * rstd
    y = (normal * w.float() + b.float()).to(dtype)
    if not case["backward"]:
        return (y,)
    dy = state["dy"].float()
    g = dy * w.float()
    ds = rstd * (g - g.mean(-1, keepdim=True) - normal * (g * normal).mean(-1, keepdim=True))
    dx = ds if factor is None else ds * factor
    dw = (dy * normal).flatten(0, -2).sum(0)
    db = dy.flatten(0, -2).sum(0)
    out = [y, dx.to(dtype), dw.to(w.dtype), db.to(b.dtype)]
    if case["residual"]:
        out.append(ds.to(dtype))
    return tuple(out)


def _plain_dropout(state, case):
    x = state["x"].detach()
    factor = _plain_factor(x.shape, case["p"], state["rng"])
    y = (x.float() * factor).to(x.dtype)
    if not case["backward"]:
        return (y,)
    return y, (state["dy"].float() * factor).to(x.dtype)


def _plain_embedding(state, case):
    weight, ids = state["weight"].detach(), state["ids"]
    y = (weight[ids].float() * case["scale"]).to(weight.dtype)
    if not case["backward"]:
        return (y,)
    dw = torch.zeros(weight.shape, device="cuda")
    dw.index_add_(0, ids.flatten(), state["dy"].flatten(0, -2).float())
    if case["padding"]:
        dw[0] = 0
    return y, (dw * case["scale"]).to(weight.dtype)


_PLAIN = {"norm": _plain_norm, "dropout": _plain_dropout, "embedding": _plain_embedding}


# ---- the definitions in 64 bits -----------------------------------------------

def _exact_factor(shape, p, rng):
    """The generator on the host, with numpy's unsigned words."""

    seed, step = (int(v) for v in rng.cpu())
    n = math.prod(shape)
    blocks = -(-n // 8)
    index = np.arange(blocks, dtype=np.uint64)
    mask, shift = np.uint64(0xFFFFFFFF), np.uint64(32)
    counter = [index & mask, index >> shift, np.full(blocks, SITE, np.uint64),
               np.full(blocks, step & 0xFFFFFFFF, np.uint64)]
    key = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    for _ in range(7):
        first = counter[0] * np.uint64(0xD2511F53)
        second = counter[2] * np.uint64(0xCD9E8D57)
        counter = [(second >> shift) ^ counter[1] ^ np.uint64(key[0]), second & mask,
                   (first >> shift) ^ counter[3] ^ np.uint64(key[1]), first & mask]
        key = [(key[0] + 0x9E3779B9) & 0xFFFFFFFF, (key[1] + 0xBB67AE85) & 0xFFFFFFFF]
    fields = np.empty((blocks, 8), np.uint16)
    for word in range(4):
        fields[:, 2 * word] = counter[word] & np.uint64(0xFFFF)
        fields[:, 2 * word + 1] = counter[word] >> np.uint64(16)
    limit = _limit(p)
    kept = torch.from_numpy(fields.reshape(-1)[:n] >= limit).to("cuda").reshape(shape)
    return kept.double() / ((65536 - limit) / 65536)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "embedding":
        return _exact_embedding(state, case)
    x = state["x"].detach().double().requires_grad_()
    y, leaves = x, [x]
    if case["p"] > 0:
        y = x * _exact_factor(tuple(x.shape), case["p"], state["rng"])
    if case["op"] == "norm":
        w, b = (state[k].detach().double().requires_grad_() for k in ("weight", "bias"))
        leaves += [w, b]
        if case["residual"]:
            leaves.append(state["residual"].detach().double().requires_grad_())
            y = y + leaves[-1]
        variance, mean = torch.var_mean(y, -1, correction=0, keepdim=True)
        y = (y - mean) / torch.sqrt(variance + state["eps"]) * w + b
    if not case["backward"]:
        return (y.detach(),)
    return (y.detach(), *torch.autograd.grad(y, leaves, state["dy"].double()))


def _exact_embedding(state, case):
    weight, ids = state["weight"].detach(), state["ids"]
    y = weight.index_select(0, ids.flatten()).double().mul_(case["scale"]).view(*ids.shape, -1)
    if not case["backward"]:
        return (y,)
    dy = state["dy"].double().flatten(0, -2)
    if case["padding"]:
        dy[ids.flatten() == 0] = 0
    order = ids.flatten().argsort(stable=True)
    used, counts = torch.unique_consecutive(ids.flatten()[order], return_counts=True)
    ends = counts.cumsum(0)
    sums = dy[order].cumsum(0)[ends - 1]
    sums[1:] -= sums[:-1].clone()
    dw = torch.zeros(weight.shape, device="cuda", dtype=torch.float64)
    dw[used] = sums * case["scale"]
    return y, dw
