"""The attention and the optimiser's update of a training step as cases that can be timed.

Two operators of a DeBERTa training step, as a user calls them:

* ``attention`` - ``training.attention``: disentangled attention whose learned position rows are
  chosen by the log bucket of the relative distance, with dropout on the probabilities, and its
  backward pass (gradients of queries, keys, values and both position tables);
* ``orthogonalize`` - ``training.orthogonalize``: Newton-Schulz iterations on a batch of update
  matrices of one shape, as ``training.Muon`` takes them.

With ``own`` true, :func:`run` calls the package; with ``own`` false it computes the same
values from elementary torch operations in 32 bits, rounded once at the end.

Dropped probabilities come from the package's generator, which is part of the operator's
definition (``perf/operators.py`` states it): Philox4x32 with 7 rounds over the flattened
[B, H, L, L] tensor, eight elements a call, 16 bits each.
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
SITE = 3  # the number of the call's place in a model
BUCKETS = 256  # log buckets of the relative distance
MAX_DISTANCE = 512
COEFFICIENTS = (3.4445, -4.775, 2.0315)
EPS = 1e-7


def _attention(name, batch, length, heads, dim, dtype, modes, fill, p, backward):
    case = {"op": "attention", "batch": batch, "length": length, "heads": heads, "dim": dim,
            "dtype": dtype, "modes": modes, "fill": fill, "p": p, "backward": backward}
    return {"name": name, **case} if name else case


def _orthogonalize(name, count, rows, columns, dtype, spectrum):
    case = {"op": "orthogonalize", "count": count, "rows": rows, "columns": columns,
            "dtype": dtype, "spectrum": spectrum, "steps": 5}
    return {"name": name, **case} if name else case


def listed():
    return [
        # A layer of the 12-layer base model at the benchmark's batch, padded sequences.
        _attention("attention_base", 32, 512, 12, 64, "bf16", "both", "ragged", 0.1, True),
        # The same layer for one short sequence: latency is everything.
        _attention("attention_short", 1, 17, 12, 64, "fp16", "both", "full", 0.1, True),
        # The widest model at a middle length, where the deltas' share of the work is larger.
        _attention("attention_xlarge", 16, 200, 24, 64, "bf16", "both", "ragged", 0.1, True),
        # Full precision.
        _attention("attention_fp32", 8, 384, 12, 64, "fp32", "both", "ragged", 0.1, True),
        # Long documents: most deltas share a bucket with others.
        _attention("attention_long", 2, 2000, 12, 64, "bf16", "both", "ragged", 0.1, True),
        # Wide heads, one term, forward only (a validation loss with dropout left on).
        _attention("attention_d128_forward", 7, 437, 8, 128, "fp16", "c2p", "ragged", 0.1, False),
        # Narrow heads, the other term, no dropout.
        _attention("attention_d32", 16, 384, 16, 32, "fp16", "p2c", "full", 0.0, True),
        # The attention projections of the 12-layer base model: one batch of 48 squares.
        _orthogonalize("ortho_base", 48, 768, 768, "bf16", "decay"),
        # FFN weights of the widest model from an fp32 momentum, wide ...
        _orthogonalize("ortho_xlarge", 4, 1536, 6144, "fp32", "normal"),
        # ... and tall.
        _orthogonalize("ortho_tall", 1, 6144, 1536, "bf16", "normal"),
        # One small matrix (a classifier's pooler of a small model): latency.
        _orthogonalize("ortho_small", 1, 256, 256, "fp32", "normal"),
        # Sizes that no tile divides.
        _orthogonalize("ortho_odd", 3, 437, 1001, "fp16", "decay"),
    ]


def _spread(rng, low, high):
    """A whole number from [low, high], even over its logarithm."""

    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    if rng.random() < 0.65:
        dtype = rng.choice(["fp16", "bf16", "bf16", "fp32"])
        dim = rng.choice([32, 64, 64, 128])
        length = _spread(rng, 1, 2048)
        # B H L^2 d of the largest listed case of the type, at most
        most = (8 * 12 * 384 * 384 if dtype == "fp32" else 32 * 12 * 512 * 512) * 64
        groups = max(1, most // (length * length * dim))
        heads = min(rng.choice([1, 2, 3, 6, 8, 12, 16, 24]), groups)
        batch = _spread(rng, 1, max(1, min(32, groups // heads, 16384 // length)))
        return _attention(None, batch, length, heads, dim, dtype,
                          rng.choice(["both", "both", "c2p", "p2c"]),
                          rng.choice(["full", "ragged"]),
                          rng.choice([0.0, 0.1, 0.1, round(rng.uniform(0.01, 0.6), 3)]),
                          rng.random() < 0.7)
    rows, columns = _spread(rng, 8, 2048), _spread(rng, 8, 6144)
    if rng.random() < 0.5:
        rows, columns = max(8, rows // 8 * 8), max(8, columns // 8 * 8)
    if rng.random() < 0.3:
        rows, columns = columns, rows
    small, large = min(rows, columns), max(rows, columns)
    most = 4 * 1536 * 1536 * 6144
    if small > 1536:
        small = 1536
        rows, columns = min(rows, small) if rows < columns else rows, \
            columns if rows < columns else min(columns, small)
        small, large = min(rows, columns), max(rows, columns)
    count = _spread(rng, 1, max(1, min(48, most // (small * small * large))))
    return _orthogonalize(None, count, rows, columns, rng.choice(["fp16", "bf16", "fp32"]),
                          rng.choice(["normal", "decay"]))


# ---- the work ----------------------------------------------------------------

def _kept(case):
    """Kept tokens of each sequence: spread evenly over [L / 2, L] where they are ragged."""

    batch, length = case["batch"], case["length"]
    if case["fill"] == "full":
        return [length] * batch
    low = (length + 1) // 2
    return [low + round((length - low) * (b + 1) / batch) for b in range(batch)]


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "orthogonalize":
        m, n = sorted((case["rows"], case["columns"]))
        # X X^T and A A are symmetric: half of each.
        each = m * m * n + m ** 3 + 2 * m * m * n
        return {"bytes": case["count"] * m * n * (size + 2),
                "flops": case["count"] * case["steps"] * each}
    b, length, h, d = (case[k] for k in ("batch", "length", "heads", "dim"))
    slots = int(_slots(length)[0].numel())
    terms = 2 if case["modes"] == "both" else 1
    tensor, table = b * length * h * d * size, slots * h * d * size
    pairs = sum(n * n for n in _kept(case)) * h * d
    relative = sum(_kept(case)) * slots * h * d * terms
    moved = 4 * tensor + terms * table
    flops = 4 * pairs + 2 * relative
    if case["backward"]:
        # q, k, v, the output and its gradient again, three gradients, the tables' gradients.
        moved += 8 * tensor + 2 * terms * table
        flops += 10 * pairs + 6 * relative
    return {"bytes": moved, "flops": flops}


# ---- inputs ------------------------------------------------------------------

def _slots(length):
    """(slots in use, the place of slot(i - j) among them at i - j + L - 1)."""

    middle = BUCKETS // 2
    delta = torch.arange(1 - length, length, dtype=torch.float64)
    far = delta.abs().clamp(min=middle)
    bucket = torch.ceil(torch.log(far / middle) / math.log((MAX_DISTANCE - 1) / middle)
                        * (middle - 1)) + middle
    slot = torch.where(delta.abs() <= middle, delta, bucket * delta.sign()).long()
    slot = (slot + BUCKETS).clamp(0, 2 * BUCKETS - 1)
    used, place = torch.unique(slot, return_inverse=True)
    return used, place.to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]

    def normal(size, scale=1.0):
        return (torch.randn(size, device="cuda", generator=gen) * scale).to(dtype)

    if case["op"] == "orthogonalize":
        m, n, count = case["rows"], case["columns"], case["count"]
        update = torch.randn((count, m, n), device="cuda", generator=gen)
        if case["spectrum"] == "decay":
            # As a momentum has it: a few strong directions above a weak rest.
            r = max(1, min(m, n) // 16)
            strong = torch.randn((count, m, r), device="cuda", generator=gen)
            falling = torch.logspace(0, -2, r, device="cuda")
            strong = strong * falling @ torch.randn((count, r, n), device="cuda", generator=gen)
            update = strong + 0.05 * update
        return {"case": case, "update": (update * 1e-3).to(dtype)}

    b, length, h, d = (case[k] for k in ("batch", "length", "heads", "dim"))
    used, place = _slots(length)
    backward = case["backward"]
    state = {"case": case, "delta_to_slot": place.cuda()}
    for name in ("query", "key", "value"):
        state[name] = normal((b, length, h * d)).requires_grad_(backward)
    for name, mode in (("pos_key", "c2p"), ("pos_query", "p2c")):
        state[name] = normal((used.numel(), h * d)).requires_grad_(backward) \
            if case["modes"] in ("both", mode) else None
    state["scale"] = 1 / math.sqrt(d * (3 if case["modes"] == "both" else 2))
    kept = torch.tensor(_kept(case), device="cuda")
    kept = kept[torch.randperm(b, device="cuda", generator=gen)]
    state["mask"] = torch.arange(length, device="cuda")[None] < kept[:, None]
    state["rng"] = torch.randint(0, 1 << 62, (2,), device="cuda", generator=gen)
    state["rng"][1] %= 100000
    if backward:
        state["dy"] = normal((b, length, h, d))
    return state


# ---- the passes --------------------------------------------------------------

def run(state):
    case = state["case"]
    return _run_own(state, case) if own else _PLAIN[case["op"]](state, case)


def _run_own(state, case):
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    from disentangled_flash import training

    if case["op"] == "orthogonalize":
        return training.orthogonalize(state["update"], steps=case["steps"],
                                      coefficients=COEFFICIENTS, eps=EPS)
    b, length, h, d = (case[k] for k in ("batch", "length", "heads", "dim"))
    leaves = [state[k] for k in ("query", "key", "value")]
    tables = [state["pos_key"], state["pos_query"]]
    heads = [t.view(b, length, h, d) for t in leaves]
    rows = [None if t is None else t.view(-1, h, d).transpose(0, 1) for t in tables]
    y = training.attention(*heads, *rows, state["delta_to_slot"], state["scale"],
                           mask=state["mask"], p=case["p"], rng=state["rng"], site=SITE)
    if not case["backward"]:
        return (y,)
    leaves += [t for t in tables if t is not None]
    return (y.detach(), *torch.autograd.grad(y, leaves, state["dy"]))


def _plain_orthogonalize(state, case):
    g = state["update"].float()
    tall = case["rows"] > case["columns"]
    x = g.transpose(1, 2) if tall else g
    x = x / (x.square().sum((1, 2), keepdim=True).sqrt() + EPS)
    a, b, c = COEFFICIENTS
    for _ in range(case["steps"]):
        s = x @ x.transpose(1, 2)
        x = a * x + (b * s + c * (s @ s)) @ x
    return (x.transpose(1, 2) if tall else x).to(torch.bfloat16).contiguous()


def _limit(p):
    return min(65535, max(1, round(65536 * p)))


def _plain_factor(shape, p, rng):
    """What a probability is multiplied by: 0 or the inverse of the kept share, 32 bits."""

    n = math.prod(shape)
    low = 0xFFFFFFFF
    index = torch.arange((n + 7) // 8, device="cuda")
    k0, k1 = rng[0] & low, (rng[0] >> 32) & low
    c0, c1, c2, c3 = index & low, index >> 32, torch.full_like(index, SITE), \
        (rng[1] & low).expand(index.shape)
    for _ in range(7):
        # (64-bit products wrap; the words cut out of them are the unsigned ones.)
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack([c0, c1, c2, c3], dim=1)
    halves = torch.stack([words & 0xFFFF, words >> 16], dim=2).reshape(-1)[:n].reshape(shape)
    return (halves >= _limit(p)).float() * (65536.0 / (65536 - _limit(p)))


def _plain_attention(state, case):
    b, length, h, d = (case[k] for k in ("batch", "length", "heads", "dim"))
    dtype, scale = state["query"].dtype, state["scale"]
    q, k, v = (state[n].detach().float().view(b, length, h, d).transpose(1, 2).contiguous()
               for n in ("query", "key", "value"))
    pk, pq = (None if state[n] is None else
              state[n].detach().float().view(-1, h, d).transpose(0, 1).contiguous()
              for n in ("pos_key", "pos_query"))
    position = torch.arange(length, device="cuda")
    slot = state["delta_to_slot"].long()[position[:, None] - position[None] + length - 1]
    by_query = slot.expand(b, h, length, length)          # [.., i, j]: i's slot towards j
    by_key = slot.t().expand(b, h, length, length)        # [.., j, i]

    s = q @ k.transpose(2, 3)
    if pk is not None:
        s = s + (q @ pk.transpose(1, 2)).gather(3, by_query)
    if pq is not None:
        s = s + (k @ pq.transpose(1, 2)).gather(3, by_key).transpose(2, 3)
    mask = state["mask"]
    pair = (mask[:, None, :, None] & mask[:, None, None, :])
    s = (s * scale).masked_fill(~pair, torch.finfo(torch.float32).min)
    s = (s - s.amax(3, keepdim=True)).exp()
    prob = s / s.sum(3, keepdim=True)
    factor = _plain_factor((b, h, length, length), case["p"], state["rng"]) if case["p"] else 1.0
    dropped = prob * factor
    y = dropped @ v
    whole = (y.transpose(1, 2).to(dtype).contiguous(),)
    if not case["backward"]:
        return whole

    dy = state["dy"].float().transpose(1, 2).contiguous()
    dv = dropped.transpose(2, 3) @ dy
    dprob = (dy @ v.transpose(2, 3)) * factor
    ds = prob * (dprob - (prob * dprob).sum(3, keepdim=True))
    ds = (ds * scale).masked_fill(~pair, 0.0)
    dq, dk = ds @ k, ds.transpose(2, 3) @ q
    tables = []
    if pk is not None:
        by_slot = torch.zeros(b, h, length, pk.shape[1], device="cuda").scatter_add_(3, by_query, ds)
        dq = dq + by_slot @ pk
        tables.append((by_slot.transpose(2, 3) @ q).sum(0))
    if pq is not None:
        by_slot = torch.zeros(b, h, length, pq.shape[1], device="cuda").scatter_add_(
            3, by_key, ds.transpose(2, 3))
        dk = dk + by_slot @ pq
        tables.append((by_slot.transpose(2, 3) @ k).sum(0))
    rows = [t.transpose(1, 2).reshape(b, length, h * d).to(dtype) for t in (dq, dk, dv)]
    return (*whole, *rows, *(t.transpose(0, 1).reshape(-1, h * d).to(dtype) for t in tables))


_PLAIN = {"attention": _plain_attention, "orthogonalize": _plain_orthogonalize}


# ---- the definitions in 64 bits -----------------------------------------------

def _exact_factor(shape, p, rng):
    """The generator on the host, with numpy's unsigned words."""

    seed, step = (int(v) for v in rng.cpu())
    n = math.prod(shape)
    blocks = -(-n // 8)
    mask, shift = np.uint64(0xFFFFFFFF), np.uint64(32)
    out = torch.empty(blocks * 8, dtype=torch.bool, device="cuda")
    for first in range(0, blocks, 1 << 20):
        index = np.arange(first, min(blocks, first + (1 << 20)), dtype=np.uint64)
        c = [index & mask, index >> shift, np.full(index.size, SITE, np.uint64),
             np.full(index.size, step & 0xFFFFFFFF, np.uint64)]
        key = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
        for _ in range(7):
            x, z = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
            c = [(z >> shift) ^ c[1] ^ np.uint64(key[0]), z & mask,
                 (x >> shift) ^ c[3] ^ np.uint64(key[1]), x & mask]
            key = [(key[0] + 0x9E3779B9) & 0xFFFFFFFF, (key[1] + 0xBB67AE85) & 0xFFFFFFFF]
        fields = np.empty((index.size, 8), np.uint16)
        for word in range(4):
            fields[:, 2 * word] = c[word] & np.uint64(0xFFFF)
            fields[:, 2 * word + 1] = c[word] >> np.uint64(16)
        kept = torch.from_numpy(fields.reshape(-1) >= _limit(p))
        out[first * 8:first * 8 + kept.numel()] = kept.cuda()
    return out[:n].reshape(shape)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "orthogonalize":
        return _exact_orthogonalize(state, case)
    return _exact_attention(state, case)


def _exact_orthogonalize(state, case):
    # By the Gram matrix of the short side, whose polynomial multiplies the update once.
    g = state["update"].double()
    if case["rows"] > case["columns"]:
        g = g.mT.contiguous()
    g = g / (torch.linalg.matrix_norm(g, keepdim=True) + EPS)
    m = g.shape[1]
    one = torch.eye(m, dtype=torch.float64, device="cuda").expand(g.shape[0], m, m)
    a, b, c = COEFFICIENTS
    gram, total = g @ g.mT.contiguous(), one
    for _ in range(case["steps"]):
        step = a * one + b * gram + c * (gram @ gram)
        gram = step @ gram @ step
        total = step @ total
    x = total @ g
    return x.mT.contiguous() if case["rows"] > case["columns"] else x


def _exact_attention(state, case):
    """Sequence by sequence, the position rows laid out by delta, gradients by autograd."""

    b, length, h, d = (case[k] for k in ("batch", "length", "heads", "dim"))
    leaves = {n: state[n].detach().double().requires_grad_(case["backward"])
              for n in ("query", "key", "value", "pos_key", "pos_query") if state[n] is not None}
    at = torch.arange(length, device="cuda")
    at = at[:, None] - at[None] + length - 1
    places = state["delta_to_slot"].long()
    by_delta = {n: leaves[n].view(-1, h, d)[places].permute(1, 2, 0)
                for n in ("pos_key", "pos_query") if n in leaves}
    kept = None
    if case["p"]:
        kept = _exact_factor((b, h, length, length), case["p"], state["rng"])
        share = (65536 - _limit(case["p"])) / 65536
    outs = []
    for n in range(b):
        q, k, v = (leaves[name][n].view(length, h, d).transpose(0, 1)
                   for name in ("query", "key", "value"))
        s = torch.matmul(q, k.transpose(1, 2))
        if "pos_key" in by_delta:
            s = s + torch.matmul(q, by_delta["pos_key"]).gather(2, at.expand(h, -1, -1))
        if "pos_query" in by_delta:
            s = s + torch.matmul(k, by_delta["pos_query"]).gather(
                2, at.t().expand(h, -1, -1)).transpose(1, 2)
        here = state["mask"][n]
        s = torch.where(here[:, None] & here[None], s * state["scale"], -1e300)
        prob = torch.softmax(s, 2)
        if kept is not None:
            prob = torch.where(kept[n], prob / share, 0.0)
        outs.append(torch.matmul(prob, v).transpose(0, 1))
    y = torch.stack(outs)
    if not case["backward"]:
        return (y,)
    return (y.detach(), *torch.autograd.grad(y, list(leaves.values()), state["dy"].double()))
