"""Float64 statement of ``training.attention`` and its gradients, with bounds on what the kernels
may be off.  Tests only.

Bounds.  U = 2^-24 is fp32's half step, u the dtype's (``finfo.eps / 2``); a sum of n terms in fp32 is
off by at most n U sum|t|.

* A score is three sums of d products and two additions, scaled (twice: by ``scale`` and by log2 e):
  off by (d + 6) U (|q|.|k| + |q|.|pk| + |k|.|pq|) |scale|.  The row's statistic takes the
  largest of its scores' errors, a sum of at most L exponentials, and an exponential, a logarithm
  and a product of 2 U each (with the rounding of the base-2 exponent, U of at most 1.45 |s| and of the statistic):
  a probability is off by r = 2 max e_s + (L + 32) U + 4 U (max |s| + log L + 1) of itself.
  Beside 16-bit inputs the two relative terms are rounded to fp16, scaled: 2^-12 of each in base
  2, which is 2^-12 of it in base e too, or 2^-25.
* Probabilities with their dropout factor (R) and score gradients (G) are rounded to the dtype as
  operands: u of each, or half the dtype's smallest subnormal (unnormalised in the forward pass, where
  the largest is 1, so of 1 / sum <= 1).
* D_i = dO_i.O_i with O as rounded: |dO|.e_O and a sum of d products.
* Products over L places: (2 L + 16) U; of the tables over the batch too, and the slots' sums.
"""

from __future__ import annotations

import torch

from training_reference import U, rounding


def floor_of(dtype):
    """Half the smallest subnormal."""

    info = torch.finfo(dtype)
    return info.tiny * info.eps / 2


def by_delta(x):
    """``[.., L, L]`` -> ``[.., L, 2L - 1]``: element (i, j) at place i - j + L - 1 of row i."""

    length = x.shape[-1]
    at = torch.arange(length, device=x.device)
    at = (at[:, None] - at[None] + length - 1).expand(x.shape)
    return torch.zeros(*x.shape[:-1], 2 * length - 1, dtype=x.dtype, device=x.device).scatter_(
        -1, at, x)


def from_delta(x):
    """The inverse: row i's places i - j + L - 1."""

    length = x.shape[-2]
    at = torch.arange(length, device=x.device)
    at = (at[:, None] - at[None] + length - 1).expand(*x.shape[:-1], length)
    return x.gather(-1, at)


def expand(table, lut):
    """``[H, S, d]`` -> ``[H, 2L - 1, d]``; rows of 0 for places outside."""

    inside = (lut >= 0) & (lut < table.shape[1])
    rows = table[:, lut.long().clamp(0, table.shape[1] - 1)]
    return torch.where(inside[None, :, None], rows, torch.zeros_like(rows))


def collect(rows, lut, slots):
    """``[H, 2L - 1, d]`` -> ``[H, S, d]``: the sums of each slot."""

    inside = (lut >= 0) & (lut < slots)
    out = torch.zeros(rows.shape[0], slots, rows.shape[2], dtype=rows.dtype, device=rows.device)
    return out.index_add_(1, lut[inside].long(), rows[:, inside])


def attention(q, k, v, pk, pq, lut, scale, mask=None, mult=None, dout=None):
    """``{"out": (value, bound), ..}``; q, k, v ``[B, L, H, d]``, tables ``[H, S, d]`` or None,
    ``mult`` the dropout's factors ``[B, H, L, L]``."""

    dtype = q.dtype
    u, floor = torch.finfo(dtype).eps / 2, floor_of(dtype)
    if dtype == torch.float32:
        u = 0.0  # (nothing is rounded that is not fp32 already; rounding() counts the result)
    b, length, h, d = q.shape
    if mask is None:
        mask = torch.ones(b, length, dtype=torch.bool, device=q.device)
    mask = mask.bool()
    pair = (mask[:, None, :, None] & mask[:, None, None, :]).expand(b, h, length, length)
    heads = [t.detach().double().transpose(1, 2) for t in (q, k, v)]
    # Padded queries and keys take no part in scores.
    Q, K = (torch.where(mask[:, None, :, None], t, torch.zeros_like(t)) for t in heads[:2])
    V = heads[2]
    PK, PQ = (None if t is None else expand(t.detach().double(), lut) for t in (pk, pq))

    def scores(Q, K, PK, PQ):
        s = Q @ K.transpose(2, 3)
        if PK is not None:
            s = s + from_delta(Q @ PK.transpose(1, 2))
        if PQ is not None:
            # (K_j.PQ at i - j: place j - i counted from the other end)
            s = s + from_delta((K @ PQ.transpose(1, 2)).flip(-1)).transpose(2, 3)
        return s * scale

    def absolute(t):
        return None if t is None else t.abs()

    s = scores(Q, K, PK, PQ)
    e_s = (d + 6) * U * scores(*map(absolute, (Q, K, PK, PQ))).abs()
    if dtype in (torch.float16, torch.bfloat16):
        none = torch.zeros_like(K)
        if PK is not None:
            e_s = e_s + 2.0 ** -12 * scores(Q, none, PK, None).abs() + 2.0 ** -25
        if PQ is not None:
            e_s = e_s + 2.0 ** -12 * scores(torch.zeros_like(Q), K, None, PQ).abs() + 2.0 ** -25
    s = torch.where(pair, s, torch.full_like(s, -1e300))
    s = torch.where(mask[:, None, :, None], s, torch.zeros_like(s))  # padded queries: all equal
    prob = torch.softmax(s, -1)
    if mult is None:
        mult = torch.ones_like(prob)
    row_s = torch.where(pair, s.abs(), torch.zeros_like(s)).amax(-1, keepdim=True)
    row_e = torch.where(pair, e_s, torch.zeros_like(s)).amax(-1, keepdim=True)
    log_length = torch.tensor(float(length)).log().item()
    r = 2 * row_e + (length + 32) * U + 4 * U * (row_s + log_length + 1)
    kept = prob * mult
    most = mult.amax()
    sums = (2 * length + 16) * U
    # A padded query takes every key; of a kept one's excluded keys nothing arrives.
    taken = (pair | ~mask[:, None, :, None]).double()
    # (What is not finite at a padded key counts as 0.)
    finite_v = torch.where(torch.isfinite(V) | mask[:, None, :, None], V, torch.zeros_like(V))
    out = kept @ finite_v
    e_out = (kept * (r + u + sums)) @ finite_v.abs() + floor * most * (taken @ finite_v.abs())
    result = {"out": (out.transpose(1, 2),
                      (e_out + rounding(out, dtype)).transpose(1, 2))}
    if dout is None:
        return result

    V = finite_v
    dO = dout.detach().double().transpose(1, 2)
    dP = dO @ V.transpose(2, 3)
    e_dP = (d + 4) * U * (dO.abs() @ V.abs().transpose(2, 3))
    D = (prob * mult * dP).sum(-1, keepdim=True)
    e_D = (dO.abs() * (e_out + rounding(out, dtype))).sum(-1, keepdim=True) \
        + (d + 4) * U * (dO.abs() * out.abs()).sum(-1, keepdim=True)
    inner = torch.where(mult > 0, dP * mult, torch.zeros_like(dP)) - D
    G = torch.where(pair, prob * inner, torch.zeros_like(prob))
    e_G = torch.where(pair, prob * (r * inner.abs() + mult * e_dP + e_D
                                    + 4 * U * (mult * dP.abs() + D.abs())),
                      torch.zeros_like(prob)) * (1 + 1e-3)
    if length == 1:
        G, e_G = torch.zeros_like(G), torch.zeros_like(e_G)
    # As an operand: rounded to the dtype, summed.
    off = e_G + (u + sums) * G.abs() + floor * pair
    off_r = kept * (r + u + sums) + floor * most * taken
    scaled = abs(scale)

    def entry(value, bound, heads_last=True):
        bound = bound + 2 * U * value.abs() + rounding(value, dtype)
        return (value.transpose(1, 2), bound.transpose(1, 2)) if heads_last else (value, bound)

    dV = kept.transpose(2, 3) @ dO
    result["dv"] = entry(dV, off_r.transpose(2, 3) @ dO.abs())
    dQ, dK = G @ K, G.transpose(2, 3) @ Q
    e_dQ, e_dK = off @ K.abs(), off.transpose(2, 3) @ Q.abs()
    chain = (b * length + 2 * length + 64) * U
    if PK is not None:
        dQ = dQ + by_delta(G) @ PK
        e_dQ = e_dQ + by_delta(off) @ PK.abs()
        rows = (by_delta(G).transpose(2, 3) @ Q).sum(0)
        e_rows = (by_delta(off + chain * G.abs()).transpose(2, 3) @ Q.abs()).sum(0)
        result["dpos_key"] = entry(scale * collect(rows, lut, pk.shape[1]),
                                   scaled * collect(e_rows, lut, pk.shape[1]), False)
    if PQ is not None:
        def by_key(x):  # row j, place i - j + L - 1
            return by_delta(x.transpose(2, 3)).flip(-1)

        dK = dK + by_key(G) @ PQ
        e_dK = e_dK + by_key(off) @ PQ.abs()
        rows = (by_key(G).transpose(2, 3) @ K).sum(0)
        e_rows = (by_key(off + chain * G.abs()).transpose(2, 3) @ K.abs()).sum(0)
        result["dpos_query"] = entry(scale * collect(rows, lut, pq.shape[1]),
                                     scaled * collect(e_rows, lut, pq.shape[1]), False)
    result["dq"] = entry(scale * dQ, scaled * e_dQ)
    result["dk"] = entry(scale * dK, scaled * e_dK)
    return result
