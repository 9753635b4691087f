"""Float64 statement of the training operators, with bounds on what fp32 kernels may be off.

Tests only.  The generator is written with numpy's 64-bit words; the operators and their
gradients are the formulas in float64 on whatever device the inputs are on.

Bounds.  u = 2^-24 is fp32's half step.  A sum of terms t_i taken in chains of at most k
additions is off by at most k u sum|t_i|.  A row of layer_norm is summed in chains of at most 40
elements a lane (8191 of 16 bits: 256 lanes of 5 chunks), 6 steps across a wavefront and 3 across
four of them, so k = 49; with the division by the width and the roundings of s itself (two
products and a sum) the mean is off by 53 u.  Results are rounded once more to their dtype:
``finfo(dtype).eps / 2`` of the value, or half the smallest subnormal.
"""

from __future__ import annotations

import numpy as np
import torch

U = 2.0 ** -24
M0, M1, W0, W1 = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85


def philox(counter, key, rounds=7):
    """Four uint64 arrays holding 32-bit words; ``counter`` four arrays, ``key`` two ints."""

    low, shift = np.uint64(0xFFFFFFFF), np.uint64(32)
    c = [np.asarray(v, dtype=np.uint64) for v in counter]
    k0, k1 = key
    for _ in range(rounds):
        a, b = c[0] * np.uint64(M0), c[2] * np.uint64(M1)
        c = [(b >> shift) ^ c[1] ^ np.uint64(k0), b & low,
             (a >> shift) ^ c[3] ^ np.uint64(k1), a & low]
        k0, k1 = (k0 + W0) & 0xFFFFFFFF, (k1 + W1) & 0xFFFFFFFF
    return c


def limit_of(p):
    return int(p) * 65536 if p in (0, 1) else min(65535, max(1, round(p * 65536)))


def kept(shape, p, rng, site, first=0):
    """Bool tensor: which elements from flat index ``first`` (a multiple of 8) are kept."""

    n = int(np.prod(shape))
    blocks = np.arange(first // 8, first // 8 + -(-n // 8), dtype=np.uint64)
    seed, step = (int(v) for v in rng.cpu())
    low = np.uint64(0xFFFFFFFF)
    words = philox([blocks & low, blocks >> np.uint64(32), np.full(blocks.size, site, np.uint64),
                    np.full(blocks.size, step & 0xFFFFFFFF, np.uint64)],
                   (seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF))
    fields = np.empty((blocks.size, 8), dtype=np.int64)
    for i, word in enumerate(words):
        fields[:, 2 * i] = word & np.uint64(0xFFFF)
        fields[:, 2 * i + 1] = word >> np.uint64(16)
    return torch.from_numpy(fields.reshape(-1)[:n] >= limit_of(p)).reshape(shape).to(rng.device)


def factor(shape, p, rng, site, first=0):
    """What each element is multiplied by, float64."""

    if p == 0:
        return torch.ones(shape, dtype=torch.float64, device=rng.device)
    if p == 1:
        return torch.zeros(shape, dtype=torch.float64, device=rng.device)
    return kept(shape, p, rng, site, first).double() * (65536 / (65536 - limit_of(p)))


def rounding(value, dtype):
    """Half a step of ``dtype`` at ``value``."""

    info = torch.finfo(dtype)
    return value.abs() * (info.eps / 2) + info.tiny * info.eps / 2


def layer_norm(x, weight, bias, eps, residual=None, mult=None, dy=None):
    """Values and bounds: ``{"y": (value, bound), ...}`` in float64, gradients where ``dy`` is
    given.  ``x`` ``[rows, H]`` in its dtype, ``mult`` the dropout's factors."""

    dtype, wtype = x.dtype, weight.dtype
    c = torch.ones_like(x, dtype=torch.float64) if mult is None else mult
    xd, w, b = x.double(), weight.double(), bias.double()
    dropped = torch.where(c == 0, torch.zeros_like(xd), xd * c)
    r = torch.zeros_like(xd) if residual is None else residual.double()
    s = dropped + r
    size = (dropped.abs() + r.abs()).amax(-1, keepdim=True)
    mean = s.mean(-1, keepdim=True)
    var = (s - mean).square().mean(-1, keepdim=True)
    rstd = (var + eps).rsqrt()
    xh = (s - mean) * rstd
    ratio = size * rstd
    # xh: s and the mean are off by 53 u size; the variance by 51 u of itself (49 additions, the
    # square and the division) and by 2 x 53 u size / sigma, half of which reaches rstd, and
    # rsqrt by 2 u; products 2 u: 25.5 + 4 < 32.
    e_xh = U * (53 * ratio * (1 + xh.abs()) + 32 * xh.abs())
    y = xh * w + b
    out = {"y": (y, w.abs() * e_xh + 2 * U * ((xh * w).abs() + b.abs()) + rounding(y, dtype))}
    if dy is None:
        return out
    d = dy.double()
    g = d * w
    m1, m2 = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
    inner = g - m1 - xh * m2
    ds = rstd * inner
    size_g = g.abs() + g.abs().mean(-1, keepdim=True) \
        + xh.abs() * (g * xh).abs().mean(-1, keepdim=True)
    e_rstd = U * (32 + 53 * ratio)
    e_ds = rstd * (e_rstd * size_g + 52 * U * size_g + m2.abs() * e_xh
                   + xh.abs() * (g.abs() * e_xh).mean(-1, keepdim=True))
    out["dresidual"] = (ds, e_ds + rounding(ds, dtype))
    dx = torch.where(c == 0, torch.zeros_like(ds), ds * c)
    out["dx"] = (dx, e_ds * c + 2 * U * dx.abs() + rounding(dx, dtype))
    # Rows: a lane adds rows / 512 of them at most (one at least), then 16 groups, then 512
    # partial rows in 64 slices of 8; two roundings of the products.
    chain = (x.shape[0] / 512 + 1 + 16 + 8 + 64 + 2) * U
    dw = (d * xh).sum(0)
    out["dweight"] = (dw, (d.abs() * e_xh).sum(0) + chain * (d * xh).abs().sum(0)
                      + rounding(dw, wtype))
    db = d.sum(0)
    out["dbias"] = (db, chain * d.abs().sum(0) + rounding(db, wtype))
    return out


def embedding_gradient(ids, dy, rows, scale, padding=None):
    """``(value, bound)`` of the table's gradient; ids outside the table are left out."""

    ids, d = ids.flatten().long(), dy.double().reshape(-1, dy.shape[-1])
    used = (ids >= 0) & (ids < rows)
    if padding is not None:
        used &= ids != padding
    ids, d = ids[used], d[used]
    value = torch.zeros(rows, d.shape[-1], dtype=torch.float64, device=d.device)
    size = torch.zeros_like(value)
    value.index_add_(0, ids, d)
    size.index_add_(0, ids, d.abs())
    value, size = value * scale, size * abs(scale)
    # Up to 256 tokens one after the other; else the 32 rows of a tile, an eighth of the tiles of
    # one id, the eight parts.  Then the scale's product.
    n = ids.numel()
    chain = (n if n <= 256 else 32 + n / 256 + 1 + 8) + 2
    return value, chain * U * size + rounding(value, dy.dtype)


def check(got, want, name):
    """``got`` lies within the bound of ``want = (value, bound)``, and is finite where the value
    is: round to nearest gives infinity from half a step past the dtype's largest number, which
    is ``max = 2^E (2 - eps)`` with a step of ``2^E eps``."""

    value, bound = want
    assert got.shape == value.shape, (name, got.shape, value.shape)
    info = torch.finfo(got.dtype)
    border = info.max * (1 + info.eps / 2 / (2 - info.eps))
    beyond = value.abs() - bound >= border
    assert bool(torch.isinf(got[beyond]).all()), name
    assert torch.equal(torch.signbit(got[beyond]), torch.signbit(value[beyond])), name
    near = (value.abs() + bound >= border) & torch.isinf(got)  # either side of the border
    got, value, bound = (t[~(beyond | near)] for t in (got, value, bound))
    assert bool(torch.isfinite(got).all()), name
    over = (got.double() - value).abs() - bound
    assert not bool((over > 0).any()), (
        f"{name}: off by {(got.double() - value).abs().max().item():.3e}, "
        f"{over.max().item():.3e} past its bound")
