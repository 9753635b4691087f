"""The training operators on the GPU against their float64 statement.

Every comparison is element by element against ``training_reference``'s bounds, which are
derived there; masks are compared as they are.
"""

from __future__ import annotations

import copy
import functools

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import training_reference as ref  # noqa: E402 (tests/ is on the path)

pytestmark = pytest.mark.gpu

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SEED, STEP, SITE = 0x1234567890ABCDEF, 7, 11


@pytest.fixture(params=list(DTYPES))
def dtype(request):
    return DTYPES[request.param]


def _rng(seed=SEED, step=STEP):
    return torch.tensor([seed, step], device="cuda")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, shape, dtype, scale=1.0, at=0.0):
    return (torch.randn(shape, device="cuda", generator=gen) * scale + at).to(dtype)


# ---- dropout -----------------------------------------------------------------------


@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (3, 5), (97, 769), (2, 12, 64, 64)],
                         ids=str)
@pytest.mark.parametrize("p", [0.1, 0.5, 1.0, 1e-9, 1 - 1e-9])
def test_dropout_and_its_gradient(dtype, shape, p):
    from disentangled_flash.training import dropout

    gen = _gen(len(shape))
    x = _normal(gen, shape, dtype).requires_grad_()
    dy = _normal(gen, shape, dtype)
    rng = _rng()
    y = dropout(x, p, rng, SITE)
    (dx,) = torch.autograd.grad(y, x, dy)
    mult = ref.factor(shape, p, rng, SITE)
    for got, given in ((y, x.detach()), (dx, dy)):
        want = given.double() * mult
        assert got.dtype == dtype
        # The factor and the product in fp32, then the dtype.
        ref.check(got.detach(), (want, 2 * ref.U * want.abs() + ref.rounding(want, dtype)), "drop")
        assert torch.equal(got == 0, (mult == 0) | (given == 0))


def test_dropout_selects_and_does_not_multiply(dtype):
    from disentangled_flash.training import dropout

    x = torch.full((64, 64), float("inf"), device="cuda", dtype=dtype)
    x[32:] = float("nan")
    y = dropout(x, 0.5, _rng(), SITE)
    keep = ref.kept((64, 64), 0.5, _rng(), SITE)
    assert bool((y[~keep] == 0).all())
    assert bool(torch.isinf(y[:32][keep[:32]]).all()) and bool(torch.isnan(y[32:][keep[32:]]).all())
    assert bool((dropout(x, 1.0, _rng(), SITE) == 0).all())


def test_dropout_layouts(dtype):
    """Addresses off the 16-byte boundaries, transposed and expanded inputs and gradients."""

    from disentangled_flash.training import dropout

    store = _normal(_gen(1), (4001,), dtype)
    table = _normal(_gen(2), (40, 100), dtype)
    for x in (store[1:], store[3:-2], store[4:2004], table.t(), table[:, 1:], table[::3],
              table[:1].expand(40, 100)):
        y = dropout(x, 0.3, _rng(), SITE)
        want = x.double() * ref.factor(tuple(x.shape), 0.3, _rng(), SITE)
        ref.check(y, (want, 2 * ref.U * want.abs() + ref.rounding(want, dtype)), str(x.stride()))
    x = table.clone().requires_grad_()
    dropout(x, 0.3, _rng(), SITE).sum().backward()  # an expanded gradient
    mult = ref.factor((40, 100), 0.3, _rng(), SITE)
    ref.check(x.grad, (mult, 2 * ref.U * mult + ref.rounding(mult, dtype)), "expanded")


def test_dropout_depends_on_every_word():
    """Seed (both words), step and site each change the mask; the step's low word counts."""

    from disentangled_flash.training import dropout

    x = torch.ones(4096, device="cuda")
    base = dropout(x, 0.5, _rng(), SITE)
    assert torch.equal(base, dropout(x, 0.5, _rng(step=STEP + (1 << 32)), SITE))
    for rng, site in ((_rng(SEED + 1), SITE), (_rng(SEED ^ (1 << 40)), SITE),
                      (_rng(step=STEP + 1), SITE), (_rng(), SITE + 1), (_rng(-SEED), SITE),
                      (_rng(), (1 << 32) - 1)):
        y = dropout(x, 0.5, rng, site)
        assert not torch.equal(y, base)
        assert torch.equal(y != 0, ref.kept((4096,), 0.5, rng, site))


def test_dropout_past_32_bits():
    """More than 2^32 elements: places and counters of the last ones."""

    from disentangled_flash.training import dropout

    n = (1 << 32) + 4101
    y = dropout(torch.ones(n, device="cuda", dtype=torch.float16), 0.25, _rng(), SITE)
    first = n - 4101 - 64
    tail = ref.kept((n - first,), 0.25, _rng(), SITE, first)
    assert torch.equal(y[first:] != 0, tail)
    del y
    torch.cuda.empty_cache()


# ---- layer norm ----------------------------------------------------------------------


def _norm_case(seed, rows, hidden, dtype, weights, residual):
    gen = _gen(seed)
    x = _normal(gen, (rows, hidden), dtype, 0.7)
    r = _normal(gen, (rows, hidden), dtype, 1.3, 0.25) if residual else None
    w = _normal(gen, (hidden,), weights, 0.1, 1.0)
    b = _normal(gen, (hidden,), weights, 0.1)
    return x, r, w, b, _normal(gen, (rows, hidden), dtype)


def _check_norm(x, r, w, b, dy, eps, p, site=SITE):
    from disentangled_flash.training import layer_norm

    rng = _rng()
    leaves = [t.clone().requires_grad_() for t in (x, w, b) + (() if r is None else (r,))]
    y = layer_norm(leaves[0], leaves[1], leaves[2], eps, residual=leaves[3] if r is not None
                   else None, p=p, rng=rng, site=site)
    grads = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        alone = layer_norm(x, w, b, eps, residual=r, p=p, rng=rng, site=site)
    assert torch.equal(y, alone)  # the form that keeps no statistics
    want = ref.layer_norm(x, w, b, eps, r, ref.factor(tuple(x.shape), p, rng, site), dy)
    ref.check(y.detach(), want["y"], "y")
    for name, got, leaf in zip(("dx", "dweight", "dbias", "dresidual"), grads, leaves):
        assert got.dtype == leaf.dtype
        ref.check(got, want[name], name)


# A width of every layout and its neighbours, odd ones, and whole chunks of fp32 only.
WIDTHS = [1, 2, 3, 7, 8, 60, 64, 100, 128, 132, 250, 256, 384, 500, 512, 768, 769, 1001, 1024, 1030,
          1536, 1540, 2048, 2050, 4096, 4100, 8191, 8192]


@pytest.mark.parametrize("hidden", WIDTHS)
@pytest.mark.parametrize("p", [0.0, 0.1])
def test_layer_norm_widths(dtype, hidden, p):
    _check_norm(*_norm_case(hidden, 13, hidden, dtype, dtype, True), 1e-7 if hidden > 3 else 1e-3,
                p)


@pytest.mark.parametrize("rows", [1, 2, 9, 600, 4113])
@pytest.mark.parametrize("hidden", [64, 768, 1001])
@pytest.mark.parametrize("residual", [True, False])
def test_layer_norm_rows(dtype, rows, hidden, residual):
    p = 0.3 if residual else 0.0
    _check_norm(*_norm_case(rows, rows, hidden, dtype, dtype, residual), 1e-5, p)


@pytest.mark.parametrize("rows,hidden", [(1100, 2051), (9000, 33), (1030, 4103)])
def test_layer_norm_many_odd_rows(dtype, rows, hidden):
    """More rows than the launch has groups of lanes: each meets several of one shift."""

    _check_norm(*_norm_case(rows, rows, hidden, dtype, dtype, True), 1e-5, 0.1)


@pytest.mark.parametrize("hidden", [64, 200, 769, 1024])
@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("p", [0.0, 0.6, 1.0])
def test_layer_norm_fp32_weights(hidden, kind, p):
    _check_norm(*_norm_case(hidden, 37, hidden, kind, torch.float32, True), 1e-7, p)


def test_layer_norm_dropout_without_residual(dtype):
    _check_norm(*_norm_case(3, 21, 768, dtype, dtype, False), 1e-5, 0.2)


def test_layer_norm_drops_what_dropout_drops(dtype):
    """layer_norm(x, residual, p) is layer_norm(dropout(x) + residual): in fp32 to the last
    roundings, and the same elements are dropped at an odd width too."""

    from disentangled_flash.training import dropout, layer_norm

    for hidden in (768, 333):
        x, r, w, b, _ = _norm_case(4, 29, hidden, torch.float32, torch.float32, True)
        fused = layer_norm(x, w, b, 1e-6, r, 0.4, _rng(), SITE)
        apart = layer_norm(dropout(x, 0.4, _rng(), SITE) + r, w, b, 1e-6)
        torch.testing.assert_close(fused, apart, atol=1e-5, rtol=1e-5)


def test_layer_norm_layouts(dtype):
    from disentangled_flash.training import layer_norm

    eps = 1e-5
    x, r, w, b, dy = _norm_case(5, 96, 256, dtype, dtype, True)
    want = ref.layer_norm(x, w, b, eps, r)["y"]
    wide = torch.empty(96, 2, 256, device="cuda", dtype=dtype)
    wide[:, 1] = x
    odd = torch.empty(96 * 256 + 8, device="cuda", dtype=dtype)
    shifted = odd[1:1 + 96 * 256].view(96, 256)
    shifted.copy_(r)
    weights = torch.empty(257, device="cuda", dtype=dtype)[1:].copy_(w)
    for xs, rs, ws in ((wide[:, 1], r, w), (x.t().contiguous().t(), shifted, w), (x, r, weights),
                       (shifted.copy_(x).clone(), shifted.copy_(r), weights)):
        ref.check(layer_norm(xs, ws, b, eps, rs), want, f"{xs.stride()} {xs.data_ptr() % 16}")
    y = layer_norm(x.view(4, 3, 8, 256), w, b, eps, r.view(4, 3, 8, 256))
    ref.check(y.view(96, 256), want, "4-D")
    ref.check(layer_norm(x[0], w, b, eps, r[0])[None], tuple(t[:1] for t in want), "1-D")
    leaf = x.clone().requires_grad_()
    layer_norm(leaf, w, b, eps).sum().backward()
    ones = torch.ones_like(x)
    ref.check(leaf.grad, ref.layer_norm(x, w, b, eps, dy=ones)["dx"], "expanded gradient")
    leaf = x.clone().requires_grad_()
    layer_norm(leaf.t().contiguous().t(), w, b, eps, r).backward(dy.t().contiguous().t())
    ref.check(leaf.grad, ref.layer_norm(x, w, b, eps, r, dy=dy)["dx"], "transposed")


@pytest.mark.parametrize("wanted", ["x", "w", "b", "r", "xr", "wb"])
@pytest.mark.parametrize("p", [0.0, 0.2])
def test_layer_norm_gradients_one_by_one(wanted, p):
    from disentangled_flash.training import layer_norm

    x, r, w, b, dy = _norm_case(6, 50, 320, torch.bfloat16, torch.float32, True)
    leaves = {"x": x, "w": w, "b": b, "r": r}
    for name in wanted:
        leaves[name].requires_grad_()
    y = layer_norm(x, w, b, 1e-6, r, p, _rng(), SITE)
    grads = torch.autograd.grad(y, [leaves[name] for name in wanted], dy)
    for t in leaves.values():
        t.requires_grad_(False)
    want = ref.layer_norm(x, w, b, 1e-6, r, ref.factor((50, 320), p, _rng(), SITE), dy)
    names = {"x": "dx", "w": "dweight", "b": "dbias", "r": "dresidual"}
    for name, grad in zip(wanted, grads):
        ref.check(grad, want[names[name]], name)


def test_layer_norm_gradient_is_a_difference():
    """fp32 gradients against central differences of the float64 forward."""

    from disentangled_flash.training import layer_norm

    x, r, w, b, dy = _norm_case(7, 6, 96, torch.float32, torch.float32, True)
    leaves = {"x": x, "w": w, "b": b, "r": r}
    for t in leaves.values():
        t.requires_grad_()
    grads = torch.autograd.grad(layer_norm(x, w, b, 1e-5, r, 0.25, _rng(), SITE),
                                list(leaves.values()), dy)
    mult = ref.factor((6, 96), 0.25, _rng(), SITE)
    for (name, leaf), grad in zip(leaves.items(), grads):
        direction = torch.randn(leaf.shape, device="cuda", dtype=torch.float64, generator=_gen(8))
        step, values = 1e-5, []
        for sign in (1, -1):
            at = {n: t.detach().double() + (sign * step * direction if n == name else 0)
                  for n, t in leaves.items()}
            values.append((ref.layer_norm(at["x"], at["w"], at["b"], 1e-5, at["r"], mult)["y"][0]
                           * dy.double()).sum())
        difference = (values[0] - values[1]) / (2 * step)
        # fp32: at most 100 half steps of each of up to 576 terms of size about 3.
        assert abs((grad.double() * direction).sum() - difference) < 576 * 3 * 100 * ref.U, name


def test_layer_norm_rows_stay_apart(dtype):
    """A row of equal elements (its variance 0), one far from 0, one of NaN and one with an
    infinity: the others' outputs and gradients are what they are without them."""

    from disentangled_flash.training import layer_norm

    x, r, w, b, dy = _norm_case(9, 40, 768, dtype, dtype, True)
    clean_y = layer_norm(x, w, b, 1e-7, r)
    leaf = x.clone().requires_grad_()
    (clean_dx,) = torch.autograd.grad(layer_norm(leaf, w, b, 1e-7, r), leaf, dy)
    x2, r2 = x.clone(), r.clone()
    x2[3], r2[3] = 2.0, 1.0
    x2[11] = float("nan")
    x2[17, 5] = float("inf")
    leaf = x2.requires_grad_()
    y = layer_norm(leaf, w, b, 1e-7, r2)
    (dx,) = torch.autograd.grad(y, leaf, dy)
    others = [i for i in range(40) if i not in (3, 11, 17)]
    assert torch.equal(y[others], clean_y[others]) and torch.equal(dx[others], clean_dx[others])
    assert torch.equal(y[3], b) and bool(torch.isfinite(dx[3]).all())
    assert bool(torch.isnan(y[11]).all()) and bool(torch.isnan(y[17]).all())
    far = (x.float() + 4096).to(dtype)
    ref.check(layer_norm(far, w, b, 1e-7), ref.layer_norm(far, w, b, 1e-7)["y"], "far from 0")


def test_layer_norm_of_nothing(dtype):
    from disentangled_flash.training import dropout, embedding, layer_norm

    x = torch.empty(0, 5, 64, device="cuda", dtype=dtype, requires_grad=True)
    w = torch.ones(64, device="cuda", dtype=dtype, requires_grad=True)
    b = torch.ones(64, device="cuda", dtype=dtype, requires_grad=True)
    y = layer_norm(dropout(x, 0.1, _rng()), w, b, 1e-5, x, 0.1, _rng())
    y.sum().backward()
    assert y.shape == x.shape and x.grad.shape == x.shape
    assert torch.equal(w.grad, torch.zeros_like(w)) and torch.equal(b.grad, torch.zeros_like(b))
    table = torch.ones(5, 64, device="cuda", dtype=dtype, requires_grad=True)
    out = embedding(torch.empty(0, 3, device="cuda", dtype=torch.int64), table)
    out.sum().backward()
    assert out.shape == (0, 3, 64) and torch.equal(table.grad, torch.zeros_like(table))


def test_layer_norm_past_32_bits():
    """More than 2^31 elements: the last rows are what they are alone."""

    from disentangled_flash.training import layer_norm

    hidden, rows = 4096, (1 << 19) + 5
    x = torch.zeros(rows, hidden, device="cuda", dtype=torch.float16)
    tail = _normal(_gen(10), (37, hidden), torch.float16)
    x[-37:] = tail
    w, b = (torch.full((hidden,), v, device="cuda", dtype=torch.float16) for v in (1.5, 0.25))
    x.requires_grad_()
    y = layer_norm(x, w, b, 1e-5, None, 0.2, _rng(), SITE)
    mult = ref.factor((37, hidden), 0.2, _rng(), SITE, (rows - 37) * hidden)
    dy = torch.zeros_like(x)
    dy[-37:] = 1.0
    (dx,) = torch.autograd.grad(y, x, dy)
    want = ref.layer_norm(tail, w, b, 1e-5, None, mult, dy[-37:])
    ref.check(y[-37:].detach(), want["y"], "y")
    ref.check(dx[-37:], want["dx"], "dx")
    assert bool((dx[:1000] == 0).all())
    del x, y, dy, dx
    torch.cuda.empty_cache()


# ---- embedding -----------------------------------------------------------------------


def _check_embedding(ids, rows, hidden, dtype, scale=1.0, padding=None, seed=0):
    from disentangled_flash.training import embedding

    gen = _gen(seed)
    table = _normal(gen, (rows, hidden), dtype).requires_grad_()
    y = embedding(ids, table, scale, padding)
    dy = _normal(gen, y.shape, dtype)
    (grad,) = torch.autograd.grad(y, table, dy)
    (again,) = torch.autograd.grad(embedding(ids, table, scale, padding), table, dy)
    assert torch.equal(grad, again)
    want = table.detach()[ids.long()].double() * scale
    ref.check(y.detach(), (want, 2 * ref.U * want.abs() + ref.rounding(want, dtype)), "lookup")
    value, bound = ref.embedding_gradient(ids, dy, rows, scale, padding)
    assert grad.dtype == dtype
    ref.check(grad, (value, bound), "gradient")
    unused = torch.ones(rows, dtype=torch.bool, device="cuda")
    unused[ids.flatten().long()] = False
    if padding is not None:
        unused[padding] = True
    assert bool((grad[unused] == 0).all())


def _ids(kind, n, rows, seed=0):
    gen = _gen(seed + 100)
    if kind == "one":
        return torch.full((n,), rows - 1, device="cuda")
    if kind == "distinct":
        return torch.randperm(max(n, rows), device="cuda", generator=gen)[:n] % rows
    if kind == "frequent":  # a few ids take most of the tokens
        u = torch.rand(n, device="cuda", generator=gen)
        return (u.pow(6) * rows).long().clamp_(max=rows - 1)
    return torch.randint(0, rows, (n,), device="cuda", generator=gen)


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 64, 65, 255, 256, 257, 300, 1000, 1025, 4097])
@pytest.mark.parametrize("kind", ["uniform", "one", "distinct", "frequent"])
def test_embedding_tokens(dtype, n, kind):
    _check_embedding(_ids(kind, n, 513), 513, 96, dtype, seed=n)


@pytest.mark.parametrize("rows", [1, 2, 3, 511, 512, 513, 5000, 128100, 300001])
def test_embedding_tables(rows):
    """Tables of one id up to three digits of the sort."""

    for padding in (None, 0, rows - 1):
        for n in (150, 700, 9000):
            _check_embedding(_ids("frequent", n, rows), rows, 64, torch.bfloat16, 1.5, padding)
    _check_embedding(_ids("frequent", 100, rows), rows, 13, torch.bfloat16)


@pytest.mark.parametrize("hidden", [1, 2, 7, 8, 12, 64, 100, 250, 256, 264, 513, 768, 1024, 1537])
def test_embedding_widths(dtype, hidden):
    _check_embedding(_ids("frequent", 211, 50).view(1, 211), 50, hidden, dtype, 27.7)
    _check_embedding(_ids("frequent", 811, 50), 50, hidden, dtype, 27.7)


@pytest.mark.parametrize("n", [8191, 8192, 8193, 10240, 16385, 40000])
@pytest.mark.parametrize("kind", ["uniform", "one", "frequent"])
@pytest.mark.parametrize("rows", [2, 1500])
def test_embedding_many_tokens(n, kind, rows):
    """Either side of the forms for few, some and many tokens; ranges that are merged."""

    _check_embedding(_ids(kind, n, rows, n), rows, 72, torch.float16)
    _check_embedding(_ids(kind, n, rows, n), rows, 5, torch.float32, 2.0, 0)


@pytest.mark.parametrize("n", [16384, 65536, 65537, 131073, 300000])
@pytest.mark.parametrize("kind", ["uniform", "one", "frequent"])
def test_embedding_runs_that_are_merged(n, kind):
    """More tokens than one run holds: one, two and three launches that join runs."""

    _check_embedding(_ids(kind, n, 70001, n), 70001, 16, torch.bfloat16, 1.0, 3)


@pytest.mark.parametrize("n", [9, 300, 9000])
def test_embedding_most_rows(n):
    """The largest table that is taken, and its last rows."""

    from disentangled_flash.training import embedding

    rows = (1 << 31) - 2
    table = torch.zeros(rows, 1, device="cuda", dtype=torch.float16, requires_grad=True)
    ids = rows - 1 - torch.arange(n, device="cuda") % 7
    dy = torch.ones(n, 1, device="cuda", dtype=torch.float16)
    (grad,) = torch.autograd.grad(embedding(ids, table), table, dy)
    counts = torch.bincount(rows - 1 - ids, minlength=7).flip(0).half()
    assert torch.equal(grad[-7:, 0], counts)
    assert int(torch.count_nonzero(grad[:-7])) == 0
    del table, grad
    torch.cuda.empty_cache()


def test_operators_called_by_name_refuse_what_does_not_fit():
    """Past the Python checks: nothing is launched."""

    from disentangled_flash import training

    x, w = torch.zeros(4, 8, device="cuda"), torch.zeros(8, device="cuda")
    rng, ids = _rng(), torch.zeros(4, device="cuda", dtype=torch.int64)
    training.layer_norm(x, w, w, 1e-5)  # (loads the operators)
    ops = torch.ops.disentangled_flash
    stats = torch.zeros(2, 4, device="cuda")
    sparse, wide = torch.zeros(4, 16, device="cuda")[:, ::2], torch.zeros(4, 9, device="cuda")
    for call in (
        lambda: ops.dropout(sparse, rng, 0.1, 0),
        lambda: ops.dropout(x, rng.cpu(), 0.1, 0),
        lambda: ops.dropout(x, rng.int(), 0.1, 0),
        lambda: ops.dropout(x, rng, 0.1, -1),
        lambda: ops.dropout(x, rng, 0.1, 1 << 32),
        lambda: ops.dropout_layernorm(sparse, None, w, w, None, 1e-5, 0.0, 0),
        lambda: ops.dropout_layernorm(x[:, :0], None, w[:0], w[:0], None, 1e-5, 0.0, 0),
        lambda: ops.dropout_layernorm(x[0, 0], None, w, w, None, 1e-5, 0.0, 0),
        lambda: ops.dropout_layernorm(x, wide, w, w, None, 1e-5, 0.0, 0),
        lambda: ops.dropout_layernorm(x, x.half(), w, w, None, 1e-5, 0.0, 0),
        lambda: ops.dropout_layernorm(x, None, w[:7], w[:7], None, 1e-5, 0.0, 0),
        lambda: ops.dropout_layernorm(x, None, w, w.half(), None, 1e-5, 0.0, 0),
        lambda: ops.dropout_layernorm(x, None, w.cpu(), w.cpu(), None, 1e-5, 0.0, 0),
        lambda: ops.dropout_layernorm_train(x[0, 0], None, w, w, None, 1e-5, 0.0, 0),
        lambda: ops.dropout_layernorm_backward(wide, x, None, w, stats, None, 0.0, 0, *[True] * 3),
        lambda: ops.dropout_layernorm_backward(x, x, None, w, stats[:1], None, 0.0, 0,
                                               *[True] * 3),
        lambda: ops.embedding_lookup(ids.short(), x, 1.0, -1),
        lambda: ops.embedding_lookup(ids.cpu(), x, 1.0, -1),
        lambda: ops.embedding_lookup(ids, sparse, 1.0, -1),
        lambda: ops.embedding_lookup(ids, w, 1.0, -1),
        lambda: ops.embedding_gradient(wide[:3], ids, 5, 1.0, -1),
        lambda: ops.embedding_gradient(x, ids, 0, 1.0, -1),
        lambda: ops.embedding_gradient(x, ids, 1 << 31, 1.0, -1),
    ):
        with pytest.raises(ValueError, match="does not fit"):
            call()
    for call in (  # refused by the library
        lambda: ops.dropout(x, rng, 1.5, 0),
        lambda: ops.dropout_layernorm(x, None, w, w, None, 1e-5, 0.1, 0),  # no rng
        lambda: ops.dropout_layernorm(x, None, w.half(), w.half(), None, 1e-5, 0.0, 0),
        lambda: ops.dropout_layernorm(torch.zeros(1, 8200, device="cuda"), None,
                                      *[torch.zeros(8200, device="cuda")] * 2, None, 1e-5, 0.0, 0),
    ):
        with pytest.raises(RuntimeError, match="failed with code"):
            call()


def test_embedding_ids_of_other_kinds(dtype):
    from disentangled_flash.training import embedding

    ids = _ids("uniform", 300, 77).view(5, 60)
    _check_embedding(ids.int(), 77, 40, dtype)
    _check_embedding(ids.t(), 77, 40, dtype)
    _check_embedding(ids[:, ::7], 77, 40, dtype)
    _check_embedding(ids[2, 3], 77, 40, dtype)
    table = _normal(_gen(0), (77, 40), dtype)
    assert torch.equal(embedding(ids, table, padding_idx=-1), table[ids])
    shifted = torch.empty(77 * 40 + 1, device="cuda", dtype=dtype)[1:].view(77, 40).copy_(table)
    assert torch.equal(embedding(ids, shifted), table[ids])


@pytest.mark.parametrize("hidden", [64, 33])
def test_embedding_ids_outside_the_table(dtype, hidden):
    """They give NaN, add to nothing, and leave every other row as it is."""

    from disentangled_flash.training import embedding

    ids = _ids("uniform", 200, 30)
    bad = ids.clone()
    where = torch.arange(0, 200, 9, device="cuda")
    bad[where] = torch.tensor([-1, 30, 31, -(1 << 40), 1 << 40, 2 ** 63 - 1, -2 ** 63, -30],
                              device="cuda").repeat(3)[:where.numel()]
    gen = _gen(3)
    table = _normal(gen, (30, hidden), dtype).requires_grad_()
    dy = _normal(gen, (200, hidden), dtype)
    y = embedding(bad, table)
    (grad,) = torch.autograd.grad(y, table, dy)
    good = torch.ones(200, dtype=torch.bool, device="cuda")
    good[where] = False
    assert bool(torch.isnan(y[where]).all()) and torch.equal(y[good], table[ids[good]])
    ref.check(grad, ref.embedding_gradient(ids[good], dy[good], 30, 1.0), "gradient")
    # NaN in the gradient rows of such tokens, and of padding, reaches nothing.
    dy[where] = float("nan")
    dy[bad == 4] = float("inf")
    (again,) = torch.autograd.grad(embedding(bad, table, 1.0, 4), table, dy)
    # (The padding's tokens are sorted behind the others, so sums meet other tiles' edges: the
    # same terms in another grouping, each within the bound of its exact sum.)
    good &= bad != 4
    ref.check(again, ref.embedding_gradient(ids[good], dy[good], 30, 1.0), "with padding")
    every = torch.full((40,), 99, device="cuda")
    (none,) = torch.autograd.grad(embedding(every, table), table, dy[:40])
    assert torch.equal(none, torch.zeros_like(none))


def test_embedding_past_32_bits():
    """A table of more than 2^31 elements: lookups and gradients at its end."""

    from disentangled_flash.training import embedding

    rows, hidden = (1 << 21) + 9, 1024
    table = torch.zeros(rows, hidden, device="cuda", dtype=torch.float16)
    last = _normal(_gen(5), (9, hidden), torch.float16)
    table[-9:] = last
    table.requires_grad_()
    ids = torch.arange(rows - 9, rows, device="cuda").repeat(3)
    y = embedding(ids, table)
    assert torch.equal(y, last.repeat(3, 1))
    dy = _normal(_gen(6), (27, hidden), torch.float16)
    (grad,) = torch.autograd.grad(y, table, dy)
    local = torch.arange(9, device="cuda").repeat(3)
    ref.check(grad[-9:], ref.embedding_gradient(local, dy, 9, 1.0), "last rows")
    assert int(torch.count_nonzero(grad[:-9])) == 0
    del table, grad
    torch.cuda.empty_cache()


# ---- how they are called ---------------------------------------------------------------


def test_gradients_have_fakes():
    """Forward and backward trace through the ops' fake implementations."""

    from disentangled_flash import training

    with FakeTensorMode():
        x = torch.empty(3, 5, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        r = torch.empty(3, 5, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        w, b = (torch.empty(64, device="cuda", requires_grad=True) for _ in range(2))
        table = torch.empty(11, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        ids = torch.empty(3, 5, device="cuda", dtype=torch.int32)
        rng = torch.empty(2, dtype=torch.int64, device="cuda")
        y = training.embedding(ids, table, 2.0, 0) + training.dropout(x, 0.2, rng, 1)
        y = training.layer_norm(y, w, b, 1e-7, r, 0.1, rng, 2)
        grads = torch.autograd.grad(y.sum(), [x, r, w, b, table])
        for grad, leaf in zip(grads, (x, r, w, b, table)):
            assert grad.shape == leaf.shape and grad.dtype == leaf.dtype


def _tail_step(table, ids, w, b, state):
    """Embedding, dropout, and an output block's tail, with every gradient."""

    from disentangled_flash import training

    rng = state.rng
    e = training.embedding(ids, table, 3.0, 0)
    h = training.dropout(e, 0.2, rng, 1)
    y = training.layer_norm(h, w, b, 1e-6, residual=e, p=0.1, rng=rng, site=2)
    return (y.detach(), *torch.autograd.grad(y, [table, w, b], 2 * y.detach()))


def _tail_leaves():
    gen = _gen(12)
    table = _normal(gen, (300, 96), torch.bfloat16).requires_grad_()
    w = _normal(gen, (96,), torch.float32, 0.1, 1.0).requires_grad_()
    b = _normal(gen, (96,), torch.float32, 0.1).requires_grad_()
    return table, w, b


def test_run_of_the_operators_against_float64():
    """The three together as a model uses them, against autograd in float64 with the same
    masks and the same roundings between the operators."""

    from disentangled_flash import training

    table, w, b = _tail_leaves()
    ids = _ids("frequent", 120, 300).view(4, 30)
    state = training.DropoutState(77, "cuda")
    state.advance()
    y, dtable, dw, db = _tail_step(table, ids, w, b, state)
    e = training.embedding(ids, table.detach(), 3.0, 0)
    h = training.dropout(e, 0.2, state.rng, 1)
    m2 = ref.factor((120, 96), 0.1, state.rng, 2)
    flat = lambda t: t.reshape(120, 96)  # noqa: E731
    dy = 2 * y
    want = ref.layer_norm(flat(h), w.detach(), b.detach(), 1e-6, flat(e), m2, flat(dy))
    ref.check(flat(y), want["y"], "y")
    ref.check(dw, want["dweight"], "dw")
    ref.check(db, want["dbias"], "db")
    # de = dresidual + drop'(dx), rounded to bf16 after each operator and after the sum.
    m1 = ref.factor((120, 96), 0.2, state.rng, 1)
    de = want["dresidual"][0] + want["dx"][0] * m1
    slack = want["dresidual"][1] + want["dx"][1] * m1 + 2 * ref.rounding(want["dx"][0] * m1,
                                                                        torch.bfloat16) \
        + 2 * ref.rounding(de, torch.bfloat16)
    value, bound = ref.embedding_gradient(ids, de, 300, 3.0, 0)
    spread, _ = ref.embedding_gradient(ids, slack, 300, 3.0, 0)
    ref.check(dtable, (value, bound + spread * (1 + 2.0 ** -7) + ref.rounding(value, torch.bfloat16)),
              "table")


def test_captured_step_draws_new_masks_and_equals_the_eager_one():
    """Replays of a captured step advance the state; each equals the eager step of its number.
    Eager work and synchronisations lie between the replays."""

    from disentangled_flash import training

    leaves = _tail_leaves()
    ids = _ids("frequent", 120, 300).view(4, 30)
    state = training.DropoutState(5, "cuda")
    static_ids = ids.clone()

    def step():
        state.advance()
        table, w, b = (t.detach().requires_grad_() for t in leaves)
        return _tail_step(table, static_ids, w, b, state)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outputs = step()
    torch.cuda.current_stream().wait_stream(side)
    state.counter[1] = 10
    seen = []
    for i in range(4):
        static_ids.copy_(ids.flip(0) if i == 2 else ids)
        graph.replay()
        got = [t.clone() for t in outputs]
        torch.cuda.synchronize()
        eager = training.DropoutState(5, "cuda")
        eager.counter[1] = 11 + i
        want = _tail_step(*(t.detach().requires_grad_() for t in leaves[:1]), static_ids,
                          *(t.detach().requires_grad_() for t in leaves[1:]), eager)
        for a, c in zip(got, want):
            assert torch.equal(a, c), i
        torch.cuda.synchronize()
        seen.append(got[0])
    assert not torch.equal(seen[0], seen[1])


def test_calls_on_other_streams():
    """Two streams at once, each with its own workspaces."""

    leaves = _tail_leaves()
    from disentangled_flash import training

    ids = _ids("uniform", 4000, 300).view(40, 100)
    state = training.DropoutState(3, "cuda")
    want = _tail_step(leaves[0], ids, leaves[1], leaves[2], state)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for _ in range(3):
        for stream in streams:
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                results.append(_tail_step(leaves[0], ids, leaves[1], leaves[2], state))
    torch.cuda.synchronize()
    for got in results:
        for a, c in zip(got, want):
            assert torch.equal(a, c)


def test_compiled_step_is_the_eager_one():
    """Traced as one graph (fake implementations, the ops' autograd), run eagerly: equal bits."""

    from disentangled_flash import training

    leaves = _tail_leaves()
    ids = _ids("frequent", 120, 300).view(4, 30)
    state = training.DropoutState(6, "cuda")
    rng = state.rng

    def tail(table, ids, w, b, rng):
        e = training.embedding(ids, table, 3.0, 0)
        h = training.dropout(e, 0.2, rng, 1)
        return training.layer_norm(h, w, b, 1e-6, residual=e, p=0.1, rng=rng, site=2)

    want = _tail_step(leaves[0], ids, leaves[1], leaves[2], state)
    y = torch.compile(tail, backend="aot_eager", fullgraph=True)(leaves[0], ids, leaves[1],
                                                                 leaves[2], rng)
    grads = torch.autograd.grad(y, leaves, 2 * y.detach())
    for got, expected in zip((y.detach(), *grads), want):
        assert torch.equal(got, expected)


def test_residual_may_be_the_input():
    """layer_norm(x, residual=x): both gradients reach the one leaf."""

    from disentangled_flash.training import layer_norm

    for p in (0.0, 0.3):
        x, _, w, b, dy = _norm_case(13, 20, 192, torch.float32, torch.float32, False)
        leaf = x.clone().requires_grad_()
        layer_norm(leaf, w, b, 1e-5, residual=leaf, p=p, rng=_rng(), site=SITE).backward(dy)
        mult = ref.factor((20, 192), p, _rng(), SITE)
        want = ref.layer_norm(x, w, b, 1e-5, x, mult, dy)
        value = want["dx"][0] + want["dresidual"][0]
        bound = want["dx"][1] + want["dresidual"][1] + ref.rounding(value, torch.float32)
        ref.check(leaf.grad, (value, bound), "both")


def test_second_derivatives_raise():
    from disentangled_flash.training import dropout, embedding, layer_norm

    x = torch.randn(4, 64, device="cuda", requires_grad=True)
    w, b = torch.ones(64, device="cuda"), torch.zeros(64, device="cuda")
    for y in (layer_norm(x, w, b, 1e-5), embedding(torch.arange(4, device="cuda"), x)):
        (grad,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiate"):
            grad.sum().backward()
    # Dropout is linear: d/dx of (drop'(2 drop(x))) drops the same elements twice.
    y = dropout(x, 0.5, _rng(), SITE)
    (grad,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    (second,) = torch.autograd.grad(grad.sum(), x)
    mult = ref.factor((4, 64), 0.5, _rng(), SITE)
    assert torch.equal(second.double(), 2 * mult * mult)


def test_changing_rng_before_the_backward_pass_raises():
    from disentangled_flash.training import dropout

    rng = _rng()
    x = torch.randn(64, device="cuda", requires_grad=True)
    y = dropout(x, 0.5, rng)
    rng += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_gradients_accumulate_over_micro_batches():
    """Two forwards before their backward passes: each keeps its own step's masks."""

    from disentangled_flash import training

    state = training.DropoutState(1, "cuda")
    x = torch.randn(32, 64, device="cuda", requires_grad=True)
    ys, masks = [], []
    for _ in range(2):
        state.advance()
        ys.append(training.dropout(x, 0.5, state.rng, 3))
        masks.append(ref.factor((32, 64), 0.5, state.rng, 3))
    (ys[0] + ys[1]).sum().backward()
    assert torch.equal(x.grad.double(), masks[0] + masks[1])


# ---- a model -------------------------------------------------------------------------


def _backbone(p):
    from transformers import DebertaV2Config, DebertaV2Model

    torch.manual_seed(5)
    return DebertaV2Model(DebertaV2Config(
        vocab_size=100, hidden_size=64, num_hidden_layers=2, num_attention_heads=2,
        intermediate_size=128, hidden_act="gelu", type_vocab_size=2, max_position_embeddings=64,
        relative_attention=True, position_buckets=16, pos_att_type=["p2c", "c2p"],
        norm_rel_ebd="layer_norm", share_att_key=True, conv_kernel_size=3, conv_act="gelu",
        position_biased_input=True, hidden_dropout_prob=p, attention_probs_dropout_prob=p))


def _batch():
    gen = torch.Generator().manual_seed(2)
    ids = torch.randint(1, 100, (3, 24), generator=gen)
    mask = torch.arange(24)[None] < torch.tensor([[24], [9], [1]])
    types = torch.randint(0, 2, (3, 24), generator=gen)
    return (ids.masked_fill(~mask, 0).cuda(), mask.long().cuda(), types.cuda())


def _loss(model, batch):
    ids, mask, types = batch
    out = model(ids, attention_mask=mask, token_type_ids=types).last_hidden_state
    return ((out.double() * mask[..., None]).square().sum(-1)
            * torch.linspace(0.5, 1.5, 24, device="cuda")).sum()


def test_model_gradients_without_dropout():
    """A training step of a Hugging Face backbone: every parameter's gradient is as close to
    the float64 model's as the unchanged fp32 model's is."""

    from disentangled_flash import enable_deberta_training

    plain = _backbone(0.0).cuda().train()
    exact, ours = copy.deepcopy(plain).double(), enable_deberta_training(copy.deepcopy(plain))
    batch = _batch()
    for model in (plain, exact, ours):
        _loss(model, batch).backward()
    size = max(e.grad.abs().max().item() for e in exact.parameters() if e.grad is not None)
    for (name, e), p, o in zip(exact.named_parameters(), plain.parameters(), ours.parameters()):
        if e.grad is None:
            assert o.grad is None, name
            continue
        error = (o.grad.double() - e.grad).abs().max().item()
        before = (p.grad.double() - e.grad).abs().max().item()
        # 200 half steps of the largest: what a chain of about 20 operators may add.
        assert error <= 2 * before + 200 * ref.U * size, (name, error, before, size)


def test_model_with_dropout_steps():
    """Each training forward draws new masks; the same seed and step give the same bits; eval
    drops nothing; a checkpointed layer's recomputation drops what its forward did."""

    from torch.utils.checkpoint import checkpoint

    from disentangled_flash import enable_deberta_training, training

    model = enable_deberta_training(_backbone(0.1).cuda().train(), seed=21)
    twin = copy.deepcopy(model)
    batch = _batch()
    first, second = _loss(model, batch).item(), _loss(model, batch).item()
    assert first != second and model.dropout_state.counter.tolist() == [21, 2]
    assert _loss(twin, batch).item() == first and _loss(twin, batch).item() == second
    model.eval()
    with torch.no_grad():
        assert _loss(model, batch).item() == _loss(model, batch).item()
    assert model.dropout_state.counter.tolist() == [21, 2]

    block = model.encoder.layer[0].output.train()
    assert isinstance(block, training.OutputBlock)
    x, r = torch.randn(5, 128, device="cuda"), torch.randn(5, 64, device="cuda")
    grads = []
    for run in (block, lambda *a: checkpoint(block, *a, use_reentrant=False)):
        leaf = x.clone().requires_grad_()
        run(leaf, r).square().sum().backward()
        grads.append(leaf.grad)
    assert torch.equal(grads[0], grads[1])


def test_checkpointed_layers_recompute_their_own_forward():
    """Two forwards before one backward pass over both, with and without checkpointed layers:
    the same gradients.  (Other masks would change them by their own size.)"""

    from torch.utils.checkpoint import checkpoint

    from disentangled_flash import enable_deberta_training

    grads = []
    for checkpointed in (False, True):
        model = enable_deberta_training(_backbone(0.2).cuda().train(), seed=8)
        if checkpointed:
            for layer in model.encoder.layer:
                block = layer.output
                block.forward = functools.partial(checkpoint, block.forward, use_reentrant=False)
        ids, mask, types = _batch()
        first = _loss(model, (ids, mask, types))
        second = _loss(model, (ids.flip(0), mask.flip(0), types))
        (first + second).backward()
        third = _loss(model, (ids, mask, types))
        third.backward()
        grads.append({n: p.grad for n, p in model.named_parameters() if p.grad is not None})
    assert grads[0].keys() == grads[1].keys()
    for name in grads[0]:
        # torch adds the gradients of the attention's gathers with atomics: the same terms in
        # another order, through two layers and three forwards; 100 half steps of the largest.
        size = grads[0][name].abs().max().item()
        difference = (grads[1][name] - grads[0][name]).abs().max().item()
        assert difference <= 100 * ref.U * size, (name, difference, size)


def test_compiled_model_draws_the_masks_of_its_step():
    """A compiled backbone steps and drops as the eager one; the counter is not baked in."""

    from disentangled_flash import enable_deberta_training

    batch, grads = _batch(), []
    for compiled in (False, True):
        model = enable_deberta_training(_backbone(0.2).cuda().train(), seed=8)
        call = torch.compile(model, backend="aot_eager") if compiled else model
        steps = []
        for _ in range(3):
            model.zero_grad()
            _loss(call, batch).backward()
            steps.append({n: p.grad for n, p in model.named_parameters() if p.grad is not None})
        assert model.dropout_state.counter.tolist() == [8, 3]
        grads.append(steps)
    for eager, compiled in zip(*grads):
        assert eager.keys() == compiled.keys()
        for name in eager:
            # torch's own operators may be decomposed otherwise: 1000 half steps of the largest,
            # where other masks would change a gradient by its own size.
            size = eager[name].abs().max().item()
            difference = (compiled[name] - eager[name]).abs().max().item()
            assert difference <= 1000 * ref.U * size, (name, difference, size)


def test_output_block_under_autocast():
    from disentangled_flash import enable_deberta_training

    model = enable_deberta_training(_backbone(0.0).cuda().train())
    batch = _batch()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = _loss(model, batch)
    loss.backward()
    for name, p in model.named_parameters():
        assert p.grad is None or bool(torch.isfinite(p.grad).all()), name


def test_trained_model_goes_on_to_inference():
    from disentangled_flash import enable_deberta_training, optimize_deberta

    model = enable_deberta_training(_backbone(0.1).cuda().train())
    _loss(model, _batch()).backward()
    model.eval()
    ids, mask, types = _batch()
    with torch.inference_mode():
        want = model(ids, attention_mask=mask, token_type_ids=types).last_hidden_state
        optimize_deberta(model, sequence_lengths=[24])
        got = model(ids, attention_mask=mask, token_type_ids=types).last_hidden_state
    kept = mask.bool()[..., None]
    assert ((got - want).abs() * kept).max().item() <= 1e-5
