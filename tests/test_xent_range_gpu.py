"""fp32 values of any size on the products' path: a row, a feature, a class or a row weight far
above the others changes nothing for them.

Bounds per output, from the absolute values that enter that output alone (u = 2^-24):
  products   an fp32 operand is held exactly, as three parts of 8 bits; what is left out of a
             product, the last two parts' with each other, is below 3 x 2^-23 of |x||w|
  sums       K / 16 + 32 additions a part in fp32, each at most 2u of the sum of absolute values
  logits     E_i = (products + sums) max_j (sum_k |x_ik w_jk| + |b_j|)
  loss       2 E_i + 32u (|z_y| + |lse| + 1)
  g          p r (2 E_i + 32u (1 + |lse| + |z|)) and 2^-22 of g
  gradients  those through |x| or |w|, the products' and sums' share of sum |g||x|, and u of the result
"""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from gafime_b200 import _native, ops as o
    _native.load()
    return o


def data(n=400, d=40, c=130, seed=0, order="rows"):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((n, d), generator=g, device="cuda")
    if order == "columns":
        x = x.t().contiguous().t()
    w = torch.randn((c, d), generator=g, device="cuda") * (1.5 / math.sqrt(d))
    b = torch.randn(c, generator=g, device="cuda")
    labels = torch.randint(0, c, (n,), generator=g, device="cuda")
    r = torch.rand(n, generator=g, device="cuda") + 0.25
    return x, w, labels, b, r


def reference(x, w, labels, b, r):
    n, d = x.shape
    c = w.shape[0]
    kept = labels >= 0
    X, W, B = torch.where(kept[:, None], x.double(), 0.0), w.double(), b.double()
    Z = X @ W.t() + B
    lse = torch.logsumexp(Z, 1)
    at = labels.clamp(min=0)[:, None]
    zy = Z.gather(1, at)[:, 0]
    # the loss by differences, so that large logits do not cancel
    loss = torch.logsumexp(Z - zy[:, None], 1)
    R = torch.where(kept, r.double(), 0.0)
    P = torch.exp(Z - lse[:, None])
    G = P.clone()
    G.scatter_add_(1, at, -torch.ones_like(at, dtype=torch.float64))
    G *= R[:, None]
    held = 3 * 2.0 ** -23

    def sums(k):
        return 6 * (k / 16 + 32) * 2 * U

    E = (held + sums(d)) * (X.abs() @ W.abs().t() + B.abs()).amax(1)
    tol = 2 * E + 32 * U * (zy.abs() + lse.abs() + 1)
    dG = P * R[:, None] * (2 * E + 32 * U * (1 + lse.abs() + Z.abs().amax(1)))[:, None] + G.abs() * (2.0 ** -22 + 8 * U)
    A = G.abs() + dG

    def result(value, t):
        return value, t * (1 + 2 * U) + U * (value.abs() + t) + 1e-38

    return {"loss": (torch.where(kept, loss, 0.0), torch.where(kept, tol, 0.0)),
            "dw": result(G.t() @ X, dG.t() @ X.abs() + (held + sums(n)) * (A.t() @ X.abs())),
            "dx": result(G @ W, dG @ W.abs() + (held + sums(c)) * (A @ W.abs())),
            "dbias": (G.sum(0), dG.sum(0) + 64 * U * A.sum(0) + U * G.sum(0).abs())}


def compare(name, got, want, rows=None):
    value, tol = want
    if rows is not None:
        got, value, tol = got[rows], value[rows], tol[rows]
    err = (got.double() - value).abs()
    assert bool((err <= tol).all()), (name, int((~(err <= tol)).sum()), float((err / tol.clamp(min=1e-300)).max()))


def check(ops, x, w, labels, b, r, rows=None):
    want = reference(x, w, labels, b, r)
    compare("loss alone", ops.softmax_xent(x, w, labels, b), want["loss"], rows)
    g = ops.softmax_xent_grad(x, w, labels, b, row_weight=r)
    compare("loss", g.loss, want["loss"], rows)
    compare("dx", g.dx, want["dx"], rows)
    compare("dw", g.dw, want["dw"])
    compare("dbias", g.dbias, want["dbias"])


@pytest.mark.parametrize("order", ["rows", "columns"])
@pytest.mark.parametrize("c", [17, 130, 300])
@pytest.mark.parametrize("entry", [1e5, 1e7, 1e9, -999999999.0, 1e12, 1e30, 3.4e38])
def test_a_large_value_stays_in_its_row(ops, entry, c, order):
    """The other rows' losses and gradients are those of the same batch without that row, bit by bit."""
    x, w, labels, b, r = data(c=c, order=order)
    x[77, 13] = entry
    others = torch.ones(len(labels), dtype=torch.bool, device="cuda")
    others[77] = False
    without = torch.where(others, labels, torch.full_like(labels, -1))
    a = ops.softmax_xent_grad(x, w, labels, b, row_weight=r)
    q = ops.softmax_xent_grad(x, w, without, b, row_weight=r)
    assert torch.equal(a.loss[others], q.loss[others]) and torch.equal(a.dx[others], q.dx[others])
    assert torch.equal(ops.softmax_xent(x, w, labels, b)[others], ops.softmax_xent(x, w, without, b)[others])
    check(ops, x, w, without, b, r)
    if abs(entry) <= 1e30:   # (past that the row's own logits leave fp32)
        check(ops, x, w, labels, b, r)


@pytest.mark.parametrize("n,d,c", [(400, 40, 9), (60, 2100, 3), (9, 40, 30)])
def test_a_large_value_at_the_paths_borders(ops, n, d, c):
    """The smallest class counts with gradients, many features, few rows."""
    x, w, labels, b, r = data(n, d, c, seed=1)
    x[5, 3] = 1e10
    check(ops, x, w, labels, b, r)


@pytest.mark.parametrize("order", ["rows", "columns"])
@pytest.mark.parametrize("size", [1.0, 1e-4, 1e-6, 1e-8, 1e-18])
def test_a_feature_of_zeros_beside_small_ones(ops, size, order):
    """Its weights multiply nothing, whatever the others' sizes; its dx is that of any feature."""
    x, w, labels, b, r = data(c=300, d=64, seed=2, order=order)
    x *= size
    w /= size
    x[:, 5] = 0.0
    labels[::3] = -1
    x[:, 6] = torch.where(labels < 0, x[:, 6], torch.zeros_like(x[:, 6]))   # zero where it counts
    check(ops, x, w, labels, b, r)


@pytest.mark.parametrize("unit", [2.0 ** 20, 2.0 ** 26, 2.0 ** 30, 2.0 ** 40, 2.0 ** -30])
def test_gradients_beside_a_feature_of_another_size(ops, unit):
    """dx of a feature is a sum over its own weights, however large another column is."""
    x, w, labels, b, r = data(c=64, seed=3)
    x[:, 7] *= unit
    check(ops, x, w, labels, b, r)


def test_mixed_units_that_the_weights_do_not_make_up_for(ops):
    x, w, labels, b, r = data(c=90, d=36, seed=4)
    x *= 10.0 ** torch.linspace(-8, 8, 36, device="cuda")
    check(ops, x, w, labels, b, r)


@pytest.mark.parametrize("big", [2.0 ** 20, 2.0 ** 40, 2.0 ** 80])
def test_one_row_weight_far_above_the_others(ops, big):
    x, w, labels, b, r = data(c=90, seed=5)
    r[11] *= big
    check(ops, x, w, labels, b, r)


@pytest.mark.parametrize("big", [1e6, 1e12, 1e24])
def test_one_class_of_large_weights(ops, big):
    """The others' weights keep their bits in dx (the class itself takes every row, or none)."""
    x, w, labels, b, r = data(c=90, seed=6)
    w[17] *= big
    check(ops, x, w, labels, b, r)


def test_an_outlier_without_weight(ops):
    """A row of weight zero, as a mask leaves it, takes no part in dw, however large its values."""
    x, w, labels, b, r = data(c=70, seed=7)
    x[40] = 1e15
    r[40] = 0.0
    w *= 1e-16
    check(ops, x, w, labels, b, r)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("big", [2.0 ** 10, 2.0 ** 20])
def test_row_weights_in_16_bits(ops, big, dtype):
    """dx of the other rows is within its type's roundings (g once, the result once)."""
    x, w, labels, b, r = data(c=90, seed=8)
    x, w = x.to(dtype), w.to(dtype)
    r /= big
    r[11] = 1.0
    want = reference(x, w, labels, b, r)
    half = torch.finfo(dtype).eps / 2
    A = want["dx"][0].abs() + (torch.softmax(x.double() @ w.double().t() + b, 1).scatter_add(
        1, labels[:, None], torch.ones_like(labels[:, None], dtype=torch.float64)) * r.double()[:, None]) @ w.double().abs()
    g = ops.softmax_xent_grad(x, w, labels, b, row_weight=r)
    err = (g.dx.double() - want["dx"][0]).abs()
    tol = want["dx"][1] + half * 2.1 * A + (2.0 ** -25 if dtype == F16 else 0.0)
    if dtype == F16:     # g itself: 2^-38 of the largest row weight
        tol = tol + 2.0 ** -37 * w.double().abs().sum(0)
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("n,c", [(20, 5), (200, 40), (300, 300), (20, 16), (4, 64)])
def test_a_weight_of_minus_infinity_excludes_its_class(ops, n, c):
    """z of that class is -inf in rows whose feature is positive: no part in their softmax, as with a
    bias of -inf; a row whose feature is negative gets +inf and a loss that is no number."""
    x, w, labels, b, _ = data(n, 24, c, seed=9)
    w[4, 2] = float("-inf")
    x[:, 2] = x[:, 2].abs() + 0.1
    x[0, 2] *= -1.0
    labels = torch.where(labels == 4, torch.zeros_like(labels), labels)
    z = x[1:].double() @ torch.where(torch.isinf(w), 0.0, w.double()).t() + b.double()
    z[:, 4] = float("-inf")
    want = torch.logsumexp(z - z.gather(1, labels[1:, None]), 1)
    for got in (ops.softmax_xent(x, w, labels, b), ops.softmax_xent_grad(x, w, labels, b).loss):
        assert torch.isnan(got[0])
        assert ((got[1:].double() - want).abs() <= 64 * U * (want.abs() + 16)).all()
    # without the row of +inf: dw as with the class left out
    g = ops.softmax_xent_grad(x[1:], w, labels[1:], b, need_dx=False)
    p = torch.softmax(z, 1)
    p.scatter_add_(1, labels[1:, None], -torch.ones((n - 1, 1), device="cuda", dtype=torch.float64))
    size = p.abs().t() @ x[1:].double().abs()
    assert ((g.dw.double() - p.t() @ x[1:].double()).abs() <= 256 * U * size + 1e-30).all()
    assert not g.dw[4].any() and g.dbias[4] == 0
    # dx: 0 x inf is no number, as the definition has it; the other features hold theirs
    g = ops.softmax_xent_grad(x[1:], w, labels[1:], b)
    assert torch.isnan(g.dx[:, 2]).all()
    rest = [k for k in range(24) if k != 2]
    size = p.abs() @ w.double().abs()[:, rest]
    assert ((g.dx[:, rest].double() - p @ w.double()[:, rest]).abs() <= 256 * U * size + 1e-30).all()
    # its label: an infinite loss
    labels[1] = 4
    got = ops.softmax_xent(x, w, labels, b)
    assert math.isinf(float(got[1])) and float(got[1]) > 0


@pytest.mark.parametrize("order", ["rows", "columns"])
@pytest.mark.parametrize("n,d,c", [(300, 200, 100), (700, 520, 300), (260, 130, 60), (40, 700, 4000)])
def test_infinite_weights_in_tables_of_several_blocks(ops, n, d, c, order):
    """Every width of a class tile, several blocks of features, and the losses after the backward pass."""
    x, w, labels, b, r = data(n, d, c, seed=10, order=order)
    x[:, d - 3] = x[:, d - 3].abs() + 0.1
    labels = torch.where(labels % 7 == 3, torch.zeros_like(labels), labels)
    off = (torch.arange(c, device="cuda") % 7 == 3)
    excluded = torch.where(off, float("-inf"), b)
    finite = w.clone()
    w[off, d - 3] = float("-inf")
    want = ops.softmax_xent_grad(x, finite, labels, excluded, row_weight=r)
    got = ops.softmax_xent_grad(x, w, labels, b, row_weight=r)
    assert torch.equal(got.loss, want.loss) and torch.equal(got.dw, want.dw) and torch.equal(got.dbias, want.dbias)
    rest = [k for k in range(d) if k != d - 3]
    assert torch.equal(got.dx[:, rest], want.dx[:, rest]) and torch.isnan(got.dx[:, d - 3]).all()
    leaf = w.clone().requires_grad_()
    loss = ops.softmax_xent(x, leaf, labels, b)
    assert torch.equal(loss, ops.softmax_xent(x, finite, labels, excluded))
    loss.backward(r)
    assert torch.isfinite(leaf.grad).all() and not leaf.grad[off].any()
