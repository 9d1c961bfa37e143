"""Softmax cross entropy of a linear head, and its gradients, against the definition in 64 bits.

Tolerances are worst-case bounds of the arithmetic, computed per output from the absolute values
that enter it (u = 2^-24, half a step of fp32):
  products   16-bit operands multiply exactly; fp32 operands are held to 2^-22 each on the tensor
             cores, and their lo lo product (2^-22) is dropped: 3 x 2^-22 of |x||w|; values far
             below their feature's largest are held to 2^-38 of it
  sums       K / 16 + 32 additions an operand pair in fp32, each at most 2u of the sum of
             absolute values (the tensor cores may cut instead of rounding)
  logits     E_i = (products + sums) max_j (sum_k |x_ik w_jk| + |b_j|)
  loss       2 E_i, and 32u of |z_y| + |lse| + 1 for the exponentials, the logarithm and the end
  g          p r (2 E_i + 32u (1 + |lse| + |z|)) and its rounding to the products' type:
             finfo.eps / 2 in 16 bits, 2^-22 where it is split
  gradients  those through |x| or |w|, the products' and sums' share of sum |g||x|, and the
             rounding of the result, finfo.eps / 2
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from gafime_b200 import _native, ops as o
    _native.load()
    return o


def data(n, d, c, dtype=F32, order="rows", left_out=0.0, seed=0, bias=True, w_order="rows"):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def matrix(rows, cols, order, scale):
        t = torch.randn((rows, cols), generator=g, device="cuda") * scale
        if order == "columns":
            return t.to(dtype).t().contiguous().t()
        if order == "pitched":        # rows longer than the features
            wide = torch.zeros((rows, cols + 5), device="cuda", dtype=dtype)
            wide[:, 2:2 + cols] = t.to(dtype)
            return wide[:, 2:2 + cols]
        if order == "aligned":        # rows longer than the features, on 16-byte boundaries
            wide = torch.zeros((rows, (cols + 7) // 8 * 8 + 8), device="cuda", dtype=dtype)
            wide[:, :cols] = t.to(dtype)
            return wide[:, :cols]
        if order == "every other":    # no unit stride
            wide = torch.zeros((rows, 2 * cols), device="cuda", dtype=dtype)
            wide[:, ::2] = t.to(dtype)
            return wide[:, ::2]
        return t.to(dtype)

    x = matrix(n, d, order, 1.0)
    w = matrix(c, d, w_order, 1.5 / math.sqrt(d))
    b = torch.randn(c, generator=g, device="cuda") if bias else None
    labels = torch.randint(0, c, (n,), generator=g, device="cuda")
    labels[torch.rand(n, generator=g, device="cuda") < left_out] = -1
    r = torch.rand(n, generator=g, device="cuda") + 0.25
    return x, w, labels, b, r


def reference(x, w, labels, bias, r):
    """Definition in fp64 with the bounds: {name: (value, tolerance)}."""
    n, d = x.shape
    c = w.shape[0]
    dtype = x.dtype
    kept = labels >= 0
    X = torch.where(kept[:, None], x.double(), 0.0)
    W = w.double()
    b = torch.zeros(c, dtype=torch.float64, device=x.device) if bias is None else bias.double()
    Z = X @ W.t() + b
    lse = torch.logsumexp(Z, 1)
    at = labels.clamp(min=0)[:, None]
    zy = Z.gather(1, at)[:, 0]
    loss = torch.where(kept, lse - zy, 0.0)
    R = torch.where(kept, r.double(), 0.0)
    P = torch.exp(Z - lse[:, None])
    Gm = P.clone()
    Gm.scatter_add_(1, at, -torch.ones_like(at, dtype=torch.float64))
    Gm *= R[:, None]

    held = 3 * 2.0 ** -22 if dtype == F32 else 0.0
    passes = 3 if dtype == F32 else 1

    def sums(k):
        return passes * (k / 16 + 32) * 2 * U

    fb = torch.where(torch.isfinite(b), b.abs(), 0.0)
    floor = 0.0
    if dtype == F32:
        # 2^-38 of a feature's largest value (of the largest scaled weight) times the other side
        cm = X.abs().amax(0)
        floor = 2.0 ** -37 * d * float((W.abs() * cm).max())
    E = (held + sums(d)) * ((X.abs() @ W.abs().t()) + fb).amax(1) + floor
    finite_z = torch.where(torch.isfinite(Z), Z.abs(), 0.0).amax(1)
    tol_loss = 2 * E + 32 * U * (zy.abs() + lse.abs() + 1)
    rounding = HALF[dtype] if dtype != F32 else 2.0 ** -22
    rmax = float(R.max()) if n else 0.0
    dG = P * R[:, None] * (2 * E + 32 * U * (1 + lse.abs() + finite_z))[:, None] + Gm.abs() * (rounding + 8 * U) \
        + (2.0 ** -37 * rmax if dtype != BF16 else 2.0 ** -120)
    dG = torch.where(kept[:, None], dG, 0.0)
    out = {"loss": (loss, torch.where(kept, tol_loss, 0.0)),
           "lse": (torch.where(kept, lse, 0.0), torch.where(kept, tol_loss, 0.0))}
    A = Gm.abs() + dG

    def result(value, tol):
        return value, tol * (1 + 2 * U) + HALF[dtype] * (value.abs() + tol) + (2.0 ** -25 if dtype == F16 else 1e-38)

    fx = 2.0 ** -37 * (X.abs().amax(0)[None, :] * A.sum(0)[:, None]) if dtype == F32 else 0.0
    out["dw"] = result(Gm.t() @ X, dG.t() @ X.abs() + (held + sums(n)) * (A.t() @ X.abs()) + fx)
    fw = floor / max(d, 1) * A.sum(1, keepdim=True) / torch.where(cm > 0, cm, 1.0) if dtype == F32 else 0.0
    out["dx"] = result(Gm @ W, dG @ W.abs() + (held + sums(c)) * (A @ W.abs()) + fw)
    out["dx"] = (out["dx"][0], torch.where(kept[:, None], out["dx"][1], 0.0))
    db = Gm.sum(0)
    out["dbias"] = (db, dG.sum(0) + 64 * U * A.sum(0) + U * db.abs())
    return out


def compare(name, got, want):
    value, tol = want
    assert got.shape == value.shape, name
    err = (got.double() - value).abs()
    bad = ~(err <= tol)
    assert not bool(bad.any()), (name, int(bad.sum()), float((err - tol).max()), float((err / tol.clamp(min=1e-300)).max()))


def check(ops, x, w, labels, b, r, need_dx=True):
    want = reference(x, w, labels, b, r)
    loss = ops.softmax_xent(x, w, labels, b)
    compare("loss", loss, want["loss"])
    g = ops.softmax_xent_grad(x, w, labels, b, row_weight=r, need_dx=need_dx)
    compare("loss of the gradient call", g.loss, want["loss"])
    compare("lse", g.lse, want["lse"])
    compare("dw", g.dw, want["dw"])
    if b is None:
        assert g.dbias is None
    else:
        compare("dbias", g.dbias, want["dbias"])
    if need_dx:
        compare("dx", g.dx, want["dx"])
        assert g.dx.dtype == x.dtype and g.dw.dtype == w.dtype
    else:
        assert g.dx is None


FEW = [(1, 1, 1), (1, 5, 2), (2, 1, 3), (7, 33, 2), (31, 50, 16), (257, 31, 4), (1000, 50, 2), (1003, 129, 5),
       (4099, 257, 3), (500, 513, 7), (333, 1024, 16), (777, 1500, 8), (130, 2048, 2), (64, 2047, 8), (20001, 8, 9)]
MANY = [(1, 8, 17), (1, 1000, 300), (3, 1, 33), (127, 64, 64), (129, 65, 65), (128, 128, 128), (300, 200, 129),
        (1000, 50, 257), (513, 333, 1000), (200, 2049, 3), (65, 1537, 16), (2000, 96, 5000), (1, 64, 50001)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,d,c", FEW + MANY)
def test_sizes(ops, n, d, c, dtype):
    check(ops, *data(n, d, c, dtype, left_out=0.2, seed=n + d + c))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("order", ["columns", "pitched", "aligned", "every other"])
@pytest.mark.parametrize("n,d,c", [(515, 45, 3), (96, 1025, 2), (260, 72, 40), (150, 45, 300)])
def test_orders_of_x(ops, n, d, c, order, dtype):
    check(ops, *data(n, d, c, dtype, order=order, left_out=0.1, seed=3))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("order", ["columns", "rows"])
@pytest.mark.parametrize("d", [1, 16, 33, 64, 65, 128, 129, 256, 300])
@pytest.mark.parametrize("n,c", [(20008, 2), (19040, 3), (33056, 5), (20008, 8)])
def test_whole_tiles_of_rows(ops, n, d, c, order, dtype):
    """Enough rows that every SM has tiles of 32 rows, and some at the end without any."""
    x, w, labels, b, r = data(n, d, c, dtype, order=order, left_out=0.1, seed=12)
    out = labels < 0
    x[out.nonzero()[::3, 0]] = float("nan")
    want = reference(x, w, labels, b, r)
    compare("loss", ops.softmax_xent(x, w, labels, b), want["loss"])
    for need_dx in (False, True):
        g = ops.softmax_xent_grad(x, w, labels, b, row_weight=r, need_dx=need_dx)
        for name in ("loss", "lse", "dw", "dbias") + (("dx",) if need_dx else ()):
            compare(name, getattr(g, name), want[name])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("order", ["columns", "pitched", "aligned", "every other"])
@pytest.mark.parametrize("n,d,c", [(100, 45, 3), (140, 72, 70)])
def test_orders_of_w(ops, n, d, c, order, dtype):
    check(ops, *data(n, d, c, dtype, w_order=order, seed=4))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,d,c", [(4000, 64, 20_000), (170_000, 32, 200), (40_000, 24, 3000)])
def test_several_pieces_of_the_gradient(ops, n, d, c, dtype):
    check(ops, *data(n, d, c, dtype, left_out=0.1, seed=5))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("c", [17, 32, 33, 64, 65, 96, 128, 129, 200, 256, 257])
def test_every_class_in_one_tile(ops, c, dtype):
    """Loss and gradients from one computation of the logits, and from a loss call before."""
    x, w, labels, b, r = data(389, 70, c, dtype, left_out=0.2, seed=13)
    x[(labels < 0).nonzero()[::2, 0]] = float("nan")
    want = reference(x, w, labels, b, r)
    g = ops.softmax_xent_grad(x, w, labels, b, row_weight=r)
    for name in ("loss", "lse", "dw", "dx", "dbias"):
        compare(name, getattr(g, name), want[name])
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    loss = ops.softmax_xent(leaves[0], leaves[1], labels, leaves[2])
    compare("loss", loss.detach(), want["loss"])
    loss.backward(r)
    for name, leaf in zip(("dx", "dw", "dbias"), leaves):
        compare(name + " of the backward pass", leaf.grad, want[name])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("c,kept", [(256, (0, 128)), (256, (128, 256)), (100, (0, 50)), (100, (64, 100)), (40, (39, 40))])
def test_a_run_of_classes_excluded(ops, c, kept, dtype):
    x, w, labels, b, r = data(200, 32, c, dtype, seed=14)
    out = torch.ones(c, dtype=torch.bool, device="cuda")
    out[kept[0]:kept[1]] = False
    labels = labels % (kept[1] - kept[0]) + kept[0]
    for shift in (0.0, -300.0, 300.0):
        bias = torch.where(out, float("-inf"), b + shift)
        want = reference(x, w, labels, bias, r)
        g = ops.softmax_xent_grad(x, w, labels, bias, row_weight=r)
        for name in ("loss", "lse", "dx"):
            compare(name, getattr(g, name), want[name])
        assert not g.dw[out].any() and not g.dbias[out].any()


def test_one_tile_of_classes_in_several_pieces(ops):
    check(ops, *data(300_000, 8, 200, F32, left_out=0.1, seed=15))


@pytest.mark.parametrize("c", [2, 60])
def test_without_a_bias(ops, c):
    check(ops, *data(300, 40, c, F32, bias=False, seed=6))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("c", [3, 90])
def test_rows_left_out_hold_anything(ops, c, dtype):
    """NaN and infinities in left-out rows reach nothing; a batch of such rows alone is all zeros."""
    x, w, labels, b, r = data(517, 64, c, dtype, left_out=0.3, seed=7)
    x[labels < 0] = float("nan")
    x[(labels < 0).nonzero()[::2, 0]] = float("-inf")
    r[labels < 0] = float("nan")
    want = reference(x, w, labels, b, torch.where(labels < 0, torch.ones_like(r), r))
    g = ops.softmax_xent_grad(x, w, labels, b, row_weight=r)
    for name in ("loss", "lse", "dw", "dx", "dbias"):
        compare(name, getattr(g, name), want[name])
    g = ops.softmax_xent_grad(x, w, torch.full_like(labels, -100), b, row_weight=r)
    for name in ("loss", "lse", "dw", "dx", "dbias"):
        assert not getattr(g, name).any(), name


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("c", [4, 70])
def test_excluded_classes(ops, c, dtype):
    """A bias of -inf takes a class out; one of the type's lowest value does nearly so."""
    x, w, labels, b, r = data(200, 32, c, dtype, seed=8)
    b[0] = float("-inf")
    b[1] = torch.finfo(torch.float32).min
    labels = torch.where(labels < 2, torch.full_like(labels, 2), labels)
    want = reference(x, w, labels, b, r)
    g = ops.softmax_xent_grad(x, w, labels, b, row_weight=r)
    for name in ("loss", "dx"):
        compare(name, getattr(g, name), (want[name][0], want[name][1]))
    assert not g.dw[:2].any() and not g.dbias[:2].any()
    # a row whose own class is excluded has an infinite loss, and leaves the others as they are
    labels[5] = 0
    loss = ops.softmax_xent(x, w, labels, b)
    assert math.isinf(float(loss[5])) and float(loss[5]) > 0
    assert torch.isfinite(torch.cat([loss[:5], loss[6:]])).all()


@pytest.mark.parametrize("c", [5, 130])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_values_that_are_not_finite_stay_in_their_row(ops, c, dtype):
    x, w, labels, b, r = data(140, 40, c, dtype, seed=9)
    x[17, 3] = float("nan")
    x[99, 0] = float("inf")
    labels[60] = c           # no such class
    g = ops.softmax_xent_grad(x, w, labels, b, row_weight=r)
    odd = torch.zeros(140, dtype=torch.bool, device="cuda")
    odd[[17, 99, 60]] = True
    assert torch.isnan(g.loss[odd]).all() and torch.isfinite(g.loss[~odd]).all()
    assert torch.isnan(g.dx[odd]).all() and torch.isfinite(g.dx[~odd]).all()
    assert torch.isnan(g.dw).all() and torch.isnan(g.dbias).all()


@pytest.mark.parametrize("c", [2, 300])
def test_no_rows(ops, c):
    x, w, labels, b, r = data(0, 12, c)
    assert ops.softmax_xent(x, w, labels, b).shape == (0,)
    g = ops.softmax_xent_grad(x, w, labels, b, row_weight=r)
    assert g.dx.shape == (0, 12) and not g.dw.any() and not g.dbias.any()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("c", [6, 200])
def test_features_of_very_different_scale(ops, c, dtype):
    """Features of sizes 1e-4 .. 1e4, with weights that make up for it, as in a table of mixed units."""
    x, w, labels, b, r = data(400, 36, c, torch.float32, seed=10)
    unit = 10.0 ** torch.linspace(-4, 4, 36, device="cuda")
    if dtype == F16:
        unit = unit.clamp(1e-2, 1e2)
    x, w = (x * unit).to(dtype), (w / unit).to(dtype)
    check(ops, x, w, labels, b, r)


@pytest.mark.parametrize("c", [4, 80])
def test_large_logits(ops, c):
    """Logits of some hundreds: the exponentials of most classes vanish, the loss stays exact."""
    x, w, labels, b, r = data(300, 64, c, seed=11)
    check(ops, x * 20.0, w * 5.0, labels, b, r)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("weight", [1e-6, 1.0, 3e4])
def test_row_weights_of_any_size(ops, weight, dtype):
    x, w, labels, b, r = data(300, 64, 90, dtype, seed=12)
    want = reference(x, w, labels, b, r * weight)
    g = ops.softmax_xent_grad(x, w, labels, b, row_weight=r, scale=weight)
    if dtype != F16 or weight == 1.0:
        compare("dw", g.dw, want["dw"])
        compare("dx", g.dx, want["dx"])
    compare("dbias", g.dbias, want["dbias"])
    g = ops.softmax_xent_grad(x, w, labels, b, scale=0.0)
    assert not g.dw.any() and not g.dx.any() and not g.dbias.any()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,d,c", [(300, 40, 3), (300, 40, 90)])
def test_autograd(ops, n, d, c, dtype):
    x, w, labels, b, r = data(n, d, c, dtype, left_out=0.2, seed=13)
    want = reference(x, w, labels, b, r)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    loss = ops.softmax_xent(leaves[0], leaves[1], labels, leaves[2])
    held = loss.detach().clone()
    (loss * r).sum().backward()
    compare("dx", leaves[0].grad, want["dx"])
    compare("dw", leaves[1].grad, want["dw"])
    compare("dbias", leaves[2].grad, want["dbias"])
    # a mean hands down one value for all rows, and only what needs a gradient gets one
    x2 = x.clone()
    w2 = w.clone().requires_grad_(True)
    ops.softmax_xent(x2, w2, labels, b).mean().backward()
    want = reference(x, w, labels, b, torch.full_like(r, 1.0 / n))
    compare("dw of the mean", w2.grad, want["dw"])
    assert x2.grad is None
    # the backward pass reads the loss: a write into it is noticed, as torch's own operators do
    w3 = w.clone().requires_grad_(True)
    loss = ops.softmax_xent(x, w3, labels, b)
    with torch.no_grad():
        loss.mul_(0.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(loss, w3, torch.ones_like(loss))
    assert torch.equal(held, ops.softmax_xent(x, w, labels, b))


def test_broadcast_inputs(ops):
    """One row of features for all rows, one weight row for all classes: expanded views."""
    x, w, labels, b, r = data(64, 24, 40, seed=14)
    x1 = x[:1].clone().requires_grad_(True)
    loss = ops.softmax_xent(x1.expand(64, 24), w, labels, b)
    (loss * r).sum().backward()
    want = reference(x1.detach().expand(64, 24).contiguous(), w, labels, b, r)
    compare("dx", x1.grad[0], (want["dx"][0].sum(0), want["dx"][1].sum(0) + 64 * U * want["dx"][0].abs().sum(0)))
    g = ops.softmax_xent_grad(x, w[:1].expand(40, 24), labels, b, row_weight=r)
    want = reference(x, w[:1].expand(40, 24).contiguous(), labels, b, r)
    compare("dw", g.dw, want["dw"])


@pytest.mark.parametrize("c", [3, 45])
def test_gradient_against_differences(ops, c):
    """Central differences of the summed loss along random directions: third-order terms of a
    step h are below h^2 |direction|^3, the losses' rounding below 2^-20 of their sum over h."""
    x, w, labels, b, r = data(64, 20, c, seed=15)
    g = ops.softmax_xent_grad(x, w, labels, b, row_weight=r)
    gen = torch.Generator(device="cuda").manual_seed(1)
    h = 2.0 ** -7

    def total(xx, ww, bb):
        return float((ops.softmax_xent(xx, ww, labels, bb).double() * r.double()).sum())

    size = total(x, w, b)
    for name, t in (("dx", x), ("dw", w), ("dbias", b)):
        v = torch.randn(t.shape, generator=gen, device="cuda")
        v /= v.norm()
        args = {"dx": x, "dw": w, "dbias": b}
        up, down = dict(args), dict(args)
        up[name], down[name] = t + h * v, t - h * v
        slope = (total(up["dx"], up["dw"], up["dbias"]) - total(down["dx"], down["dw"], down["dbias"])) / (2 * h)
        want = float((getattr(g, name).double() * v.double()).sum())
        # |d^3 loss_i| <= (largest logit change)^3, the change at most |x_i| or |w|_2 or 1 a unit
        reach = {"dx": float(w.norm()), "dw": float(x.norm(dim=1).max()), "dbias": 1.0}[name]
        assert abs(slope - want) <= h * h * reach ** 3 * float(r.sum()) / 3 + 2.0 ** -20 * size / h


@pytest.mark.parametrize("c", [2, 12, 100, 3000])
def test_results_are_the_same_every_time(ops, c):
    x, w, labels, b, r = data(3001, 77, c, left_out=0.1, seed=16)
    first = ops.softmax_xent_grad(x, w, labels, b, row_weight=r)
    for _ in range(3):
        again = ops.softmax_xent_grad(x, w, labels, b, row_weight=r)
        for a, q in zip(first, again):
            assert torch.equal(a, q)


@pytest.mark.parametrize("c", [3, 64])
def test_streams_and_graphs(ops, c):
    """A call on a side stream; a captured step replayed on new data, while eager work goes on."""
    x, w, labels, b, r = data(700, 40, c, left_out=0.1, seed=17)
    plain = ops.softmax_xent_grad(x, w, labels, b, row_weight=r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.softmax_xent_grad(x, w, labels, b, row_weight=r)
    torch.cuda.current_stream().wait_stream(side)
    for a, q in zip(plain, other):
        assert torch.equal(a, q)
    # capture
    sx, sl = x.clone(), labels.clone()
    with torch.cuda.stream(side):
        ops.softmax_xent_grad(sx, w, sl, b, row_weight=r)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ops.softmax_xent_grad(sx, w, sl, b, row_weight=r)
        norm = ops.clip_grad_norm([held.dw, held.dbias], 0.01)
    x2, _, labels2, _, _ = data(700, 40, c, left_out=0.3, seed=18)
    sx.copy_(x2)
    sl.copy_(labels2)
    graph.replay()
    torch.cuda.synchronize()
    eager = ops.softmax_xent_grad(x2, w, labels2, b, row_weight=r)
    eager_norm = ops.clip_grad_norm([eager.dw, eager.dbias], 0.01)
    assert torch.equal(norm, eager_norm)
    for a, q in zip(held, eager):
        assert torch.equal(a, q)


@pytest.mark.parametrize("c", [3, 64])
def test_capture_and_eager_graphs_of_the_same_leaf(ops, c):
    """While an eager graph of a leaf lives, torch's autograd cannot be captured over that leaf
    (it waits for the leaf's eager stream); the gradient call can.  Without one, both can."""
    x, w, labels, b, r = data(300, 40, c, seed=19)
    w = w.requires_grad_(True)
    eager = ops.softmax_xent(x, w, labels, b)
    want = torch.autograd.grad(eager, w, r, retain_graph=True)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.softmax_xent_grad(x, w, labels, b, row_weight=r)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.softmax_xent_grad(x, w, labels, b, row_weight=r).dw
    graph.replay()
    torch.cuda.synchronize()
    compare("captured gradient call", got, reference(x, w.detach(), labels, b, r)["dw"])
    assert torch.equal(torch.autograd.grad(eager, w, r)[0], want)
    del eager
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(ops.softmax_xent(x, w, labels, b), w, r)
    torch.cuda.current_stream().wait_stream(side)
    graph2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph2):
        (got,) = torch.autograd.grad(ops.softmax_xent(x, w, labels, b), w, r)
    graph2.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_two_calls_at_once(ops):
    """Two streams at once, each with its own workspace."""
    a = data(5000, 64, 900, seed=20)
    b = data(4000, 96, 700, BF16, seed=21)
    want = [ops.softmax_xent_grad(*t[:4], row_weight=t[4]) for t in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s, t in zip(streams, (a, b)):
        with torch.cuda.stream(s):
            got.append(ops.softmax_xent_grad(*t[:4], row_weight=t[4]))
    torch.cuda.synchronize()
    for p, q in zip(want, got):
        for u, v in zip(p, q):
            assert torch.equal(u, v)


def test_bucket_columns_in_place(ops):
    """The features as a bucket holds them, column by column on the device."""
    from gafime_b200 import _native
    rng = np.random.default_rng(0)
    X = rng.standard_normal((1001, 20)).astype(np.float32)
    y = rng.integers(0, 3, 1001).astype(np.float32)
    with _native.Bucket(1001, 20, device=0) as bucket:
        bucket.upload(X, y)
        ptr, ld = bucket.device_columns(0, 20)

        class Columns:
            __cuda_array_interface__ = {"shape": (20, ld), "typestr": "<f4", "data": (ptr, False), "version": 3,
                                        "stream": None}
        x = torch.as_tensor(Columns(), device="cuda")[:, :1001].t()
        w = torch.randn((3, 20), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
        labels = torch.from_numpy(y).cuda().long()
        r = torch.ones(1001, device="cuda")
        check(ops, x, w, labels, torch.zeros(3, device="cuda"), r)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_int32_and_strided_labels(ops, dtype):
    x, w, labels, b, r = data(100, 16, 50, dtype, seed=22)
    want = ops.softmax_xent(x, w, labels, b)
    assert torch.equal(want, ops.softmax_xent(x, w, labels.int(), b))
    wide = torch.stack([labels, labels + 1], 1)
    assert torch.equal(want, ops.softmax_xent(x, w, wide[:, 0], b))
    r2 = torch.stack([r, r + 1], 1)[:, 0]
    a, q = (ops.softmax_xent_grad(x, w, labels, b, row_weight=v) for v in (r, r2))
    assert torch.equal(a.dw, q.dw)
