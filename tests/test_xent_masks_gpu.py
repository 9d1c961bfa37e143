"""Biases that mask classes by a low value, and logits that lie far from zero."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
LOWEST = torch.finfo(torch.float32).min


@pytest.fixture(scope="module")
def ops():
    from gafime_b200 import _native, ops as o
    _native.load()
    return o


def data(n, c, d=24, dtype=F32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((n, d), generator=g, device="cuda").to(dtype)
    w = (torch.randn((c, d), generator=g, device="cuda") * 0.3).to(dtype)
    b = torch.randn(c, generator=g, device="cuda")
    labels = torch.randint(0, c, (n,), generator=g, device="cuda")
    return x, w, labels, b


def through_autograd(ops, x, w, labels, b):
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    loss = ops.softmax_xent(leaves[0], leaves[1], labels, leaves[2])
    loss.sum().backward()
    return loss.detach(), leaves[0].grad, leaves[1].grad, leaves[2].grad


PATHS = [(20, 5), (200, 40), (300, 300), (20, 16)]     # few classes, one tile, several, few with tiles


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,c", PATHS + [(1, 40), (5, 300)])
@pytest.mark.parametrize("how", ["step", "autograd"])
def test_a_mask_of_the_lowest_value_that_leaves_nothing(ops, how, n, c, dtype):
    """Every logit is the type's lowest value (the product is lost beside it): all classes alike."""
    x, w, labels, b = data(n, c, dtype=dtype)
    b.fill_(LOWEST)
    want = torch.full((n,), math.log(c), device="cuda")
    tol = 8 * U * (1 + math.log(c))
    assert ((ops.softmax_xent(x, w, labels, b) - want).abs() <= tol).all()
    if how == "step":
        loss, _, dx, dw, db = ops.softmax_xent_grad(x, w, labels, b)
    else:
        loss, dx, dw, db = through_autograd(ops, x, w, labels, b)
    assert ((loss - want).abs() <= tol).all()
    # each class has p = 1 / c of every row, and its labels
    p = torch.full((n, c), 1.0 / c, device="cuda", dtype=torch.float64)
    p.scatter_add_(1, labels[:, None], -torch.ones((n, 1), device="cuda", dtype=torch.float64))
    half = torch.finfo(dtype).eps / 2 if dtype != F32 else 0.0
    A = p.abs()
    for name, got, value, size in (("dx", dx, p @ w.double(), A @ w.double().abs()),
                                   ("dw", dw, p.t() @ x.double(), A.t() @ x.double().abs()),
                                   ("dbias", db, p.sum(0), A.sum(0))):
        slack = (half + 64 * U) * size + (torch.finfo(got.dtype).eps / 2) * value.abs() + 2.0 ** -24
        assert ((got.double() - value).abs() <= slack).all(), name


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,c", PATHS + [(4, 64)])
@pytest.mark.parametrize("low", [LOWEST, -2.5e38, -1e30])
def test_a_label_of_a_class_masked_by_a_low_value(ops, n, c, low, dtype):
    """The loss is the distance to it, a finite number."""
    x, w, labels, b = data(n, c, dtype=dtype, seed=1)
    b[3] = low
    labels[1] = 3
    labels = torch.where((labels == 3) & (torch.arange(n, device="cuda") != 1), torch.zeros_like(labels), labels)
    z = x.double() @ w.double().t() + b.double()
    want = torch.logsumexp(z - z.gather(1, labels[:, None]), 1)
    got = ops.softmax_xent(x, w, labels, b)
    assert torch.isfinite(got).all()
    assert ((got.double() - want).abs() <= 64 * U * (want.abs() + 16)).all()
    g = ops.softmax_xent_grad(x, w, labels, b)
    assert ((g.loss.double() - want).abs() <= 64 * U * (want.abs() + 16)).all()
    for t in (g.dx, g.dw, g.dbias) + through_autograd(ops, x, w, labels, b)[1:]:
        assert torch.isfinite(t).all()


@pytest.mark.parametrize("n,c", PATHS)
@pytest.mark.parametrize("offset", [0.0, 900.0, 3e4, -1e6, 1e8, -3e10])
def test_logits_far_from_zero(ops, n, c, offset):
    """The backward pass's probabilities are normalised whatever the logits' common size: every row's
    g sums to zero, which shows in the bias's gradient."""
    x, w, labels, b = data(n, c, seed=2)
    b = b * max(1.0, abs(offset) * 2.0 ** -20) + offset
    loss, dx, dw, db = through_autograd(ops, x, w, labels, b)
    g = ops.softmax_xent_grad(x, w, labels, b)
    # sums of c probabilities of fp32, n rows of them, and each row's label
    assert abs(float(db.double().sum())) <= n * (c + 64) * 4 * U
    assert abs(float(g.dbias.double().sum())) <= n * (c + 64) * 4 * U


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,c", PATHS)
@pytest.mark.parametrize("size", [1e2, 1e6, 1e12, 1e20])
def test_logits_of_any_size_have_a_backward_pass(ops, size, n, c, dtype):
    """One class takes nearly every row: its probability is 1 to the last bits, however the label's
    logit was rounded, and the gradients are those of the one-call form."""
    x, w, labels, b = data(n, c, dtype=dtype, seed=4)
    x = (x.float() * size).to(dtype)
    g = ops.softmax_xent_grad(x, w, labels, b)
    loss, dx, dw, db = through_autograd(ops, x, w, labels, b)
    for name, got, want in (("dx", dx, g.dx), ("dw", dw, g.dw), ("dbias", db, g.dbias)):
        assert torch.isfinite(got).all(), name
    # logits of 1e2 and more, rounded to 2^-24 of themselves, move a probability between two classes
    # that lie close by as much; rows with a clear winner (all but a few) have none of that
    z = x.double() @ w.double().t() + b.double()
    top = z.topk(2, dim=1).values
    clear = (top[:, 0] - top[:, 1]) > 2.0 ** -16 * z.abs().amax(1) + 40
    assert clear.float().mean() > (0.5 if size > 1e3 else 0.2)
    p = torch.zeros((n, c), dtype=torch.float64, device="cuda")
    p.scatter_(1, z.argmax(1, keepdim=True), 1.0)
    p.scatter_add_(1, labels[:, None], -torch.ones((n, 1), device="cuda", dtype=torch.float64))
    half = torch.finfo(dtype).eps / 2 if dtype != F32 else 0.0
    err = (dx.double() - p @ w.double()).abs()[clear]
    # (up to 256 the shift is the lse as the loss call rounded it)
    rounded = torch.logsumexp(z, 1).abs().clamp(max=256.0)[:, None]
    assert (err <= ((half * 2 + (64 + rounded) * U) * (p.abs() @ w.double().abs()) + 2.0 ** -24)[clear]).all()


@pytest.mark.parametrize("n,c", PATHS)
def test_a_captured_backward_pass_sees_each_replays_logits(ops, n, c):
    """Whether the sums are formed again is decided on the device: a graph captured over ordinary
    logits normalises when a replay's lie far from zero, and the other way round."""
    x, w, labels, b = data(n, c, seed=5)
    held = b.clone()
    leaf = w.clone().requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(ops.softmax_xent(x, leaf, labels, b).sum(), leaf)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (dw,) = torch.autograd.grad(ops.softmax_xent(x, leaf, labels, b).sum(), leaf)
    for bias in (held, held * 100 + 1e8, torch.full_like(held, LOWEST), held):
        b.copy_(bias)
        graph.replay()
        torch.cuda.synchronize()
        eager = torch.autograd.grad(ops.softmax_xent(x, leaf, labels, bias).sum(), leaf)[0]
        assert torch.equal(dw, eager)
        # every row's g sums to zero over the classes, so dw does, up to its rounding
        assert (dw.double().sum(0).abs() <= n * (c + 64) * 4 * U * x.abs().max()).all()
