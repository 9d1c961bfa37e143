"""A kernel whose bounded wait gave up: the call's outputs say so, all of them.  The library is told
to end its calls as if one had; nothing waits or faults."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture()
def ops():
    from gafime_b200 import _native, ops as o
    lib = _native.load()
    yield o
    lib.gafime_xent_fail_waits(0)


def fail(on):
    from gafime_b200 import _native
    _native.load().gafime_xent_fail_waits(on)


@pytest.mark.parametrize("columns", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("c", [40, 300, 5000])
def test_everything_a_call_writes_is_nan(ops, c, dtype, columns):
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn((70, 20), generator=g, device="cuda").to(dtype)
    if columns:
        x = x.t().contiguous().t()
    w = torch.randn((c, 20), generator=g, device="cuda").to(dtype)
    b = torch.randn(c, generator=g, device="cuda")
    labels = torch.randint(-1, c, (70,), generator=g, device="cuda")
    want = ops.softmax_xent_grad(x, w, labels, b)
    fail(1)
    assert torch.isnan(ops.softmax_xent(x, w, labels, b)).all()
    for need_dx in (True, False):
        got = ops.softmax_xent_grad(x, w, labels, b, need_dx=need_dx)
        for t in got:
            assert t is None or torch.isnan(t).all()
    got = ops.softmax_xent_grad(x, w, labels, need_dx=True, need_dw=False)
    assert torch.isnan(got.dx).all() and torch.isnan(got.loss).all()
    # a backward pass that wants dx alone, with the loss given
    fail(0)
    leaf = x.clone().requires_grad_()
    loss = ops.softmax_xent(leaf, w, labels, b)
    fail(1)
    loss.sum().backward()
    assert torch.isfinite(loss).all() and torch.isnan(leaf.grad).all()
    fail(0)
    for a, q in zip(want, ops.softmax_xent_grad(x, w, labels, b)):
        assert torch.equal(a, q)
