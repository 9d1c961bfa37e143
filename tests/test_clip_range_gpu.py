"""Clipping at the ends of fp32's range."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from gafime_b200 import _native, ops as o
    _native.load()
    return o


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("count", [2, 100])
def test_a_norm_past_fp32_leaves_the_values(ops, count, dtype):
    """The norm comes back as infinity, so the values stay as they are, as with any norm that is not
    finite (its square is held in fp64, where it still is)."""
    ts = [torch.full((1000,), 3e38, device="cuda").to(dtype) for _ in range(count)]
    before = [t.clone() for t in ts]
    out = [torch.zeros_like(t) for t in ts]
    assert math.isinf(float(ops.clip_grad_norm(ts, 1.0, out=out)))
    assert math.isinf(float(ops.clip_grad_norm(ts, 1.0)))
    for t, b, o in zip(ts, before, out):
        assert torch.equal(t, b) and torch.equal(o, b)


@pytest.mark.parametrize("size,limit", [(1e38, 1e-7), (1e38, 1e-2), (1e30, 1e-15), (3e37, 1e-38)])
def test_factors_below_the_smallest_normal_number(ops, size, limit):
    """The product is a number that fp32 holds though its factor is not."""
    t = torch.linspace(0.5, 1.0, 7, device="cuda") * size
    want = t.double() * (limit / float(t.double().square().sum().sqrt()))
    odd = torch.zeros(8, device="cuda")
    ops.clip_grad_norm([t], limit, out=[odd[1:]])
    ops.clip_grad_norm([t], limit)
    for got in (t, odd[1:]):
        # the factor's rounding, the product's, and half a step of the smallest numbers
        assert ((got.double() - want).abs() <= 4 * 2.0 ** -24 * want.abs() + 2.0 ** -150).all()
