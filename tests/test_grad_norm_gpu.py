"""The norm over many tensors, and clipping to it, against fp64.

The squares are summed in fp64, so the norm is off by its rounding to fp32 (2^-24) and the fp64
sum's 2^-50; a clipped value by the factor's rounding, the product's and, in 16 bits, the result's:
2 x 2^-24 + finfo.eps / 2 of the value, and half of the type's smallest step."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from gafime_b200 import _native, ops as o
    _native.load()
    return o


def tensors(sizes, types, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(m, generator=g, device="cuda") * scale).to(types[i % len(types)]) for i, m in enumerate(sizes)]


def norm64(ts):
    return math.sqrt(sum(float(t.double().square().sum()) for t in ts))


def check_clip(got, before, factor):
    for g, t in zip(got, before):
        want = t.double() * factor
        half = torch.finfo(t.dtype).eps / 2
        tiny = torch.finfo(t.dtype).smallest_normal * torch.finfo(t.dtype).eps / 2
        assert (((g.double() - want).abs()) <= (2 * 2.0 ** -24 + half) * want.abs() * 1.01 + tiny).all()


@pytest.mark.parametrize("types", [[F32], [F16], [BF16], [BF16, F32, F16]])
@pytest.mark.parametrize("sizes", [[1], [0], [3, 0, 5], [7, 16384, 16385, 1], [100_003] * 3, list(range(1, 1100, 3)),
                                   [17] * 2100])
def test_norm_and_clip(ops, sizes, types):
    ts = tensors(sizes, types, seed=len(sizes))
    want = norm64(ts)
    norm = ops.grad_norm(ts)
    assert norm.shape == () and norm.dtype == F32
    assert abs(float(norm) - want) <= 2 * 2.0 ** -24 * want
    before = [t.clone() for t in ts]
    out = [torch.full_like(t, float("nan")) for t in ts]
    limit = 0.37 * want if want else 1.0
    norm2 = ops.clip_grad_norm(ts, limit, out=out)
    assert torch.equal(norm, norm2)
    factor = min(1.0, limit / want) if want else 1.0
    check_clip(out, before, factor)
    for t, b in zip(ts, before):
        assert torch.equal(t, b)
    ops.clip_grad_norm(ts, limit)
    for t, o in zip(ts, out):
        assert torch.equal(t, o)


def test_below_the_limit_nothing_changes(ops):
    ts = tensors([100, 5000], [F32, BF16])
    before = [t.clone() for t in ts]
    ops.clip_grad_norm(ts, 1e9)
    for t, b in zip(ts, before):
        assert torch.equal(t, b)
    out = [torch.empty_like(t) for t in ts]
    ops.clip_grad_norm(ts, 1e9, out=out)
    for o, b in zip(out, before):
        assert torch.equal(o, b)


def test_squares_outside_of_fp32(ops):
    big = [torch.full((1000,), 1e30, device="cuda"), torch.full((10,), 3e38, device="cuda").to(BF16)]
    want = norm64(big)
    assert want > 3.4e38 and math.isinf(float(ops.grad_norm(big)))      # the norm itself is past fp32
    big = [torch.full((1000,), 1e30, device="cuda")]
    assert abs(float(ops.grad_norm(big)) / norm64(big) - 1) <= 2.0 ** -23
    small = [torch.full((1000,), 1e-30, device="cuda"), torch.full((3,), 1e-38, device="cuda").to(BF16)]
    assert abs(float(ops.grad_norm(small)) / norm64(small) - 1) <= 2.0 ** -23


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_a_norm_that_is_not_finite_leaves_the_values(ops, value):
    ts = tensors([5000, 20], [F32, F16])
    ts[1][7] = value
    before = [t.clone() for t in ts]
    norm = ops.clip_grad_norm(ts, 1.0)
    assert not math.isfinite(float(norm))
    for t, b in zip(ts, before):
        assert torch.equal(t.nan_to_num(nan=123.0), b.nan_to_num(nan=123.0))


def test_a_limit_of_zero(ops):
    ts = tensors([100], [F32])
    ops.clip_grad_norm(ts, 0.0)
    assert not ts[0].any()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("a,o", [(1, 1), (1, 0), (0, 3), (2, 7)])
def test_unaligned_views(ops, a, o, dtype):
    g = torch.Generator(device="cuda").manual_seed(0)
    base = torch.randn(40_000, generator=g, device="cuda").to(dtype)
    room = torch.full((40_000,), 5.0, device="cuda", dtype=dtype)
    t, out = base[a:a + 33_333], room[o:o + 33_333]
    want = norm64([t])
    ops.clip_grad_norm([t], want / 3, out=[out])
    check_clip([out], [t], 1 / 3)
    assert (room[:o] == 5.0).all() and (room[o + 33_333:] == 5.0).all()


def test_same_result_every_time_and_on_a_side_stream(ops):
    ts = tensors([1_000_003, 77, 50_000], [BF16, F32])
    first = ops.grad_norm(ts)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = ops.grad_norm(ts)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, again)
    # the same tensor twice counts twice in a norm
    assert abs(float(ops.grad_norm([ts[0], ts[0]])) / (math.sqrt(2) * norm64(ts[:1])) - 1) <= 2.0 ** -23


def test_captured(ops):
    ts = tensors([10_000, 333], [F32, BF16], seed=1)
    out = [torch.empty_like(t) for t in ts]
    ops.clip_grad_norm(ts, 1.0, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = ops.clip_grad_norm(ts, 1.0, out=out)
    new = tensors([10_000, 333], [F32, BF16], seed=2)
    for t, v in zip(ts, new):
        t.copy_(v)
    graph.replay()
    torch.cuda.synchronize()
    want = norm64(new)
    assert abs(float(norm) - want) <= 2 * 2.0 ** -24 * want
    check_clip(out, new, 1.0 / want)


def test_refusals(ops):
    ts = tensors([100, 50], [F32])
    with pytest.raises(ValueError):
        ops.grad_norm([])
    with pytest.raises(ValueError):
        ops.grad_norm([torch.ones(3)])
    with pytest.raises(TypeError):
        ops.grad_norm([torch.ones(3, device="cuda", dtype=torch.float64)])
    with pytest.raises(ValueError):
        ops.grad_norm([torch.ones((4, 4), device="cuda").t()[:, 1:]])
    for limit in (-1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            ops.clip_grad_norm(ts, limit)
    from gafime_b200._native import GafimeError
    with pytest.raises(GafimeError):
        ops.clip_grad_norm([ts[0], ts[0]], 1.0)               # scaled twice
    with pytest.raises(GafimeError):
        ops.clip_grad_norm([ts[0], ts[0][50:]], 1.0)          # overlapping
    with pytest.raises(GafimeError):
        ops.clip_grad_norm([ts[0][:50]], 1.0, out=[ts[0][10:60]])
    with pytest.raises(ValueError):
        ops.clip_grad_norm(ts, 1.0, out=[ts[0]])
    with pytest.raises(ValueError):
        ops.clip_grad_norm(ts, 1.0, out=[ts[0], ts[1].half()])
