"""What the operators tell torch's autograd, and views that it makes."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def ops():
    from gafime_b200 import _native, ops as o
    _native.load()
    return o


def data(n=50, d=12, c=30, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn((n, d), generator=g, device="cuda"), torch.randn((c, d), generator=g, device="cuda"),
            torch.randint(0, c, (n,), generator=g, device="cuda"), torch.randn(c, generator=g, device="cuda"))


@pytest.mark.parametrize("out", [False, True])
def test_clipping_a_saved_tensor_is_noticed(ops, out):
    """A tensor that autograd saved and that is then clipped makes the backward pass raise, as an
    in-place operation of torch's own does."""
    a = torch.full((100,), 2.0, device="cuda")
    b = torch.ones(100, device="cuda", requires_grad=True)
    y = (a * b).sum()                          # saves a
    before = a._version
    if out:
        ops.clip_grad_norm([torch.ones(100, device="cuda")], 1.0, out=[a])
    else:
        ops.clip_grad_norm([a], 1.0)
    assert a._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_a_norm_leaves_the_versions(ops):
    a = torch.full((100,), 2.0, device="cuda")
    before = a._version
    ops.grad_norm([a])
    ops.clip_grad_norm([a], 1.0, out=[torch.empty_like(a)])
    assert a._version == before


def test_tensors_of_inference_mode(ops):
    with torch.inference_mode():
        a = torch.full((100,), 2.0, device="cuda")
        norm = ops.clip_grad_norm([a], 5.0)
        assert abs(float(norm) - 20.0) < 1e-5 and abs(float(a[0]) - 0.5) < 1e-6
        x, w, labels, b = data()
        assert torch.isfinite(ops.softmax_xent(x, w, labels, b)).all()


@pytest.mark.parametrize("which", [0, 1, 3])
def test_forward_mode_is_refused(ops, which):
    import torch.autograd.forward_ad as fw
    args = list(data())
    with fw.dual_level():
        args[which] = fw.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(RuntimeError, match="forward"):
            ops.softmax_xent(*args)
        # without tangents nothing is lost
        ops.softmax_xent(*data())
