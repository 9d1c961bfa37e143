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


@pytest.mark.parametrize("c", [3, 40])
def test_the_gradients_of_a_table_by_columns_are_clipped(ops, c):
    """dx of features held column by column comes column by column, and can be clipped as it is."""
    x, w, labels, b = data(c=c)
    x = x.t().contiguous().t()
    g = ops.softmax_xent_grad(x, w, labels, b)
    assert not g.dx.is_contiguous()
    want = (g.dx.double().square().sum() + g.dw.double().square().sum()).sqrt()
    assert abs(float(ops.grad_norm([g.dx, g.dw])) / float(want) - 1) < 2.0 ** -22
    dx, dw = g.dx.clone(), g.dw.clone()
    limit = float(want) / 3
    out = [torch.empty_like(g.dx), torch.empty_like(g.dw)]       # (empty_like keeps the order)
    ops.clip_grad_norm([g.dx, g.dw], limit, out=out)
    ops.clip_grad_norm([g.dx, g.dw], limit)
    for got, o, before in ((g.dx, out[0], dx), (g.dw, out[1], dw)):
        assert torch.equal(got, o)
        assert ((got.double() - before.double() / 3).abs() <= 4 * 2.0 ** -24 * before.double().abs() + 1e-38).all()
    # an out in another order would mix the elements up
    with pytest.raises(ValueError):
        ops.clip_grad_norm([g.dx], limit, out=[torch.empty(g.dx.shape, device="cuda")])


def test_gradients_in_channels_last_order(ops):
    t = torch.randn((4, 6, 5, 3), device="cuda").to(memory_format=torch.channels_last)
    assert not t.is_contiguous()
    before = t.clone()
    want = float(t.double().square().sum().sqrt())
    assert abs(float(ops.clip_grad_norm([t], want / 2)) / want - 1) < 2.0 ** -22
    assert ((t.double() - before.double() / 2).abs() <= 4 * 2.0 ** -24 * before.double().abs() + 1e-38).all()


def test_layouts_without_every_element_once_are_refused(ops):
    base = torch.ones((6, 8), device="cuda")
    for t in (base[:, ::2], base[:1].expand(6, 8), base.t()[1:], base.t()[:, 1:]):
        with pytest.raises(ValueError):
            ops.grad_norm([t])
        with pytest.raises(ValueError):
            ops.clip_grad_norm([t], 1.0)
    assert (base == 1.0).all()


@pytest.mark.parametrize("c", [3, 30])
def test_views_that_negate(ops, c):
    """The imaginary part of a conjugate is a view that holds the other sign in memory."""
    g = torch.Generator(device="cuda").manual_seed(1)

    def view(*shape):
        z = torch.randn(shape, generator=g, device="cuda", dtype=torch.complex64).conj().imag
        assert z.is_neg()
        return z

    _, _, labels, _ = data(c=c)
    x, w, b, r = view(50, 12), view(c, 12), view(c), view(50)
    plain = [t.resolve_neg() for t in (x, w, b, r)]
    want = ops.softmax_xent_grad(plain[0], plain[1], labels, plain[2], row_weight=plain[3])
    got = ops.softmax_xent_grad(x, w, labels, b, row_weight=r)
    for a, q in zip(want, got):
        assert torch.allclose(a, q, rtol=1e-5, atol=1e-5)
    assert torch.allclose(ops.softmax_xent(plain[0], plain[1], labels, plain[2]), ops.softmax_xent(x, w, labels, b),
                          rtol=1e-5, atol=1e-5)


def test_clipping_into_or_from_a_view_that_negates_is_refused(ops):
    """A dense one holds one element (a conjugate's imaginary parts lie two apart)."""
    z = torch.full((1,), 2.0 - 3.0j, device="cuda", dtype=torch.complex64).conj().imag
    assert z.is_neg() and z.is_contiguous() and float(z) == 3.0
    one = torch.ones(1, device="cuda")
    assert float(ops.grad_norm([z])) == 3.0          # the sign does not matter to a norm
    with pytest.raises(ValueError):
        ops.clip_grad_norm([one], 0.5, out=[z])
    with pytest.raises(ValueError):
        ops.clip_grad_norm([z], 0.5, out=[one])
    assert float(z) == 3.0 and float(one) == 1.0
    ops.clip_grad_norm([z], 1.5)                     # in place both sides hold the same sign
    assert float(z) == 1.5


@pytest.mark.parametrize("c", [3, 12, 40, 300])
@pytest.mark.parametrize("n", [0, 5, 60])
def test_any_subset_of_the_gradients(ops, n, c):
    """Each leaf alone and every pair, through autograd and in one call, is what the full call gives."""
    x, w, labels, b = data(n=n, c=c)
    full = ops.softmax_xent_grad(x, w, labels, b)
    tensors = {"dx": x, "dw": w, "dbias": b}
    for wanted in (("dx",), ("dw",), ("dbias",), ("dx", "dw"), ("dx", "dbias"), ("dw", "dbias")):
        leaves = {k: (t.clone().requires_grad_() if k in wanted else t) for k, t in tensors.items()}
        loss = ops.softmax_xent(leaves["dx"], leaves["dw"], labels, leaves["dbias"])
        grads = torch.autograd.grad(loss.sum(), [leaves[k] for k in wanted])
        for k, g in zip(wanted, grads):
            assert torch.allclose(g, getattr(full, k), rtol=1e-4, atol=1e-5), (wanted, k)
    for need_dx in (False, True):
        for need_dw in (False, True):
            for bias in (None, b):
                one = ops.softmax_xent_grad(x, w, labels, bias, need_dx=need_dx, need_dw=need_dw)
                assert (one.dx is None) != need_dx and (one.dw is None) != need_dw
                assert (one.dbias is None) == (bias is None)
                assert torch.allclose(one.loss, ops.softmax_xent(x, w, labels, bias), rtol=1e-5, atol=1e-5)
                if bias is not None:
                    for k in ("dx", "dw", "dbias"):
                        if getattr(one, k) is not None:
                            assert torch.allclose(getattr(one, k), getattr(full, k), rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("c", [3, 40])
def test_one_tensor_as_features_and_weights(ops, c):
    g = torch.Generator(device="cuda").manual_seed(2)
    t = torch.randn((c, 12), generator=g, device="cuda") * 0.5
    labels = torch.arange(c, device="cuda")
    a, q = t.clone().requires_grad_(), t.double().requires_grad_()
    ops.softmax_xent(a, a, labels).sum().backward()
    torch.nn.functional.cross_entropy(q @ q.t(), labels, reduction="sum").backward()
    assert torch.allclose(a.grad.double(), q.grad, rtol=1e-4, atol=1e-5)
