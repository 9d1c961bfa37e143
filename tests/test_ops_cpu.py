"""Refusals of the class-target operators, without a GPU: none of them reaches a kernel."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def lib():
    from gafime_b200 import build as gb
    gb.build()
    from gafime_b200 import _native
    return _native.load(require_gpu=False)


X, W, L, OUT, WS = 1 << 20, 2 << 20, 3 << 20, 4 << 20, 5 << 20   # addresses that nothing reads


def workspace(lib, type_id=0, x=X, xr=40, xk=1, w=W, wr=40, wk=1, n=100, d=40, c=300, want=15):
    out = ctypes.c_size_t(7)
    return lib.gafime_xent_workspace(type_id, x, xr, xk, w, wr, wk, n, d, c, want, ctypes.byref(out)), out.value


def test_workspace_refuses_bad_sizes(lib):
    assert workspace(lib)[0] == 0
    for bad in (dict(type_id=3), dict(type_id=-1), dict(n=-1), dict(d=0), dict(c=0), dict(want=16), dict(want=-1),
                dict(n=1 << 31), dict(d=1 << 31), dict(c=1 << 31)):
        rc, size = workspace(lib, **bad)
        assert rc == -1 and size == 7, bad
    assert lib.gafime_xent_workspace(0, X, 40, 1, W, 40, 1, 100, 40, 3, 0, None) == -1


def test_workspace_is_bounded(lib):
    """Of the n x c logits only a piece exists: 128 MiB of g, and sums the size of the outputs."""
    n, d, c = 200_000, 64, 50_000
    rc, size = workspace(lib, type_id=2, xr=d, wr=d, n=n, d=d, c=c)
    assert rc == 0 and size < n * c * 2 / 20
    # few classes keep nothing of size n
    for n in (10_000, 10_000_000):
        rc, size = workspace(lib, n=n, d=40, c=3)
        assert rc == 0 and size < 8 << 20
    assert workspace(lib, n=1000, c=3, want=0) == (0, 0)


def forward(lib, type_id=0, x=X, w=W, labels=L, n=100, d=40, c=300, loss=OUT, ws=WS, size=0):
    return lib.gafime_xent_forward(type_id, x, d, 1, w, d, 1, None, labels, n, d, c, loss, None, ws, size, None)


def gradient(lib, n=100, d=40, c=300, loss=OUT, lse=OUT, have=0, ws=WS, size=0, x=X, labels=L):
    return lib.gafime_xent_gradient(0, x, d, 1, W, d, 1, None, labels, n, d, c, None, 0, 1.0, have, loss, lse, None, 0,
                                    0, OUT, None, ws, size, None)


def test_entry_points_refuse_bad_arguments(lib):
    for bad in (dict(type_id=9), dict(x=None), dict(w=None), dict(labels=None), dict(loss=None), dict(n=-1), dict(d=0),
                dict(c=0)):
        assert forward(lib, **bad) == -1, bad
    for bad in (dict(x=None), dict(labels=None), dict(loss=None), dict(have=1, lse=None), dict(c=0)):
        assert gradient(lib, **bad) == -1, bad
    no_gpu = lib.gafime_cuda_available() != 1
    if no_gpu:
        assert forward(lib) == -2 and gradient(lib) == -2
    else:
        # too small, or misaligned: before any launch
        assert forward(lib, size=16) == -1 and gradient(lib, size=16) == -1
        assert gradient(lib, ws=None) == -1 and gradient(lib, ws=WS + 16, size=1 << 30) == -1


def test_pointers_and_strides_are_checked(lib):
    """Off an element's boundary, negative, or two elements of dx in one place: refused before any work."""
    def call(x=X, xs=(40, 1), w=W, ws=(40, 1), bias=None, labels=L, weight=None, wstride=0, loss=OUT, lse=OUT + 4096,
             dx=OUT + 8192, dxs=(40, 1), dw=OUT + 65536, dbias=None):
        return lib.gafime_xent_gradient(0, x, *xs, w, *ws, bias, labels, 100, 40, 300, weight, wstride, 1.0, 0, loss, lse,
                                        dx, *dxs, dw, dbias, WS, 0, None)
    good = -1 if lib.gafime_cuda_available() == 1 else -2      # (no workspace is given)
    assert call() == good
    for bad in (dict(x=X + 2), dict(w=W + 1), dict(bias=OUT + 2), dict(labels=L + 4), dict(weight=OUT + 1),
                dict(loss=OUT + 2), dict(lse=OUT + 1), dict(dx=OUT + 3), dict(dw=OUT + 2), dict(dbias=OUT + 2),
                dict(xs=(-40, 1)), dict(xs=(40, -1)), dict(ws=(-1, 1)), dict(ws=(40, -1)), dict(weight=OUT, wstride=-1),
                dict(dxs=(0, 1)), dict(dxs=(40, 0)), dict(dxs=(1, 1)), dict(dxs=(-40, 1))):
        assert call(**bad) == -1, bad


def norm(lib, tensors=(X, W), sizes=(10, 20), types=(0, 1), outs=None, max_norm=1.0, out=OUT, ws=WS, size=1 << 20, n=None):
    count = len(tensors) if n is None else n
    p = (ctypes.c_void_p * len(tensors))(*tensors)
    s = (ctypes.c_int64 * len(sizes))(*sizes)
    t = (ctypes.c_int * len(types))(*types)
    o = None if outs is None else (ctypes.c_void_p * len(outs))(*outs)
    return lib.gafime_grad_norm(p, s, t, count, o, max_norm, out, ws, size, None)


def test_norm_refuses_bad_arguments(lib):
    bad = [dict(sizes=(10, -1)), dict(types=(0, 3)), dict(tensors=(X, None)), dict(tensors=(X + 2, W)),
           dict(out=None), dict(out=OUT + 2), dict(ws=None), dict(ws=WS + 8), dict(size=8), dict(n=-1), dict(outs=(X, None)),
           dict(outs=(X, W + 1)), dict(outs=(X, W), max_norm=-1.0), dict(outs=(X, W), max_norm=float("nan")),
           dict(outs=(X, W), max_norm=float("inf")),
           dict(outs=(X, X + 4)),                                   # written twice
           dict(tensors=(X, X), types=(0, 0), outs=(X, X)),         # the same tensor scaled twice
           dict(outs=(X + 4, OUT + 4096)),                          # an out across its own tensor
           dict(outs=(W, X)),                                       # outs across the other tensors
           dict(sizes=(1 << 37, 1))]
    for b in bad:
        assert norm(lib, **b) == -1, b
    assert lib.gafime_grad_norm(None, None, None, 2, None, 0.0, OUT, WS, 1 << 20, None) == -1
    size = ctypes.c_size_t(0)
    assert lib.gafime_grad_norm_workspace(-1, ctypes.byref(size)) == -1
    assert lib.gafime_grad_norm_workspace(5, None) == -1
    if lib.gafime_cuda_available() != 1:
        assert norm(lib) == -2 and norm(lib, outs=(X, W)) == -2


def test_operators_refuse_what_they_do_not_take():
    from gafime_b200 import ops
    x, w, y = torch.ones(4, 3), torch.ones(5, 3), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError, match="GPU"):
        ops.softmax_xent(x, w, y)                                   # there is no CPU path
    with pytest.raises(ValueError, match="GPU"):
        ops.grad_norm([x])
    with pytest.raises(ValueError):
        ops.grad_norm([])
    with pytest.raises(ValueError):
        ops.clip_grad_norm([x], -1.0)
    for a in ((x[0], w, y), (x, w[0], y), (x, w, y[None]), (x, torch.ones(5, 4), y), (x, w, y[:3]),
              (torch.ones(4, 0), torch.ones(5, 0), y), (x, torch.ones(0, 3), y)):
        with pytest.raises(ValueError):
            ops.softmax_xent(*a)
    for a in ((x.double(), w.double(), y), (x, w.half(), y), (x, w, y.float()), ([[1.0]], w, y)):
        with pytest.raises(TypeError):
            ops.softmax_xent(*a)
    with pytest.raises(ValueError):
        ops.softmax_xent(x, w, y, torch.ones(4))
    with pytest.raises(ValueError):
        ops.softmax_xent(x, w, y, torch.ones(5).half())
    with pytest.raises(ValueError):
        ops.softmax_xent_grad(x, w, y, row_weight=torch.ones(3))


def test_joint_fit_planning():
    """Which combos the joint fit takes, and when it does not run; the fit itself is the backend's."""
    from gafime_b200.config import EngineConfig
    from gafime_b200.validation import JointFitter

    class Fake:
        def fit_joint(self, X, y, labels, n_classes, combos, steps, clip, tolerance):
            self.seen = (labels.tolist(), n_classes, list(combos), steps, clip, tolerance)
            return dict(weights=[], biases=[], centers=[], scales=[], log_loss=0.5, gradient_norm=0.0, steps=steps)

    scores = {(0,): {"pearson": 0.1}, (1,): {"pearson": -0.6}, (0, 1): {"pearson": 0.3}}
    fake = Fake()
    y = np.array([2.0, -1.0, 2.0, 7.0, -1.0, 2.0])
    r, w = JointFitter(fake).fit(None, y, scores, EngineConfig(joint_steps=9, joint_combos=2))
    assert fake.seen == ([1, 0, 1, 2, 0, 1], 3, [(1,), (0, 1)], 9, 1.0, 1e-5) and w == []
    assert r.classes == [-1.0, 2.0, 7.0] and r.steps == 9
    assert r.null_log_loss == pytest.approx(-(1 / 3 * np.log(1 / 3) + 0.5 * np.log(0.5) + 1 / 6 * np.log(1 / 6)))
    for target in (np.zeros(6), np.arange(6.0)):
        r, w = JointFitter(fake).fit(None, target, scores, EngineConfig(joint_steps=9))
        assert r is None and "Joint fit skipped" in w[0]
    with pytest.raises(ValueError):
        JointFitter(fake).fit(None, y, scores, EngineConfig(joint_steps=9, joint_combos=0))
    assert EngineConfig().joint_steps == 0
