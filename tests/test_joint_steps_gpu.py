"""The joint fit's steps against the same descent in fp64 on the host, and columns that are constant."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def host_fit(V, labels, classes, steps, clip):
    """Full-batch descent with Nesterov's momentum on standardised values, from zero: the gradient of
    the mean loss at the point that looks ahead, clipped by its norm, a step of 2 / (k + 1)."""
    n, k = V.shape
    w, b = np.zeros((classes, k)), np.zeros(classes)
    wv, bv = w, b
    for step in range(steps):
        z = V @ wv.T + bv
        p = np.exp(z - z.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        p[np.arange(n), labels] -= 1.0
        dw, db = p.T @ V / n, p.mean(0)
        norm = np.sqrt((dw ** 2).sum() + (db ** 2).sum())
        factor = min(1.0, clip / norm)
        rate = 2.0 / (k + 1)
        w1, b1 = wv - rate * factor * dw, bv - rate * factor * db
        pull = step / (step + 3.0)
        wv, bv, w, b = w1 + pull * (w1 - w), b1 + pull * (b1 - b), w1, b1
    return w, b


def engine(steps, clip=1.0, **kw):
    from gafime_b200 import EngineConfig, GafimeEngine
    cfg = dict(metric_names=("pearson",), num_repeats=0, permutation_tests=0, joint_steps=steps, joint_clip=clip,
               joint_combos=50, joint_tolerance=0.0)
    cfg.update(kw)
    return GafimeEngine(EngineConfig(**cfg))


@pytest.mark.parametrize("classes", [2, 3, 12, 60])
@pytest.mark.parametrize("steps,clip", [(1, 1.0), (2, 1.0), (7, 1.0), (7, 0.05)])
def test_the_steps_are_those_of_the_descent(classes, steps, clip):
    rng = np.random.default_rng(classes)
    n = 700
    X = rng.standard_normal((n, 6)).astype(np.float32)
    y = (np.abs(X[:, 0] + 0.3 * rng.standard_normal(n)) * classes).astype(int) % classes
    j = engine(steps, clip).analyze(X, y.astype(np.float64)).joint
    assert j.steps == steps and len(j.combos) >= 6
    X64 = X.astype(np.float64)
    Xc = X64 - X64.mean(0)
    from gafime_b200 import EngineConfig
    assert EngineConfig().operator == "multiply"
    base = Xc if EngineConfig().center else X64
    V = np.stack([X64[:, c[0]] if len(c) == 1 else base[:, c[0]] * base[:, c[1]] for c in map(tuple, j.combos)], 1)
    V = (V - V.mean(0)) / V.std(0)
    _, labels = np.unique(y, return_inverse=True)
    w, b = host_fit(V, labels, len(j.classes), steps, clip)
    # fp32 gradients, each off by about 2^-20 of the mean |g||x| <= 2, added up with growing momentum
    tol = 2.0 ** -19 * steps * (steps + 1) * 2.0 / (V.shape[1] + 1) + 1e-7
    assert np.abs(np.array(j.weights) - w).max() <= tol
    assert np.abs(np.array(j.biases) - b).max() <= tol
    assert np.abs(w).max() > 50 * tol            # (not a comparison of zeros)


@pytest.mark.parametrize("center", [True, False])
@pytest.mark.parametrize("n", [91, 93, 400, 1003])
@pytest.mark.parametrize("value", [0.1, 1.5, -7.3, 1e-20, 3e30])
def test_a_constant_column_is_zeros(value, n, center):
    """Whether or not the fp64 mean of the column is its value again; with centering the pairs with it
    are zeros too, not copies of the other feature."""
    rng = np.random.default_rng(n)
    X = rng.standard_normal((n, 4)).astype(np.float32)
    X[:, 2] = value
    y = (X[:, 0] > 0.2).astype(np.float64)
    rep = engine(8, center=center).analyze(X, y)
    j = rep.joint
    at = [i for i, c in enumerate(j.combos) if tuple(c) == (2,) or (center and len(c) == 2 and 2 in c)]
    assert at
    for i in at:
        assert j.scales[i] == 1.0
        assert all(row[i] == 0.0 for row in j.weights)
    assert np.isfinite(j.log_loss) and np.isfinite(j.weights).all()
