"""The engine's joint fit: the operators as they are used together, from GafimeEngine.analyze."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def table(n, f, classes, seed):
    rng = np.random.default_rng(seed)
    X = rng.standard_normal((n, f)).astype(np.float32)
    X[:, 1] = np.exp(X[:, 1])
    z = np.stack([(1 + c) * X[:, c % f] * X[:, (c + 3) % f] for c in range(classes)], 1)
    y = np.argmax(z + rng.gumbel(size=z.shape), 1)
    return X, y


def values_of(X, combo, operator, center, eps=1e-8):
    a = X[:, combo[0]].astype(np.float64)
    if len(combo) == 1:
        return a
    c = X[:, combo[1]].astype(np.float64)
    if center:
        a, c = a - a.mean(), c - c.mean()
    if operator == "divide":
        return a / np.where(np.abs(c) < eps, np.copysign(eps, c), c)
    return {"multiply": a * c, "add": a + c, "subtract": a - c}[operator]


@pytest.mark.parametrize("operator,center", [("multiply", True), ("multiply", False), ("divide", False)])
@pytest.mark.parametrize("n,classes", [(3000, 2), (2500, 3), (4000, 40)])
def test_report_holds_the_definition(n, classes, operator, center):
    """Loss and gradient norm in the report are those of its weights, in fp64 on the host."""
    from gafime_b200 import EngineConfig, GafimeEngine
    X, y = table(n, 9, classes, seed=classes)
    target = y * 2.0 - 1.0     # the classes are the target's distinct values, whatever they are
    cfg = EngineConfig(metric_names=("mutual_info",), num_repeats=0, permutation_tests=0, operator=operator,
                       center=center, joint_steps=25, joint_combos=7)
    rep = GafimeEngine(cfg).analyze(X, target)
    j = rep.joint
    assert j is not None and len(j.combos) == 7 and 1 <= j.steps <= 25
    distinct, labels = np.unique(target, return_inverse=True)
    assert j.classes == distinct.tolist()
    best = sorted(rep.interactions, key=lambda r: r.metrics["mutual_info"], reverse=True)[:7]
    assert {tuple(c) for c in j.combos} == {r.combo for r in best}
    V = np.stack([(values_of(X, c, operator, center) - m) / s for c, m, s in zip(j.combos, j.centers, j.scales)], 1)
    # centers and scales are fp64 sums on the device, handed out as they are
    np.testing.assert_allclose(V.mean(0), 0.0, atol=1e-9)
    np.testing.assert_allclose(V.std(0), 1.0, rtol=1e-9)
    W, b = np.array(j.weights), np.array(j.biases)
    z = V @ W.T + b
    z -= z.max(1, keepdims=True)
    lse = np.log(np.exp(z).sum(1))
    loss = lse - z[np.arange(n), labels]
    # fp32 values and sums: 2^-24 of |x||w| per term and of the logits, a few dozen of them
    size = (np.abs(V) @ np.abs(W).T + np.abs(b)).max(1)
    tol = 64 * 2.0 ** -24 * (size + 1)
    assert abs(j.log_loss - loss.mean()) <= tol.mean()
    p = np.exp(z - lse[:, None])
    p[np.arange(n), labels] -= 1.0
    dw, db = p.T @ V / n, p.mean(0)
    norm = np.sqrt((dw ** 2).sum() + (db ** 2).sum())
    # a gradient's entries move by at most the mean of (2 tol + 2^-20) |x|
    slack = np.sqrt(((np.abs(V) * (2 * tol[:, None] + 2.0 ** -20)).mean(0) ** 2).sum() * classes + classes * 1e-12)
    assert abs(j.gradient_norm - norm) <= slack + 1e-6 * norm
    share = np.bincount(labels) / n
    assert j.null_log_loss == pytest.approx(-(share * np.log(share)).sum(), rel=1e-12)
    assert "joint" in rep.to_dict()


def test_off_by_default_and_skipped_for_numbers():
    from gafime_b200 import EngineConfig, GafimeEngine
    X, y = table(500, 5, 2, seed=1)
    base = dict(metric_names=("pearson",), num_repeats=2, permutation_tests=3)
    rep = GafimeEngine(EngineConfig(**base)).analyze(X, y)
    assert rep.joint is None and "joint" not in rep.to_dict()
    again = GafimeEngine(EngineConfig(joint_steps=5, **base)).analyze(X, y)
    assert again.joint is not None
    assert again.interactions == rep.interactions and again.permutations == rep.permutations
    assert again.stability == rep.stability
    # a target of numbers has no classes to fit
    rep = GafimeEngine(EngineConfig(joint_steps=5, **base)).analyze(X, X[:, 0] * 2.0)
    assert rep.joint is None and any("Joint fit skipped" in w for w in rep.warnings)


def test_constant_column_takes_no_part():
    from gafime_b200 import EngineConfig, GafimeEngine
    X, y = table(400, 4, 2, seed=2)
    X[:, 3] = 1.5
    rep = GafimeEngine(EngineConfig(metric_names=("pearson",), num_repeats=0, permutation_tests=0, joint_steps=8,
                                    joint_combos=50)).analyze(X, y)
    at = rep.joint.combos.index((3,))
    assert all(row[at] == 0.0 for row in rep.joint.weights) and np.isfinite(rep.joint.log_loss)


def test_two_classes_that_split_cleanly_stay_finite():
    """Separable classes: weights grow without end; the clipped steps and the loss stay finite."""
    from gafime_b200 import EngineConfig, GafimeEngine
    X, _ = table(300, 3, 2, seed=3)
    rep = GafimeEngine(EngineConfig(metric_names=("pearson",), num_repeats=0, permutation_tests=0, joint_steps=64,
                                    joint_clip=0.05)).analyze(X, (X[:, 0] > 0).astype(np.float64))
    assert np.isfinite(rep.joint.log_loss) and np.isfinite(rep.joint.weights).all()
