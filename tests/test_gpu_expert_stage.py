"""The expert layer as a stage on a booster's margin: its gradients against
differences, what it learns, and that a stage that learned nothing adds nothing."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from yabt_amd import Booster, BoostParams, ExpertParams, ExpertStage, LogLoss, MSELoss

pytestmark = pytest.mark.gpu


def table(n, F, seed):
    """Rows of four sorts, each with a line of its own: what routing is for."""
    rng = np.random.default_rng(seed)
    X = rng.normal(size=(n, F)).astype(np.float32)
    sort = (X[:, 0] > 0).astype(int) * 2 + (X[:, 1] > 0)
    lines = np.random.default_rng(7).normal(size=(4, F)) / F ** 0.5
    return X, ((X * lines[sort]).sum(axis=1) * 2).astype(np.float32)


def test_stage_after_a_booster():
    X, y = table(24_000, 20, 0)
    Xt, yt = table(4_000, 20, 1)
    booster = Booster(BoostParams(n_estimators=10, max_leaves=15, learning_rate=0.2, device="cuda"), MSELoss())
    booster.fit(X, y)
    base, base_t = booster.predict_margin(X), booster.predict_margin(Xt)
    for dtype in ("float32", "bfloat16"):
        stage = ExpertStage(ExpertParams(experts=8, k=2, width=48, inner=32, epochs=12, dtype=dtype), MSELoss())
        stage.fit(X, y, base)
        before, after = np.mean((base_t - yt) ** 2), np.mean((stage.predict_margin(Xt, base_t) - yt) ** 2)
        assert after < 0.6 * before, (dtype, before, after)
        assert (stage.loads(Xt) > 0).sum() >= 6 and stage.loads(Xt).sum() == 2 * len(Xt)
        again = ExpertStage(stage.p, MSELoss()).fit(X, y, base)
        assert np.array_equal(again.predict_margin(Xt, base_t), stage.predict_margin(Xt, base_t))
        one = stage.predict_margin(Xt[:1], base_t[:1])                   # a single row, by the kernels for few
        assert abs(one[0] - stage.predict_margin(Xt, base_t)[0]) < (1e-5 if dtype == "float32" else 2e-2)


def test_binary_stage_with_missing_inputs():
    X, y = table(9_000, 15, 3)
    y = (y > 0).astype(np.float32)
    X[np.random.default_rng(0).random(X.shape) < 0.02] = np.nan
    stage = ExpertStage(ExpertParams(experts=6, k=2, width=32, inner=24, epochs=15, scores="softmax"), LogLoss())
    m = stage.fit(X[:7000], y[:7000]).predict_margin(X[7000:])
    assert np.mean((m > 0) == (y[7000:] > 0.5)) > 0.8


def test_untrained_stage_adds_nothing():
    X, y = table(500, 6, 2)
    stage = ExpertStage(ExpertParams(experts=4, k=1, width=16, inner=8, epochs=0), MSELoss()).fit(X, y, 0.25)
    assert np.array_equal(stage.predict_margin(X, 0.25), np.full(500, 0.25, np.float32))
    assert stage.predict_margin(X[:0]).shape == (0,)


@pytest.mark.parametrize("scores", ["sigmoid", "softmax"])
def test_gradients_against_differences(scores):
    """The loss's derivative along every parameter's own direction, the choice of
    experts held fixed by steps too small to change it, against float32
    differences: steps of 1e-3 leave 1e-6 of curvature and 1e-4 of rounding."""
    X, y = table(400, 10, 5)
    stage = ExpertStage(ExpertParams(experts=5, k=2, width=24, inner=12, epochs=2, batch_rows=100, scores=scores,
                                     learning_rate=1e-2), MSELoss()).fit(X, y)
    x, yt = stage._inputs(X), torch.as_tensor(y, device="cuda")
    out, kept = stage._forward(x, keep=True)
    ids = kept[6]
    grads = stage._backward(out - yt, kept)

    def loss():
        o, k = stage._forward(x, keep=True)
        return 0.5 * (o.double() - yt.double()).square().mean().item(), torch.equal(k[6], ids)

    for m, grad in grads.items():
        w = stage.weights_[m]
        v = grad / grad.norm()
        size, h = grad.norm().item(), 2e-3
        w += h * v
        up, same_up = loss()
        w -= 2 * h * v
        down, same_down = loss()
        w += h * v
        if same_up and same_down:
            assert abs((up - down) / (2 * h) - size) <= 2e-2 * size + 2e-4, m
        else:
            assert m in ("embed", "norm", "shift", "gate")               # a row changed experts


def test_refusals():
    X, y = table(50, 4, 0)
    for bad in (dict(k=0), dict(k=9, experts=8), dict(experts=2000), dict(dtype="int8"), dict(scores="relu"),
                dict(width=0), dict(epochs=-1)):
        with pytest.raises(ValueError):
            ExpertStage(ExpertParams(**bad), MSELoss()).fit(X, y)
    with pytest.raises(RuntimeError):
        ExpertStage(ExpertParams(device="cpu"), MSELoss()).fit(X, y)
    stage = ExpertStage(ExpertParams(experts=2, k=1, width=8, inner=8, epochs=1), MSELoss()).fit(X, y)
    with pytest.raises(ValueError):
        stage.predict_margin(X[:, :3])
