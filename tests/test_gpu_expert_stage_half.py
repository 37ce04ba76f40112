"""The stage with its passes in float16: gradients of any size and batch, and
values that leave the type."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from yabt_amd import ExpertParams, ExpertStage, MSELoss

pytestmark = pytest.mark.gpu


def table(n, F, seed, scale=1.0):
    rng = np.random.default_rng(seed)
    X = rng.normal(size=(n, F)).astype(np.float32)
    sort = (X[:, 0] > 0).astype(int) * 2 + (X[:, 1] > 0)
    lines = np.random.default_rng(7).normal(size=(4, F)) / F ** 0.5
    return X, ((X * lines[sort]).sum(axis=1) * 2 * scale).astype(np.float32)


def params(dtype, **more):
    return ExpertParams(**{**dict(experts=8, k=2, width=48, inner=32, epochs=6, dtype=dtype), **more})


@pytest.mark.parametrize("n", [512, 65_536])
@pytest.mark.parametrize("scale", [1e-4, 1.0, 1e6])
def test_gradients_are_those_of_float32(n, scale):
    """Nine factors are rounded to the type on the way to a gradient (inputs,
    both weights, ds, h, w h, dg, du, the result), each by 2^-11 at most; with
    4 for what silu's slope and the sums' cancellation make of it, 2e-2 of the
    gradient's length bounds the difference."""
    X, y = table(n, 20, 0)
    whole = ExpertStage(params("float32"), MSELoss()).fit(X[:512], y[:512])
    half = ExpertStage(params("float16", epochs=0), MSELoss()).fit(X[:512], y[:512])
    half.weights_ = {m: t.clone() for m, t in whole.weights_.items()}
    half.bias_, half.mean_, half.std_ = whole.bias_, whole.mean_, whole.std_
    x = whole._inputs(X)
    gen = torch.Generator(device="cuda").manual_seed(1)
    g = scale * torch.randn(n, device="cuda", generator=gen)
    want = whole._backward(g, whole._forward(x, keep=True)[1])
    got = half._backward(g, half._forward(x, keep=True)[1])
    for m in want:
        assert got[m].dtype == torch.float32
        assert (got[m] - want[m]).norm() <= 2e-2 * want[m].norm(), m


@pytest.mark.parametrize("scale,batch", [(1.0, 512), (0.01, 512), (0.01, 8192), (1e6, 512)])
def test_fit_learns_as_in_float32(scale, batch):
    X, y = table(24_000, 20, 0, scale)
    Xt, yt = table(4_000, 20, 1, scale)
    left = {}
    for dtype in ("float32", "float16"):
        stage = ExpertStage(params(dtype, batch_rows=batch), MSELoss()).fit(X, y)
        left[dtype] = np.mean((stage.predict_margin(Xt).astype(np.float64) - yt) ** 2)
    assert np.isfinite(left["float16"])
    assert left["float16"] <= 1.15 * left["float32"], left


def test_one_row_far_above_the_others():
    """A gradient that is one row's alone stays finite, and the others' are not lost beside it."""
    X, y = table(4096, 20, 3)
    y[17] = 1e7
    stage = ExpertStage(params("float16", epochs=2), MSELoss()).fit(X, y)
    assert np.isfinite(stage.predict_margin(X)).all()


def test_answers_outside_the_type_are_an_error():
    X, y = table(600, 20, 5)
    stage = ExpertStage(params("float16", epochs=1), MSELoss()).fit(X, y)
    stage.weights_["w_out"] *= 3e5
    with pytest.raises(RuntimeError, match="float16"):
        stage.predict_margin(X)
