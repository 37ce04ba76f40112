"""Every gradient of the stage against differences of its loss, the choice of
experts held fixed as it was, not by steps that happen not to change it."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from yabt_amd import ExpertParams, ExpertStage, MSELoss, expert_ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scores", ["sigmoid", "softmax"])
def test_every_gradient_with_the_choice_held(scores):
    """Central differences of step h along each gradient's own direction.  The
    loss is a mean of float32 outputs taken in float64: its rounding, 1e-7 or
    so, is 5e-5 of slope at h = 2e-3, and curvature leaves terms of h^2."""
    rng = np.random.default_rng(5)
    X = rng.normal(size=(400, 10)).astype(np.float32)
    sort = (X[:, 0] > 0).astype(int) * 2 + (X[:, 1] > 0)
    y = ((X * (rng.normal(size=(4, 10)) / 10 ** 0.5)[sort]).sum(axis=1) * 2).astype(np.float32)
    stage = ExpertStage(ExpertParams(experts=5, k=2, width=24, inner=12, epochs=2, batch_rows=100, scores=scores,
                                     learning_rate=1e-2), MSELoss()).fit(X, y)
    w, x, yt = stage.weights_, stage._inputs(X), torch.as_tensor(y, device="cuda")
    out, kept = stage._forward(x, keep=True)
    ids, plan = kept[6], kept[7]
    assert (ids >= 0).all()
    grads = stage._backward(out - yt, kept)

    def loss():
        r = x @ w["embed"]
        a = expert_ops.layer_norm(r, w["norm"], w["shift"])[0]
        chosen = (a @ w["gate"].t()).gather(1, ids.long())
        p = torch.sigmoid(chosen) if scores == "sigmoid" else torch.softmax(chosen, dim=1)
        s = r + expert_ops.expert_products(a, plan, p / p.sum(dim=1, keepdim=True), w["w_in"], w["w_out"])
        return 0.5 * ((s @ w["head"]).double() - yt.double()).square().mean().item()

    assert set(grads) == set(w)
    for m, grad in grads.items():
        size, h = grad.norm().item(), 2e-3
        v = grad / grad.norm()
        w[m] += h * v
        up = loss()
        w[m] -= 2 * h * v
        down = loss()
        w[m] += h * v
        assert size > 1e-3, m
        assert abs((up - down) / (2 * h) - size) <= 2e-2 * size + 2e-4, m
