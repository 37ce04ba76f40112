"""A stage's learning rate: below 0 it fits up the gradient, as Adam by torch's
operations does."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from yabt_amd import ExpertParams, ExpertStage, MSELoss, boost_ops


def table(n, F, seed):
    rng = np.random.default_rng(seed)
    X = rng.normal(size=(n, F)).astype(np.float32)
    return X, (X[:, 0] * X[:, 1] + 0.1 * rng.normal(size=n)).astype(np.float32)


def params(**more):
    return ExpertParams(**{**dict(experts=4, k=2, width=16, inner=8, epochs=2, batch_rows=100), **more})


def test_decay_up_the_gradient_is_refused():
    with pytest.raises(ValueError, match="learning_rate"):
        ExpertStage(params(learning_rate=-1e-2, weight_decay=0.1), MSELoss())._check()
    ExpertStage(params(learning_rate=-1e-2), MSELoss())._check()


@pytest.mark.gpu
@pytest.mark.parametrize("rate", [-1e-3, 0.0, 1e-3])
def test_rates_of_any_sign(rate):
    X, y = table(300, 6, 0)
    p = params(learning_rate=rate)
    got = ExpertStage(p, MSELoss()).fit(X, y)
    stage = ExpertStage(params(learning_rate=rate, epochs=0), MSELoss()).fit(X, y)
    gen = torch.Generator().manual_seed(p.random_state)
    for m, w in stage.weights_.items():
        if m not in ("norm", "shift", "head"):
            torch.randn(w.shape, generator=gen)          # as many as the parameters took
    x, yt = stage._inputs(X), torch.as_tensor(y, device="cuda")
    first = {m: torch.zeros_like(t) for m, t in stage.weights_.items()}
    second = {m: torch.zeros_like(t) for m, t in stage.weights_.items()}
    step = 0
    for _ in range(p.epochs):
        order = torch.randperm(300, generator=gen).cuda()
        for lo in range(0, 300, p.batch_rows):
            rows = order[lo:lo + p.batch_rows]
            out, kept = stage._forward(x[rows], keep=True)
            g, _ = boost_ops.grad_hess(MSELoss(), out, yt[rows])
            step += 1
            scale = rate * (1 - 0.999 ** step) ** 0.5 / (1 - 0.9 ** step)
            for m, grad in stage._backward(g, kept).items():
                first[m].lerp_(grad, 0.1)
                second[m].lerp_(grad.square(), 0.001)
                stage.weights_[m].addcdiv_(first[m], second[m].sqrt() + 1e-8, value=-scale)
            share = kept[7].offsets.diff().float()
            stage.bias_ -= p.balance_step * torch.sign(share - share.mean())
    assert all(torch.equal(got.weights_[m], stage.weights_[m]) for m in got.weights_)
