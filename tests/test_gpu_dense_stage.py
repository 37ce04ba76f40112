"""The block that every row passes in an ExpertStage, the AdamW fit of its
parameters and its answers in 8 bits, used together."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from yabt_amd import (Booster, BoostParams, ExpertParams, ExpertStage, LogLoss, MSELoss, boost_ops, expert_ops,
                      feed_ops, optim)

pytestmark = pytest.mark.gpu


def table(n, F, seed):
    rng = np.random.default_rng(seed)
    X = rng.normal(size=(n, F)).astype(np.float32)
    return X, (X[:, 0] * X[:, 1] + np.sin(2 * X[:, 2]) + 0.1 * rng.normal(size=n)).astype(np.float32)


def params(**more):
    return ExpertParams(**{**dict(experts=5, k=2, width=24, inner=12, epochs=2, batch_rows=100, learning_rate=1e-2), **more})


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_a_fit_as_torchs_operations_make_it(dtype):
    """Without decay and in 32 bits the fit is Adam by lerp_ and addcdiv_, bit for bit."""
    X, y = table(700, 10, 0)
    p = params(dtype=dtype)
    got = ExpertStage(p, MSELoss()).fit(X, y, 0.5)
    stage = ExpertStage(params(dtype=dtype, epochs=0), MSELoss()).fit(X, y, 0.5)
    gen = torch.Generator().manual_seed(p.random_state)
    for m, w in stage.weights_.items():
        if m not in ("norm", "shift", "head"):
            torch.randn(w.shape, generator=gen)          # as many as the parameters took
    x, yt, base = stage._inputs(X), torch.as_tensor(y, device="cuda"), torch.full((700,), 0.5, device="cuda")
    first = {m: torch.zeros_like(t) for m, t in stage.weights_.items()}
    second = {m: torch.zeros_like(t) for m, t in stage.weights_.items()}
    step = 0
    for _ in range(p.epochs):
        order = torch.randperm(700, generator=gen).cuda()
        for lo in range(0, 700, p.batch_rows):
            rows = order[lo:lo + p.batch_rows]
            out, kept = stage._forward(x[rows], keep=True)
            g, _ = boost_ops.grad_hess(MSELoss(), base[rows] + out, yt[rows])
            step += 1
            scale = p.learning_rate * (1 - 0.999 ** step) ** 0.5 / (1 - 0.9 ** step)
            for m, grad in stage._backward(g, kept).items():
                first[m].lerp_(grad, 0.1)
                second[m].lerp_(grad.square(), 0.001)
                stage.weights_[m].addcdiv_(first[m], second[m].sqrt() + 1e-8, value=-scale)
            share = kept[7].offsets.diff().float()
            stage.bias_ -= p.balance_step * torch.sign(share - share.mean())
    assert set(got.weights_) == set(stage.weights_)
    assert all(torch.equal(got.weights_[m], stage.weights_[m]) for m in got.weights_)


def test_gradients_with_the_block_against_differences():
    """As the stage's other gradients: along each parameter's own direction, the choice of experts held fixed."""
    X, y = table(400, 10, 1)
    stage = ExpertStage(params(shared=20), MSELoss()).fit(X, y)
    w, x, yt = stage.weights_, stage._inputs(X), torch.as_tensor(y, device="cuda")
    out, kept = stage._forward(x, keep=True)
    ids, plan = kept[6], kept[7]
    grads = stage._backward(out - yt, kept)

    def loss():
        r = x @ w["embed"]
        a = expert_ops.layer_norm(r, w["norm"], w["shift"])[0]
        p = torch.sigmoid((a @ w["gate"].t()).gather(1, ids.long()))
        s = r + expert_ops.expert_products(a, plan, p / p.sum(dim=1, keepdim=True), w["w_in"], w["w_out"])
        s = s + feed_ops.feed_forward(a, w["shared_in"], w["shared_out"])
        return 0.5 * ((s @ w["head"]).double() - yt.double()).square().mean().item()

    assert set(grads) == set(w) and {"shared_in", "shared_out"} <= set(w)
    for m, grad in grads.items():
        size, h = grad.norm().item(), 2e-3
        v = grad / grad.norm()
        w[m] += h * v
        up = loss()
        w[m] -= 2 * h * v
        down = loss()
        w[m] += h * v
        assert size > 1e-4, m
        assert abs((up - down) / (2 * h) - size) <= 2e-2 * size + 2e-4, m


@pytest.mark.parametrize("scale", [1e-4, 1.0, 1e6])
def test_gradients_in_float16_are_those_of_float32(scale):
    """Nine factors rounded by 2^-11 at most each and 4 for slopes and cancelling sums: 2e-2 of the length."""
    X, y = table(2000, 20, 2)
    whole = ExpertStage(params(shared=40), MSELoss()).fit(X[:500], y[:500])
    half = ExpertStage(params(shared=40, dtype="float16", epochs=0), MSELoss()).fit(X[:500], y[:500])
    half.weights_ = {m: t.clone() for m, t in whole.weights_.items()}
    half.bias_, half.mean_, half.std_ = whole.bias_, whole.mean_, whole.std_
    x = whole._inputs(X)
    g = scale * torch.randn(2000, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    want = whole._backward(g, whole._forward(x, keep=True)[1])
    got = half._backward(g, half._forward(x, keep=True)[1])
    for m in want:
        assert got[m].dtype == torch.float32
        assert (got[m] - want[m]).norm() <= 2e-2 * want[m].norm(), m


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_the_stage_answers_in_8_bits(dtype):
    X, y = table(3000, 12, 3)
    stage = ExpertStage(params(shared=33, dtype=dtype), LogLoss()).fit(X, (y > 0).astype(np.float32))
    w, dt = stage.weights_, getattr(torch, dtype)
    codes = (*feed_ops.quantize_rows(w["shared_in"]), *feed_ops.quantize_rows(w["shared_out"]))
    for n in (1, 50, 3000):
        x = stage._inputs(X[:n])
        r = x @ w["embed"]
        a = expert_ops.layer_norm(r, w["norm"], w["shift"])[0]
        ids, weights = expert_ops.route(a @ w["gate"].t(), 2, scores="sigmoid", bias=stage.bias_)
        plan = expert_ops.expert_plan(ids, 5)
        s = r + expert_ops.expert_products(a.to(dt), plan, weights, w["w_in"].to(dt), w["w_out"].to(dt))
        s = s + feed_ops.feed_forward_int8(a.to(dt), *codes)
        assert np.array_equal(stage.predict_margin(X[:n], 0.25, int8=True), 0.25 + (s @ w["head"]).cpu().numpy())
        assert stage.predict_margin(X[:n]).shape == (n,)
    assert stage.predict_margin(X[:0], int8=True).shape == (0,)


def test_booster_block_decay_and_8_bit_moments_together():
    X, y = table(6000, 12, 4)
    booster = Booster(BoostParams(n_estimators=5, max_leaves=15, device="cuda"), MSELoss()).fit(X, y)
    base = booster.predict_margin(X)
    for dtype in ("float32", "bfloat16", "float16"):
        p = params(shared=24, dtype=dtype, weight_decay=0.1, state_bits=8, batch_rows=512)
        stage, again = (ExpertStage(p, MSELoss()).fit(X, y, base) for _ in range(2))
        for int8 in (False, True):
            m = stage.predict_margin(X, base, int8=int8)
            assert np.isfinite(m).all() and np.array_equal(m, again.predict_margin(X, base, int8=int8))


def test_what_decays():
    """With gradients of zero the matrices shrink by the decay alone, the vectors stay."""
    X, y = table(300, 8, 5)
    p = params(shared=8, weight_decay=0.5, epochs=0)
    stage = ExpertStage(p, MSELoss()).fit(X, y)
    before = {m: t.clone() for m, t in stage.weights_.items()}
    for names, decay, state in stage._groups():
        optim.adamw_step([stage.weights_[m] for m in names], [torch.zeros_like(stage.weights_[m]) for m in names], state, 1,
                         lr=0.1, weight_decay=decay)
    for m, t in stage.weights_.items():
        want = before[m] * float(np.float32(1 - 0.1 * 0.5)) if t.dim() > 1 else before[m]
        assert torch.equal(t, want), m
