"""yabt_route, its gradient and yabt_expert_plan against the definitions in
float64, row by row.  Ids are compared exactly: logits and biases lie on grids
on which two float32 keys are equal or far apart (checked).  Weights are off by
the exponentials' and divisions' few roundings and those of sums over at most
1024 terms in 16 + 6 steps: 64 rounding units."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from yabt_amd import expert_ops as X

from expert_plain import TINY, U32, UNIT, choose, plan, scores_of, weights_grad, weights_of

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def name(dt):
    return str(dt).replace("torch.", "")


def logits_of(n, E, dt, seed, masked=0.1, ties=True):
    rng = np.random.default_rng(seed)
    x = np.round(rng.normal(size=(n, E)) * (8 if ties else 32)) / 16      # exact in every type
    if masked:
        x[rng.random((n, E)) < masked] = -np.inf
        x[rng.random((n, E)) < masked / 10] = np.nan
        if n > 2:
            x[1] = -np.inf                                 # nothing left
            x[2] = -np.inf
            x[2, E // 2] = 0.25                            # one left
    return torch.from_numpy(x).to(dt)


def check(x, k, scores, bias, groups, keep, renormalise, scale, seed):
    n, E = x.shape
    xd = x.double().numpy()
    how = dict(scores=scores, renormalise=renormalise, scale=scale)
    ids, w = X.route(x.cuda(), k, bias=None if bias is None else torch.from_numpy(bias).cuda(), groups=groups,
                     keep_groups=keep, **how)
    got, gw = ids.cpu().numpy(), w.double().cpu().numpy()
    xo = np.where(np.isnan(xd), -np.inf, xd)
    dw = np.random.default_rng(seed).normal(size=(n, k)).astype(np.float32)
    dl = X.route_grad(torch.from_numpy(dw).cuda(), x.cuda(), ids, **how).double().cpu().numpy()
    dt = name(x.dtype)
    for r in range(n):
        want = choose(xo[r], k, scores, bias, groups, keep)
        assert list(got[r]) == want, f"row {r}"
        ref = weights_of(xo[r], want, scores, renormalise, scale)
        assert np.all(np.abs(gw[r] - ref) <= 64 * U32 * np.abs(ref) + 1e-37), f"row {r}"
        rd = weights_grad(xo[r], want, dw[r].astype(np.float64), scores, renormalise, scale)
        p = scores_of(xo[r], scores)
        big = scale * np.abs(dw[r]).max() * (1.0 if scores == "softmax" or not renormalise else
                                             1.0 / max(sum(p[i] for i in want if i >= 0), 1e-30))
        size = np.zeros(E)
        for j, i in enumerate(want):
            if i >= 0:
                size[i] = ref[j] / scale if scores == "softmax" else p[i]
        tol = 128 * U32 * big * (size + (p if scores == "softmax" and not renormalise else 0.0))
        assert np.all(np.abs(dl[r] - rd) <= tol + UNIT[dt] * np.abs(rd) + TINY[dt]), f"row {r}"


@pytest.mark.parametrize("dt", TYPES, ids=name)
@pytest.mark.parametrize("E,k", [(1, 1), (2, 2), (7, 3), (16, 16), (17, 4), (33, 8), (60, 4), (64, 32), (65, 6),
                                 (128, 17), (200, 8), (256, 8), (257, 5), (512, 32), (1000, 9), (1024, 32)])
def test_every_score(E, k, dt):
    for scores in ("softmax", "sigmoid"):
        for renormalise in (True, False):
            print(f"route E={E} k={k} {name(dt)} {scores} {renormalise}", flush=True)
            check(logits_of(41, E, dt, E + k), k, scores, None, 1, 1, renormalise, 2.5, E)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups,keep,k", [(6, 2, 1, 2), (64, 8, 4, 8), (64, 64, 5, 6), (60, 12, 3, 4), (256, 8, 4, 8),
                                             (255, 5, 2, 7), (1024, 64, 9, 32), (1000, 8, 1, 3), (32, 4, 4, 4)])
def test_groups_and_bias(E, groups, keep, k, scores):
    rng = np.random.default_rng(E)
    for bias in (None, (np.round(rng.normal(size=E) * 8) / 64).astype(np.float32)):
        x = logits_of(67, E, torch.float32, groups, masked=0.3)
        check(x, k, scores, bias, groups, keep, True, 1.0, k)


def test_equal_keys_go_to_the_lowest_index():
    x = torch.zeros((3, 300))
    x[1, 100:] = -0.0                                      # equal to 0
    x[2, 7] = x[2, 250] = 1.0
    ids, w = X.route(x.cuda(), 4)
    assert ids.tolist() == [[0, 1, 2, 3], [0, 1, 2, 3], [7, 250, 0, 1]]
    assert torch.equal(w[0].cpu(), torch.full((4,), 0.25))


def test_extreme_logits():
    """Logits that over- and underflow an exponential, the type's lowest value and infinity."""
    low = torch.finfo(torch.float32).min
    x = torch.tensor([[1e4, -1e4, 0.0, low, 1e4], [low, low, low, low, low], [200.0, -200.0, 100.0, -100.0, 0.0]])
    for scores in ("softmax", "sigmoid"):
        for renormalise in (True, False):
            check(x, 3, scores, None, 1, 1, renormalise, 1.0, 0)
    ids, w = X.route(torch.tensor([[0.0, float("inf"), 3.0, float("nan")]]).cuda(), 3, scores="sigmoid",
                     renormalise=False)
    assert ids.tolist() == [[1, 2, 0]] and w[0, 0] == 1.0


def test_keys_do_not_overlap_by_accident():
    """The grids of these tests: equal or at least 1e-6 apart, float32's step near 1 being 1.2e-7."""
    grid = np.arange(-64, 65) / 16
    p = 1.0 / (1.0 + np.exp(-grid))
    keys = np.unique((p.astype(np.float32)[:, None] + (np.arange(-40, 41) / 64).astype(np.float32)[None]).ravel().astype(np.float64))
    gap = np.diff(keys)
    assert (gap[gap > 3e-7] > 1e-6).mean() > 0.99          # what the seeds above draw is checked by their passing


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalise", [True, False])
def test_gradient_against_differences(scores, renormalise):
    """Central differences of the float64 weights, the choice held fixed."""
    x = logits_of(9, 40, torch.float32, 5, ties=False)
    ids, _ = X.route(x.cuda(), 5, scores=scores, renormalise=renormalise, scale=1.7)
    dw = np.random.default_rng(2).normal(size=(9, 5)).astype(np.float32)
    dl = X.route_grad(torch.from_numpy(dw).cuda(), x.cuda(), ids, scores=scores, renormalise=renormalise, scale=1.7)
    dl, xd, got = dl.double().cpu().numpy(), np.where(np.isnan(x.double().numpy()), -np.inf, x.double().numpy()), ids.cpu().numpy()
    h = 1e-5
    for r in range(9):
        for e in range(40):
            if not xd[r, e] > -np.inf:
                assert dl[r, e] == 0
                continue
            up, down = xd[r].copy(), xd[r].copy()
            up[e] += h
            down[e] -= h
            both = [(weights_of(v, list(got[r]), scores, renormalise, 1.7) * dw[r]).sum() for v in (up, down)]
            assert abs(dl[r, e] - (both[0] - both[1]) / (2 * h)) <= 1e-6 * max(1.0, np.abs(dw[r]).sum())


def test_strides_and_id_types():
    wide = logits_of(50, 90, torch.bfloat16, 8)
    for view in (wide[:, 5:69], wide[::3, 1:65], wide[:64, :50].t()):
        a = X.route(view.cuda() if view.is_contiguous() else wide.cuda().as_strided(view.shape, view.stride(), view.storage_offset()), 4)
        b = X.route(view.contiguous().cuda(), 4)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    ids, _ = X.route(wide.cuda(), 4)
    dw = torch.randn((50, 8), device="cuda")[:, ::2]
    assert torch.equal(X.route_grad(dw, wide.cuda(), ids.long()), X.route_grad(dw.contiguous(), wide.cuda(), ids))
    far = torch.tensor([[2 ** 32 + 1, -5, 3]], device="cuda")      # neither names an expert
    assert X.expert_plan(far, 8).slots.tolist() == [2, -1, -1]


@pytest.mark.parametrize("n,k,E", [(1, 1, 1), (1, 6, 64), (63, 2, 5), (700, 3, 1024), (2048, 1, 7), (2049, 1, 7),
                                   (5000, 4, 33), (40_001, 8, 256), (3_000_000, 1, 3)])
def test_plan(n, k, E):
    rng = np.random.default_rng(n)
    ids = rng.integers(-1, E + 1, size=(n, k)).astype(np.int32)        # -1 and E: no expert
    if E > 4:
        ids[ids == 3] = 2                                              # an expert without rows
    got = X.expert_plan(torch.from_numpy(ids).cuda(), E)
    offsets, slots, rows = plan(ids, E)
    assert np.array_equal(got.offsets.cpu().numpy(), offsets)
    assert np.array_equal(got.slots.cpu().numpy(), slots) and np.array_equal(got.rows.cpu().numpy(), rows)
    assert got.experts == E


@pytest.mark.parametrize("n,k,E", [(8193, 1, 2), (65_536, 2, 64), (131_073, 1, 64), (16_384, 4, 512), (16_385, 4, 513),
                                   (16_400, 8, 1024)])
def test_plan_of_few_and_many_blocks(n, k, E):
    test_plan(n, k, E)


def test_nothing_routed():
    plan_ = X.expert_plan(torch.full((10, 2), -1, dtype=torch.int32, device="cuda"), 4)
    assert plan_.offsets.tolist() == [0] * 5 and plan_.slots.tolist() == [-1] * 20
    empty = X.expert_plan(torch.empty((0, 2), dtype=torch.int32, device="cuda"), 4)
    assert empty.offsets.tolist() == [0] * 5 and empty.slots.numel() == 0
    ids, w = X.route(torch.empty((0, 5), device="cuda"), 2)
    assert ids.shape == (0, 2) and X.route_grad(w, torch.empty((0, 5), device="cuda"), ids).shape == (0, 5)


def test_many_rows_and_another_stream():
    x = logits_of(20_000, 96, torch.float32, 4)
    ids, w = X.route(x.cuda(), 6)
    few, fw = X.route(x[-777:].cuda(), 6)
    assert torch.equal(ids[-777:], few) and torch.equal(w[-777:], fw)
    s = torch.cuda.Stream()
    xs = x.cuda()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = X.route(xs, 6)
        got = X.expert_plan(other[0], 96)
    s.synchronize()
    assert torch.equal(other[0], ids) and torch.equal(got.slots, X.expert_plan(ids, 96).slots)


def test_refusals():
    x = torch.zeros((4, 12), device="cuda")
    ids, w = X.route(x, 2)
    for call in (lambda: X.route(x, 0), lambda: X.route(x, 13), lambda: X.route(torch.zeros((1, 64), device="cuda"), 33),
                 lambda: X.route(torch.zeros((1, 1025), device="cuda"), 2), lambda: X.route(x, 2, scores="relu"),
                 lambda: X.route(x, 2, groups=5), lambda: X.route(x, 2, groups=4, keep_groups=5),
                 lambda: X.route(x, 2, bias=torch.zeros(11, device="cuda")), lambda: X.route(x.double(), 2),
                 lambda: X.route(x[0], 2), lambda: X.route_grad(w[:3], x, ids), lambda: X.route_grad(w, x, ids[:3]),
                 lambda: X.route_grad(w, x, ids.float()), lambda: X.route_grad(w, x, ids, scores="?"),
                 lambda: X.expert_plan(ids, 0), lambda: X.expert_plan(ids, 1025), lambda: X.expert_plan(ids[0], 4)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: X.route(x.cpu(), 2), lambda: X.expert_plan(ids.cpu(), 4), lambda: X.route_grad(w, x, ids.cpu())):
        with pytest.raises(RuntimeError):
            call()
