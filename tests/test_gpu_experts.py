"""yabt_experts and yabt_experts_grad against the formulas in float64, within
the bounds that expert_plain.products derives from the roundings on the way."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from yabt_amd import expert_ops as X

from expert_plain import products

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def name(dt):
    return str(dt).replace("torch.", "")


def inputs(n, D, F, E, k, dt, seed, unused=0.05, skew=0.0):
    """x, ids, weights, w_in, w_out, dy; expert E - 1 of three or more stays
    without rows, and some slots without an expert."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((n, D), generator=gen).to(dt)
    w_in = (torch.randn((E, 2 * F, D), generator=gen) / D ** 0.5).to(dt)
    w_out = (torch.randn((E, D, F), generator=gen) / F ** 0.5).to(dt)
    gate = torch.randn((n, E), generator=gen) + skew * torch.arange(E)
    if E > 2 and k < E:
        gate[:, E - 1] = -1e9
    ids = gate.topk(k, dim=1).indices.to(torch.int32)
    weights = torch.rand((n, k), generator=gen) + 0.1
    off = torch.rand((n, k), generator=gen) < unused
    ids[off] = -1
    weights[off] = 0.0
    dy = torch.randn((n, D), generator=gen).to(dt)
    return x, ids, weights, w_in, w_out, dy


def run(x, ids, weights, w_in, w_out, dy=None):
    plan = X.expert_plan(ids, w_in.shape[0])
    if dy is None:
        return dict(y=X.expert_products(x, plan, weights, w_in, w_out))
    y, inner = X.expert_products(x, plan, weights, w_in, w_out, keep_inner=True)
    grads = X.expert_products_grad(dy, x, plan, weights, w_in, w_out, inner)
    return dict(zip(("y", "dx", "dweights", "dw_in", "dw_out"), (y,) + tuple(grads)))


def check(args, grad=True, got=None):
    x, ids, weights, w_in, w_out, dy = args
    if got is None:
        got = run(*(t.cuda() for t in (args if grad else args[:5])))
    d = [t.double().numpy() for t in (x, weights, w_in, w_out, dy)]
    want = products(d[0], ids.numpy(), d[1], d[2], d[3], name(x.dtype), d[4] if grad else None)
    for m, (value, bound) in want.items():
        off = np.abs(got[m].double().cpu().numpy() - value)
        assert np.all(off <= bound), f"{m}: {np.max(off / bound):.3g} of the bound"
    return got


# widths below, at and past the pieces of 16 bytes, the steps of 128 and the tiles
SIZES = [(1, 1, 1, 1, 1), (3, 1, 2, 2, 2), (5, 3, 1, 3, 1), (40, 20, 7, 5, 2), (33, 64, 32, 4, 4), (100, 28, 65, 3, 1),
         (257, 100, 60, 7, 1), (300, 50, 33, 6, 3), (129, 128, 64, 2, 1), (130, 136, 72, 9, 2), (515, 129, 130, 2, 2),
         (64, 500, 100, 20, 8)]


@pytest.mark.parametrize("dt", TYPES, ids=name)
@pytest.mark.parametrize("n,D,F,E,k", SIZES)
def test_products_and_gradients(n, D, F, E, k, dt):
    print(f"experts n={n} D={D} F={F} E={E} k={k} {name(dt)}", flush=True)
    args = inputs(n, D, F, E, k, dt, n + D)
    got = check(args)
    again = run(*(t.cuda() for t in args))
    assert all(torch.equal(got[m], again[m]) for m in got)
    check(args, grad=False)


@pytest.mark.parametrize("dt", TYPES, ids=name)
@pytest.mark.parametrize("n,D,F,E,k", [(1100, 200, 192, 2, 1), (700, 256, 264, 2, 2), (1000, 321, 193, 3, 2),
                                       (1037, 320, 448, 4, 2)])
def test_large_tiles(n, D, F, E, k, dt):
    """Enough rows per expert for the large tiles; ends inside a tile on every side."""
    check(inputs(n, D, F, E, k, dt, n))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=name)
@pytest.mark.parametrize("n,D,F,E,k", [(7000, 400, 520, 16, 1), (6001, 397, 515, 8, 2), (9000, 1032, 392, 16, 1)])
def test_large_tiles_of_every_product(n, D, F, E, k, dt):
    """Enough tiles and sums long enough that 256 x 256 tiles make all six products or some of them."""
    check(inputs(n, D, F, E, k, dt, n))


@pytest.mark.parametrize("dt", TYPES, ids=name)
@pytest.mark.parametrize("n,D,F,E,k", [(1, 300, 70, 64, 6), (2, 129, 33, 20, 8), (9, 64, 48, 3, 1), (60, 96, 130, 2, 1),
                                       (250, 40, 33, 100, 2), (120, 33, 20, 4, 1), (500, 24, 17, 200, 1)])
def test_few_rows(n, D, F, E, k, dt):
    """The kernels for few rows: one, several and more than 16 slots an expert, more experts than waves."""
    check(inputs(n, D, F, E, k, dt, n + E), grad=False)
    check(inputs(n, D, F, E, k, dt, n + E, unused=0.5))


@pytest.mark.parametrize("dt", TYPES, ids=name)
def test_uneven_experts(dt):
    """One expert with most rows, others with a few or none; an expert that no id names."""
    args = inputs(900, 72, 40, 12, 2, dt, 3, skew=0.7)
    got = check(args)
    for m in ("dw_in", "dw_out"):
        assert torch.count_nonzero(got[m][11]) == 0


@pytest.mark.parametrize("dt", TYPES, ids=name)
@pytest.mark.parametrize("k", [1, 3])
def test_rows_without_an_expert(k, dt):
    x, ids, weights, w_in, w_out, dy = inputs(70, 48, 24, 4, k, dt, 8)
    ids[::3] = -1
    ids[1::7] = 99
    got = check((x, ids, weights, w_in, w_out, dy))
    assert torch.count_nonzero(got["y"][::3]) == 0 and torch.count_nonzero(got["dx"][::3]) == 0
    assert torch.count_nonzero(got["dweights"][::3]) == 0
    none = torch.full_like(ids, -1)
    got = run(*(t.cuda() for t in (x, none, weights, w_in, w_out, dy)))
    assert all(torch.count_nonzero(v) == 0 for v in got.values())


@pytest.mark.parametrize("dt", TYPES, ids=name)
def test_one_slot_a_row_writes_every_row(dt):
    """k = 1 in tiles: rows without an expert, single, in runs and at the end, in
    memory that held NaN before."""
    n, D, F, E = 1500, 70, 40, 3
    args = list(inputs(n, D, F, E, 1, dt, 9))
    for rows in (slice(0, 1), slice(100, 400), slice(1499, 1500), slice(700, 900, 2)):
        args[1][rows] = -1
        args[2][rows] = 0.0
    out = torch.full((n, D), float("nan"), dtype=dt, device="cuda")
    del out                                           # y is likely to get this memory
    got = check(args)
    empty = (args[1] < 0).flatten()
    assert torch.all(got["y"].cpu()[empty] == 0) and torch.all(got["dx"].cpu()[empty] == 0)


@pytest.mark.parametrize("dt", TYPES, ids=name)
def test_nothing_leaks_between_rows_and_experts(dt):
    """NaN in an unused expert's weights and in a row of its own stay there, at
    sizes that end inside pieces, steps and tiles."""
    for D, F in ((40, 24), (37, 19)):
        x, ids, weights, w_in, w_out, dy = inputs(150, D, F, 4, 1, dt, D, unused=0.0)
        clean = run(*(t.cuda() for t in (x, ids, weights, w_in, w_out, dy)))
        w_in[3], w_out[3] = float("nan"), float("nan")         # expert 3 has no rows
        x[17], x[149] = float("nan"), float("inf")
        got = run(*(t.cuda() for t in (x, ids, weights, w_in, w_out, dy)))
        good = [r for r in range(150) if r not in (17, 149)]
        assert torch.equal(got["y"][good], clean["y"][good]) and torch.equal(got["dx"][good], clean["dx"][good])
        assert torch.isnan(got["y"][17]).all()
        free = [e for e in range(4) if e not in (int(ids[17]), int(ids[149]))]
        assert torch.equal(got["dw_in"][free], clean["dw_in"][free])
        assert torch.equal(got["dw_out"][free], clean["dw_out"][free])


@pytest.mark.parametrize("dt", TYPES, ids=name)
def test_strides_and_alignment(dt):
    """x and dy inside wider matrices, at starts that no 16-byte access is aligned to."""
    x, ids, weights, w_in, w_out, dy = inputs(90, 64, 32, 3, 2, dt, 2)
    want = run(*(t.cuda() for t in (x, ids, weights, w_in, w_out, dy)))
    for wide, start in ((80, 8), (67, 3), (65, 1)):
        xw, dw = torch.full((90, wide), float("nan"), dtype=dt), torch.full((90, wide), float("nan"), dtype=dt)
        xw[:, start:start + 64], dw[:, start:start + 64] = x, dy
        got = run(xw.cuda()[:, start:start + 64], *(t.cuda() for t in (ids, weights, w_in, w_out)),
                  dw.cuda()[:, start:start + 64])
        check((x, ids, weights, w_in, w_out, dy), got=got)
    flat = torch.empty(w_in.numel() + 1, dtype=dt, device="cuda")
    moved = flat[1:].view(w_in.shape).copy_(w_in)              # weights off 16 bytes
    check((x, ids, weights, w_in, w_out, dy), got=run(x.cuda(), ids.cuda(), weights.cuda(), moved, w_out.cuda(), dy.cuda()))
    turned = run(x.cuda().t().contiguous().t(), ids.cuda().long(), weights.cuda().double(),
                 w_in.cuda().transpose(1, 2).contiguous().transpose(1, 2), w_out.cuda(), dy.cuda())
    assert all(torch.equal(turned[m], want[m]) for m in want)


def test_large_gates():
    """Gates whose exponential over- and underflows: silu is g or 0."""
    args = list(inputs(40, 16, 8, 2, 1, torch.float32, 6, unused=0.0))
    args[0] = args[0] * 200.0
    got = run(*(t.cuda() for t in args))
    assert all(torch.isfinite(v).all() for v in got.values())
    check(tuple(args), got=got)


@pytest.mark.parametrize("k", [1, 2])
def test_gradient_against_differences(k):
    """The directional derivative of sum(c y) by central differences of the
    float64 formula, and by the gradients in float32."""
    x, ids, weights, w_in, w_out, dy = inputs(37, 24, 20, 3, k, torch.float32, 12)
    got = {m: v.double().cpu().numpy() for m, v in run(*(t.cuda() for t in (x, ids, weights, w_in, w_out, dy))).items()}
    base = dict(x=x, dweights=weights, dw_in=w_in, dw_out=w_out)
    rng = np.random.default_rng(1)
    v = {m: rng.normal(size=tuple(t.shape)) for m, t in base.items()}
    v["dweights"][ids.numpy() < 0] = 0.0
    h = 1e-5

    def loss(s):
        a = {m: t.double().numpy() + s * h * v[m] for m, t in base.items()}
        y = products(a["x"], ids.numpy(), a["dweights"], a["dw_in"], a["dw_out"], "float32")["y"][0]
        return (y * dy.double().numpy()).sum()

    slope = (got["dx"] * v["x"]).sum() + sum((got[m] * v[m]).sum() for m in ("dweights", "dw_in", "dw_out"))
    size = np.sqrt((got["dx"] ** 2).sum() + sum((got[m] ** 2).sum() for m in ("dweights", "dw_in", "dw_out")))
    assert abs(slope - (loss(1) - loss(-1)) / (2 * h)) <= 1e-5 * size


def test_no_rows_and_other_streams():
    x, ids, weights, w_in, w_out, dy = (t.cuda() for t in inputs(60, 32, 16, 3, 2, torch.bfloat16, 4))
    empty = run(x[:0], ids[:0], weights[:0], w_in, w_out, dy[:0])
    assert empty["y"].shape == (0, 32) and all(torch.count_nonzero(v) == 0 for v in empty.values())
    want = run(x, ids, weights, w_in, w_out, dy)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run(x, ids, weights, w_in, w_out, dy)
    s.synchronize()
    assert all(torch.equal(got[m], want[m]) for m in want)


def test_graph_replays():
    """The whole layer captured into a HIP graph, replayed with new inputs and eager work in between."""
    x, ids, weights, w_in, w_out, dy = (t.cuda() for t in inputs(90, 48, 24, 5, 2, torch.bfloat16, 5))
    run(x, ids, weights, w_in, w_out, dy)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(x, ids, weights, w_in, w_out, dy)
    for seed in range(3):
        for have, new in zip((x, ids, weights, w_in, w_out, dy), inputs(90, 48, 24, 5, 2, torch.bfloat16, 50 + seed)):
            have.copy_(new)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = run(x, ids, weights, w_in, w_out, dy)
        assert all(torch.equal(got[m], want[m]) for m in want), f"replay {seed}"


def test_refusals():
    x, ids, weights, w_in, w_out, dy = (t.cuda() for t in inputs(12, 16, 8, 3, 2, torch.float32, 7))
    plan = X.expert_plan(ids, 3)
    y, inner = X.expert_products(x, plan, weights, w_in, w_out, keep_inner=True)
    for call in (lambda: X.expert_products(x[:5], plan, weights, w_in, w_out),
                 lambda: X.expert_products(x, X.expert_plan(ids, 4), weights, w_in, w_out),
                 lambda: X.expert_products(x, plan, weights[:, :1], w_in, w_out),
                 lambda: X.expert_products(x, plan, weights, w_in[:, :7], w_out),
                 lambda: X.expert_products(x, plan, weights, w_in[0], w_out),
                 lambda: X.expert_products(x.half(), plan, weights, w_in, w_out),
                 lambda: X.expert_products(x, plan, weights, w_in.cpu(), w_out),
                 lambda: X.expert_products_grad(dy[:3], x, plan, weights, w_in, w_out, inner),
                 lambda: X.expert_products_grad(dy.half(), x, plan, weights, w_in, w_out, inner),
                 lambda: X.expert_products_grad(dy, x, plan, weights, w_in, w_out, inner[:, :8]),
                 lambda: X.expert_products_grad(dy, x, plan, weights, w_in, w_out, inner.double())):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError, match="HIP device"):
        X.expert_products(x.cpu(), plan, weights, w_in, w_out)
