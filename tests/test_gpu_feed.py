"""yabt_feed_forward and its gradients against the formulas in float64, within
the bounds that dense_plain.feed derives from the roundings on the way."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from yabt_amd import feed_ops as X

from dense_plain import feed

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = sorted(X.ACTIVATIONS)


def name(dt):
    return str(dt).replace("torch.", "")


def inputs(n, D, F, O, dt, seed):
    gen = torch.Generator().manual_seed(seed)
    return ((1.5 * torch.randn((n, D), generator=gen)).to(dt), (torch.randn((2 * F, D), generator=gen) / D ** 0.5).to(dt),
            (torch.randn((O, F), generator=gen) / F ** 0.5).to(dt), torch.randn((n, O), generator=gen).to(dt))


def run(x, w_in, w_out, dy, act):
    y, inner = X.feed_forward(x, w_in, w_out, activation=act, keep_inner=True)
    grads = X.feed_forward_grad(dy, x, w_in, w_out, inner, activation=act)
    return dict(zip(("y", "dx", "dw_in", "dw_out"), (y,) + tuple(grads)))


def check(args, act, got=None):
    x, w_in, w_out, dy = args
    got = got or run(*(t.cuda() for t in args), act)
    want = feed(*(t.double().numpy() for t in (x, w_in, w_out)), act, name(x.dtype), dy.double().numpy())
    for m, (value, bound) in want.items():
        y, most = got[m].double().cpu().numpy(), torch.finfo(x.dtype).max
        # rounding to the type makes what is half a step past its largest value infinite
        past = np.isinf(y) & (np.sign(y) * value + bound > most)
        off = np.where(past, 0.0, np.abs(y - value))
        assert np.all(off <= bound), f"{m}: {np.max(off / bound):.3g} of the bound"
    return got


# rows around the groups of 16, widths below, at and past the pieces of 16 bytes, the steps of 128 and the
# tiles; O other than D; a long sum with few tiles
SIZES = [(1, 1, 1, 1), (2, 3, 1, 5), (16, 64, 32, 64), (17, 20, 7, 33), (33, 136, 72, 16), (64, 100, 61, 100),
         (65, 64, 64, 64), (66, 28, 65, 30), (130, 129, 130, 128), (257, 100, 60, 100), (129, 128, 256, 1),
         (700, 50, 33, 40), (100, 40, 3000, 24), (1500, 16, 24, 8), (48, 200, 2050, 700), (20, 520, 2048, 1100),
         (200, 1024, 640, 520), (90, 520, 1040, 72)]


@pytest.mark.parametrize("dt", TYPES, ids=name)
@pytest.mark.parametrize("n,D,F,O", SIZES)
def test_block_and_gradients(n, D, F, O, dt):
    act = ACTS[(n + D) % 4]
    print(f"feed n={n} D={D} F={F} O={O} {act} {name(dt)}", flush=True)
    args = inputs(n, D, F, O, dt, n + D)
    got = check(args, act)
    dev = [t.cuda() for t in args]
    again = run(*dev, act)
    assert all(torch.equal(got[m], again[m]) for m in got)
    assert torch.equal(X.feed_forward(*dev[:3], activation=act), got["y"])


@pytest.mark.parametrize("dt", TYPES, ids=name)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("n", [40, 200])
def test_activations(n, act, dt):
    x, w_in, w_out, dy = inputs(n, 48, 80, 56, dt, 5)
    check((4 * x, w_in, w_out, dy), act)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dt", TYPES, ids=name)
def test_gates_far_out(act, dt):
    """Gates from -300 to 300 and 0: values and slopes stay finite and right."""
    g = torch.cat([torch.linspace(-300, 300, 99), torch.tensor([0.0])]).to(dt)
    n = g.numel()
    x = torch.stack([g, torch.ones(n, dtype=dt)], 1)
    w_in, w_out = torch.eye(2, dtype=dt), torch.ones((1, 1), dtype=dt)
    check((x, w_in, w_out, torch.ones((n, 1), dtype=dt)), act)


def large(n, D, F, O, dt, act):
    """The same on the device in float64, for sizes of the large tiles."""
    args = [t.cuda() for t in inputs(n, D, F, O, dt, n)]
    got = run(*args, act)
    x, w_in, w_out, dy = (t.double().requires_grad_(i < 3) for i, t in enumerate(args))
    g, u = (x @ w_in.t()).chunk(2, dim=1)
    f = torch.nn.functional
    a = {"silu": f.silu, "relu": f.relu, "gelu": f.gelu, "gelu_tanh": lambda t: f.gelu(t, approximate="tanh")}[act](g)
    y = (a * u) @ w_out.t()
    grads = torch.autograd.grad(y, [x, w_in, w_out], dy)
    unit = torch.finfo(dt).eps / 2
    for m, want in zip(("y", "dx", "dw_in", "dw_out"), (y.detach(),) + grads):
        off = (got[m].double() - want)
        # a rounding of the result, one of each factor of the sum, whose errors add like its terms' squares:
        # sums of hundreds of terms with independent signs and no term far above the others, so that
        # 8 of their standard deviations bound all of a few million values
        rms = float(want.square().mean().sqrt())
        assert float(off.square().mean().sqrt()) <= 1.2 * unit * rms, m
        assert bool((off.abs() <= unit * want.abs() + 8 * unit * rms).all()), m
    return got


@pytest.mark.parametrize("n,D,F,O", [(2048, 384, 2048, 4096), (2050, 392, 2056, 4104), (4100, 2048, 1025, 2049),
                                     (4096, 2048, 2048, 4096), (4120, 2056, 2064, 4104), (4097, 2049, 2050, 4099), (16_390, 520, 600, 512)])
@pytest.mark.parametrize("dt", TYPES[1:], ids=name)
def test_large_tiles(n, D, F, O, dt):
    print(f"feed large n={n} D={D} F={F} O={O} {name(dt)}", flush=True)
    large(n, D, F, O, dt, "silu")


def test_rows_of_other_pitch_and_address():
    for dt in TYPES:
        for n, D, F, O in ((70, 64, 40, 32), (9, 33, 17, 20), (300, 128, 64, 64)):
            x, w_in, w_out, dy = (t.cuda() for t in inputs(n, D, F, O, dt, 3))
            want = run(x, w_in, w_out, dy, "silu")
            wide_x = torch.full((n, D + 13), float("nan"), dtype=dt, device="cuda")
            wide_dy = torch.full((n + 1, O + 5), float("nan"), dtype=dt, device="cuda")
            wide_x[:, 3:3 + D], wide_dy[1:, 1:1 + O] = x, dy
            got = run(wide_x[:, 3:3 + D], w_in.t().contiguous().t(), w_out, wide_dy[1:, 1:1 + O], "silu")
            assert all(torch.equal(want[m], got[m]) for m in want)


@pytest.mark.parametrize("n", [5, 64, 90, 700])
def test_a_row_that_is_not_finite_stays_alone(n):
    x, w_in, w_out, dy = (t.cuda() for t in inputs(n, 64, 40, 32, torch.bfloat16, 4))
    want = X.feed_forward(x, w_in, w_out)
    bad = x.clone()
    bad[n - 2, 7], bad[1, 0] = float("nan"), float("inf")
    got = X.feed_forward(bad, w_in, w_out)
    keep = torch.ones(n, dtype=torch.bool, device="cuda")
    keep[n - 2] = keep[1] = False
    assert torch.equal(got[keep], want[keep]) and bool(torch.isnan(got[n - 2]).all())
    assert not bool(torch.isfinite(got[1]).all())


def test_no_rows():
    for dt in TYPES:
        x, w_in, w_out, dy = (t.cuda() for t in inputs(0, 24, 10, 12, dt, 1))
        got = run(x, w_in, w_out, dy, "gelu")
        assert got["y"].shape == (0, 12) and got["dx"].shape == (0, 24)
        assert not bool(got["dw_in"].any()) and not bool(got["dw_out"].any())


@pytest.mark.parametrize("n", [3, 500])
def test_captured_and_replayed(n):
    """Two graphs of forward and backward, replayed in turn with other work between them."""
    sets = [[t.cuda() for t in inputs(n, 96, 64, 48, torch.bfloat16, s)] for s in (1, 2)]
    graphs = []
    for s in sets:
        run(*s, "silu")
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(*s, "silu")
        graphs.append((graph, out))
    for k in range(5):
        for s, (graph, out) in zip(sets, graphs):
            s[0].mul_(0.9)
            graph.replay()
        eager = [run(*s, "silu") for s in sets]
        torch.cuda.synchronize()
        for e, (_, out) in zip(eager, graphs):
            assert all(torch.equal(e[m], out[m]) for m in e), k


def test_on_two_streams_at_once():
    sets = [[t.cuda() for t in inputs(n, 200, 100, 72, torch.float16, n)] for n in (40, 900)]
    want = [run(*s, "relu") for s in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], []
    for _ in range(3):
        got = []
        for s, on in zip(sets, streams):
            with torch.cuda.stream(on):
                got.append(run(*s, "relu"))
        torch.cuda.synchronize()
        assert all(torch.equal(a[m], b[m]) for a, b in zip(want, got) for m in a)


def test_half_beyond_its_range():
    """In float16 an h beyond 65504 makes its own row alone infinite or NaN."""
    for n in (8, 100):
        x, w_in, w_out, _ = (t.cuda() for t in inputs(n, 16, 8, 8, torch.float16, 2))
        x[2] *= 3000.0
        y = X.feed_forward(x, w_in, w_out, activation="relu")
        keep = torch.arange(n, device="cuda") != 2
        assert bool(torch.isfinite(y[keep]).all()) and not bool(torch.isfinite(y[2]).all())


def test_an_inner_that_was_moved():
    """From a multiple of 256 bytes on it serves as it did; elsewhere its parts would be
    looked for beside where they are, and it is refused."""
    x, w_in, w_out, dy = (t.cuda() for t in inputs(70, 40, 24, 30, torch.bfloat16, 6))
    y, inner = X.feed_forward(x, w_in, w_out, keep_inner=True)
    want = X.feed_forward_grad(dy, x, w_in, w_out, inner)
    packed = torch.zeros(inner.numel() + 1024, dtype=torch.uint8, device="cuda")
    for at in (0, 512, 768):
        packed[at:at + inner.numel()] = inner
        got = X.feed_forward_grad(dy, x, w_in, w_out, packed[at:at + inner.numel()])
        assert all(torch.equal(a, b) for a, b in zip(got, want)), at
    for at in (16, 128, 300):
        with pytest.raises(ValueError, match="multiple of 256"):
            X.feed_forward_grad(dy, x, w_in, w_out, packed[at:at + inner.numel()])


@pytest.mark.parametrize("n", [5, 40, 90, 700])
def test_a_float32_row_that_is_not_finite_stays_alone(n):
    x, w_in, w_out, dy = (t.cuda() for t in inputs(n, 64, 40, 32, torch.float32, 4))
    want, inner = X.feed_forward(x, w_in, w_out, keep_inner=True)
    dx = X.feed_forward_grad(dy, x, w_in, w_out, inner)[0]
    bad = x.clone()
    bad[n - 2, 7], bad[1, 0] = float("nan"), float("inf")
    got, inner = X.feed_forward(bad, w_in, w_out, keep_inner=True)
    keep = torch.ones(n, dtype=torch.bool, device="cuda")
    keep[n - 2] = keep[1] = False
    assert torch.equal(got[keep], want[keep]) and not bool(torch.isfinite(got[~keep]).any())
    assert torch.equal(X.feed_forward_grad(dy, bad, w_in, w_out, inner)[0][keep], dx[keep])


# few tiles over a long sum, which is made in parts: of [g u] over D, of dh over O; inner widths that are
# and are not whole pieces, one tile and many
@pytest.mark.parametrize("dt", TYPES, ids=name)
@pytest.mark.parametrize("n,D,F,O", [(65, 2600, 17, 2000), (83, 2520, 256, 2520), (130, 4001, 33, 1500),
                                     (300, 3000, 64, 40), (300, 40, 64, 3100), (777, 500, 1333, 500)])
def test_few_tiles_over_long_sums(n, D, F, O, dt):
    check(inputs(n, D, F, O, dt, n + F), "gelu")


@pytest.mark.parametrize("dt", TYPES, ids=name)
def test_few_tiles_over_long_sums_without_a_kept_inner(dt):
    x, w_in, w_out, _ = (t.cuda() for t in inputs(83, 2520, 250, 60, dt, 8))
    assert torch.equal(X.feed_forward(x, w_in, w_out), X.feed_forward(x, w_in, w_out, keep_inner=True)[0])


def test_sums_in_parts_captured_and_replayed():
    x, w_in, w_out, dy = (t.cuda() for t in inputs(83, 2520, 250, 2000, torch.float32, 9))
    run(x, w_in, w_out, dy, "silu")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(x, w_in, w_out, dy, "silu")
    for k in range(4):
        x.mul_(-0.75), dy.add_(0.25)
        graph.replay()
        want = run(x, w_in, w_out, dy, "silu")
        torch.cuda.synchronize()
        assert all(torch.equal(got[m], want[m]) for m in want), k
