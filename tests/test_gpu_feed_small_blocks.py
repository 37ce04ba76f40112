"""Small blocks of 16-bit types, where one large value may decide the error of all:
h and the inner gradients keep 16 bits, so that an output has its own rounding alone."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from yabt_amd import _lib, feed_ops as X

from dense_plain import feed

TYPES = [torch.bfloat16, torch.float16]
TWICE = 1 << 11
# one row and few, more than 64, whole pieces of 16 bytes and not, y by few-row kernels and by tiles, [g u], dh and the
# gradients in parts, sums shorter than a step
SIZES = [(1, 24, 24, 24), (1, 1, 1, 1), (3, 100, 61, 100), (16, 64, 128, 40), (17, 64, 64, 64), (40, 60, 100, 72), (33, 40, 90, 48),
         (58, 64, 64, 64), (63, 40, 68, 39), (60, 13, 1000, 17), (48, 16, 4000, 16), (100, 32, 40, 32), (101, 41, 27, 30),
         (300, 16, 8, 500), (700, 1, 700, 40), (500, 1, 4000, 900), (16, 40, 2050, 2100), (16, 40, 2048, 2304), (2, 24, 900, 3000),
         (1, 2000, 4000, 1000), (65, 10, 2600, 3000), (66, 2600, 40, 1500), (70, 2000, 30, 2000), (1, 2001, 4003, 1001), (0, 8, 8, 8)]


def name(dt):
    return str(dt).replace("torch.", "")


def test_sizes_are_small_blocks():
    forms = _lib.load().yabt_feed_forward_forms
    assert all(forms(dt, *s) & TWICE for s in SIZES for dt in (1, 2)) and not any(forms(0, *s) & TWICE for s in SIZES)
    assert not forms(1, 16, 512, 512, 512) & TWICE and not forms(1, 8192, 64, 64, 64) & TWICE
    # what large tiles make has one part: those sizes have many values, but for a narrow output
    assert forms(1, 256, 4096, 16_384, 2) & (TWICE | 4) == 4
    sizes = [f(1, 40, 60, 100, 72) for f in (_lib.load().yabt_feed_forward_inner_bytes, _lib.load().yabt_feed_forward_workspace_bytes,
                                             _lib.load().yabt_feed_forward_grad_workspace_bytes)]
    assert sizes[0] >= 40 * 4 * 200 + 2 * 40 * 104 * 2 and sizes[2] >= 2 * 40 * 2 * 104 * 2


def inputs(n, D, F, O, dt, seed):
    gen = torch.Generator().manual_seed(seed)
    return ((1.5 * torch.randn((n, D), generator=gen)).to(dt), (torch.randn((2 * F, D), generator=gen) / D ** 0.5).to(dt),
            (torch.randn((O, F), generator=gen) / F ** 0.5).to(dt), torch.randn((n, O), generator=gen).to(dt))


def run(x, w_in, w_out, dy, act):
    y, inner = X.feed_forward(x, w_in, w_out, activation=act, keep_inner=True)
    return (y,) + tuple(X.feed_forward_grad(dy, x, w_in, w_out, inner, activation=act))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES, ids=name)
@pytest.mark.parametrize("size", SIZES)
def test_one_rounding(size, dt):
    """Two parts leave 2^-16 of a value (fp16 near its least step: 2^-25, of values near 1): beside the outputs' own
    rounding, 2^-10 rms in bf16 and 2^-13 in fp16, that is 2% and 13% at most of it, added as squares
    1%.  20% of slack for ties that it moves among few values."""
    act = sorted(X.ACTIVATIONS)[sum(size) % 4]
    print(f"feed small {size} {act} {name(dt)}", flush=True)
    args = inputs(*size, dt, sum(size))
    dev = [t.cuda() for t in args]
    got = run(*dev, act)
    x, w_in, w_out, dy = (t.double().numpy() for t in args)
    want = feed(x, w_in, w_out, act, name(dt), dy)
    for m, a in zip(("y", "dx", "dw_in", "dw_out"), got):
        exact = torch.from_numpy(want[m][0])
        once = float((exact.to(dt).double() - exact).norm())
        least = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps * exact.numel() ** 0.5
        assert float((a.double().cpu() - exact).norm()) <= 1.2 * once + least, m
        assert np.all(np.abs(a.double().cpu().numpy() - want[m][0]) <= want[m][1]), m
    assert torch.equal(X.feed_forward(*dev[:3], activation=act), got[0])
    assert all(torch.equal(a, b) for a, b in zip(got, run(*dev, act)))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES, ids=name)
@pytest.mark.parametrize("size", [(9, 33, 17, 20), (70, 64, 40, 32)])
def test_other_pitches_a_moved_inner_and_replays(size, dt):
    n, D, F, O = size
    x, w_in, w_out, dy = (t.cuda() for t in inputs(*size, dt, 3))
    want = run(x, w_in, w_out, dy, "silu")
    wide_x = torch.full((n, D + 13), float("nan"), dtype=dt, device="cuda")
    wide_dy = torch.full((n + 1, O + 5), float("nan"), dtype=dt, device="cuda")
    wide_x[:, 3:3 + D], wide_dy[1:, 1:1 + O] = x, dy
    assert all(torch.equal(a, b) for a, b in zip(want, run(wide_x[:, 3:3 + D], w_in, w_out, wide_dy[1:, 1:1 + O], "silu")))
    y, inner = X.feed_forward(x, w_in, w_out, keep_inner=True)
    packed = torch.zeros(inner.numel() + 1024, dtype=torch.uint8, device="cuda")
    packed[512:512 + inner.numel()] = inner
    again = X.feed_forward_grad(dy, x, w_in, w_out, packed[512:512 + inner.numel()])
    assert all(torch.equal(a, b) for a, b in zip(want[1:], again))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(x, w_in, w_out, dy, "silu")
    for k in range(4):
        x.mul_(0.9)
        graph.replay()
        want = run(x, w_in, w_out, dy, "silu")
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got)), k
