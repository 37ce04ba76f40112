"""An infinite input of a 16-bit block gives the infinities that the formulas give,
also where h and the inner gradients are taken in two parts."""

from __future__ import annotations

import pytest
import torch

from yabt_amd import feed_ops as X

pytestmark = pytest.mark.gpu


def plain(x, w_in, w_out, dy):
    x, w_in, w_out, dy = (t.double().cpu() for t in (x, w_in, w_out, dy))
    g, u = (x @ w_in.t()).chunk(2, dim=1)
    a, slope = g.clamp_min(0.0), (g > 0).double()
    h, dh = a * u, dy @ w_out
    d = torch.cat([dh * u * slope, dh * a], dim=1)
    return h @ w_out.t(), d @ w_in, d.t() @ x, dy.t() @ h


# one row, 16 or fewer, small blocks of more and of more than 64, and blocks that are not small
@pytest.mark.parametrize("n", [1, 5, 16, 20, 40, 90, 700])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=str)
def test_infinite_inputs(n, dt):
    gen = torch.Generator().manual_seed(n)
    D, F, O = (24, 40, 32) if n < 100 else (64, 64, 64)
    x, dy = torch.randn((n, D), generator=gen), torch.rand((n, O), generator=gen) + 0.1
    w_in, w_out = torch.randn((2 * F, D), generator=gen), torch.rand((O, F), generator=gen) + 0.1
    w_in[:F, 3] = w_in[:F, 3].abs() + 0.1                 # every gate of the row is +infinite
    x[n // 2, 3] = float("inf")
    x, dy, w_in, w_out = (t.to(dt).cuda() for t in (x, dy, w_in, w_out))
    w_in[F:, 3] = w_in[F:, 3].abs() + 0.125 if n % 2 else -(w_in[F:, 3].abs() + 0.125)
    y, inner = X.feed_forward(x, w_in, w_out, activation="relu", keep_inner=True)
    got = (y,) + tuple(X.feed_forward_grad(dy, x, w_in, w_out, inner, activation="relu"))
    want = plain(x, w_in, w_out, dy)
    assert bool(torch.isinf(want[0][n // 2]).all()) and bool(torch.isinf(want[3]).all())
    for m, a, b in zip(("y", "dx", "dw_in", "dw_out"), got, want):
        a, far = a.double().cpu(), torch.isinf(b)
        if m == "dw_in" and n < 100:                      # two parts of dg and du times an infinite x: documented as NaN
            a, b, far = (torch.cat([t[:, :3], t[:, 4:]], 1) for t in (a, b, far))
        assert torch.equal(a[far], b[far]), m
        assert bool(torch.isfinite(a[torch.isfinite(b)]).all()), m
