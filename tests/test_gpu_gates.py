"""The gates' factors of 16-bit types and of the 8-bit block, relative to themselves:
far out on the negative side the whole factor is a tail, which a bound of the
distribution function's absolute error leaves free."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from yabt_amd import feed_ops as X

from dense_plain import product8

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24


def tail(act, g):
    """act(g) and its slope in float64 without cancellation, and what float32 may make of act(g), relative.

    gelu: 18 units of U32 for the approximation, its arguments and the products, and 1.5 g^2 for
    the exponential's argument, rounded twice, times a rounded constant.  The others: s = 1 / (1 + exp(-z)), z of
    up to 7 roundings (none for silu), the exponential's argument of 2: 10 |z| and 8."""
    from scipy.special import ndtr
    if act == "gelu":
        p, d = ndtr(g), np.exp(-0.5 * g * g) / np.sqrt(2 * np.pi)
        return g * p, p + g * d, (20 + 2 * g * g) * U32
    c = np.sqrt(8 / np.pi)
    z, dz = (c * (g + 0.044715 * g ** 3), c * (1 + 3 * 0.044715 * g * g)) if act == "gelu_tanh" else (g, 1.0)
    s, t = 1 / (1 + np.exp(-z)), 1 / (1 + np.exp(z))
    return g * s, s + g * s * t * dz, (8 + 10 * np.abs(z)) * U32


@pytest.mark.parametrize("act,least", [("silu", -60.0), ("gelu", -11.0), ("gelu_tanh", -8.0)])
@pytest.mark.parametrize("n", [50, 3000])
def test_gates_in_8_bits(n, act, least):
    """One inner column: its code is 127 throughout, so that y is h but for a few units.  Gates from the
    stated least to -0.01 and their opposites; h stays above 2^-100."""
    x = torch.cat([torch.linspace(least, -0.01, n // 2), torch.linspace(0.01, -least, n - n // 2)])[:, None]
    w_in, s_in = torch.tensor([[127], [-127]], dtype=torch.int8), torch.full((2,), 1 / 127.0)
    w_out, s_out = torch.full((1, 1), 127, dtype=torch.int8), torch.full((1,), 1 / 127.0)
    y = X.feed_forward_int8(x.cuda(), *(t.cuda() for t in (w_in, s_in, w_out, s_out)), activation=act)
    q, sx = (t.numpy() for t in (torch.sign(x).to(torch.int8) * 127, (x.abs()[:, 0] * np.float32(1 / 127.0))))
    pre = product8(q, sx, w_in.numpy(), s_in.numpy()).astype(np.float64)
    g, u = pre[:, 0], pre[:, 1]
    value, _, off = tail(act, g)
    want = value * u
    # the gate times its factor, times u, the row's scale, y's three products and 1 / 127: 10 units more
    rel = np.abs(y[:, 0].double().cpu().numpy() / want - 1)
    assert np.all(rel <= off + 10 * U32), (g[np.argmax(rel / (off + 10 * U32))], rel.max())


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("act,least", [("silu", -60.0), ("gelu", -10.0), ("gelu_tanh", -7.0)])
@pytest.mark.parametrize("n", [50, 700])
def test_gates_and_slopes_in_16_bits(n, act, least, dt):
    """Rounded once as h and once as y, or as dg and dx, where these are normal numbers of the type."""
    g = torch.linspace(least, -2.0, n).to(dt)
    big = 2.0 ** 12 if dt == torch.float16 else 1.0              # u, which keeps small factors in the type's range
    x = torch.stack([g, torch.full((n,), big, dtype=dt)], 1).cuda()
    w_in, w_out = torch.eye(2, dtype=dt, device="cuda"), torch.ones((1, 1), dtype=dt, device="cuda")
    y, inner = X.feed_forward(x, w_in, w_out, activation=act, keep_inner=True)
    dx = X.feed_forward_grad(torch.ones((n, 1), dtype=dt, device="cuda"), x, w_in, w_out, inner, activation=act)[0]
    value, slope, off = tail(act, g.double().numpy())
    unit, normal = torch.finfo(dt).eps / 2, torch.finfo(dt).tiny
    # a slope has two parts, each as far off as the factor and a few units, whose magnitudes add up to
    # 3.7 times the slope's at most from -2 on (silu at -2; the others 1.6)
    for got, want, more in ((y[:, 0], value * big, off + 4 * U32), (dx[:, 0], slope * big, 4 * off + 16 * U32)):
        there = np.abs(want) >= normal
        rel = np.abs(got.double().cpu().numpy()[there] / want[there] - 1)
        assert there.sum() > n // 8 and np.all(rel <= 2.01 * unit + more[there]), (rel / unit).max()
