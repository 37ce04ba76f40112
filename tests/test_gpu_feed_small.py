"""Float32 values near the type's end: the block of more than 64 rows takes each to
2^-133, that of fewer in full, and never loses one that is larger."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from yabt_amd import feed_ops as X

pytestmark = pytest.mark.gpu

U32, STEP, LEAST = 2.0 ** -24, 2.0 ** -133, 2.0 ** -149


@pytest.mark.parametrize("n", [40, 200])
@pytest.mark.parametrize("power", [90, 105, 110, 112, 116, 120, 124, 126])
def test_small_inputs_and_their_gradients(n, power):
    """relu, whose value and slope are exact.  A sum of K terms is off by K + 8 units of the magnitudes' sum
    and by a step of each term's small factor, once a part: three steps and the sum's own least values."""
    gen = torch.Generator().manual_seed(power)
    D, F, O = 64, 48, 56
    small, large = 2.0 ** -power, 2.0 ** min(power, 119)
    x, w_out = torch.randn((n, D), generator=gen) * small, torch.randn((O, F), generator=gen) / 8
    w_in = torch.randn((2 * F, D), generator=gen) / 8
    w_in[F:] *= large                                            # so that u is near 1, and h as small as x
    dy = torch.randn((n, O), generator=gen) * small
    y, inner = X.feed_forward(*(t.cuda() for t in (x, w_in, w_out)), activation="relu", keep_inner=True)
    dx, dw_in, dw_out = X.feed_forward_grad(*(t.cuda() for t in (dy, x, w_in, w_out)), inner, activation="relu")
    x, w_in, w_out, dy = (t.double().numpy() for t in (x, w_in, w_out, dy))
    step = STEP if n > 64 else LEAST

    def product(a, ea, b, eb, step):
        """a b and its bound, a's values being small: off by ea and a step each."""
        K = a.shape[1]
        size = (np.abs(a) + ea) @ (np.abs(b) + eb)
        return a @ b, (ea + 3 * step) @ (np.abs(b) + eb) + np.abs(a) @ eb + (K + 8) * U32 * size + 8 * K * LEAST

    none = np.zeros(())
    g, eg = product(x, 0 * x, w_in[:F].T, 0 * w_in[:F].T, step)
    u, eu = product(x, 0 * x, w_in[F:].T, 0 * w_in[F:].T, step)
    on, sure = g > 0, np.abs(g) > eg
    a = np.where(on, g, none)
    h = a * u
    eh = eg * np.abs(u) + np.abs(a) * eu + eg * eu + 2 * U32 * np.abs(h) + LEAST
    want, bound = product(h, eh, w_out.T, 0 * w_out.T, step)
    off = np.abs(y.double().cpu().numpy() - want)
    assert np.all(off <= bound), np.max(off / bound)
    # the gradients go by tiles whatever n; du = dh act(g) is beyond the type where both are small
    dh, edh = product(dy, 0 * dy, w_out, 0 * w_out, STEP)
    dg = np.where(on, dh * u, none)
    edg = edh * np.abs(u) + np.abs(dh) * eu + edh * eu + 2 * U32 * np.abs(dg) + LEAST + np.where(sure, 0.0, np.abs(dh * u))
    got = dw_in[:F].double().cpu().numpy()
    # dg times x is beyond the type: 0, but for what is left of it
    assert np.all(np.abs(got) <= n * (np.abs(dg).max() + edg.max()) * np.abs(x).max() * 2 + 8 * n * LEAST)
    # of dx the gate's part: u's rows of w_in are large and du, a product of two small values, ends at LEAST
    du, edu = dh * a, edh * a + np.abs(dh) * eg + edh * eg + 2 * U32 * np.abs(dh * a) + LEAST
    part, e1 = product(dg, edg, w_in[:F], 0 * w_in[:F], STEP)
    rest, e2 = product(du, edu, w_in[F:], 0 * w_in[F:], STEP)
    off = np.abs(dx.double().cpu().numpy() - part - rest)
    assert np.all(off <= e1 + e2), np.max(off / (e1 + e2))
    assert bool(torch.isfinite(dw_out).all()) and bool(torch.isfinite(dw_in).all())


def test_small_weights():
    gen = torch.Generator().manual_seed(1)
    n, D, F, O = 300, 32, 40, 24
    x, w_in = torch.randn((n, D), generator=gen), torch.randn((2 * F, D), generator=gen)
    w_out = torch.randn((O, F), generator=gen) * 2.0 ** -120
    y = X.feed_forward(*(t.cuda() for t in (x, w_in, w_out)), activation="relu").double().cpu().numpy()
    x, w_in, w_out = (t.double().numpy() for t in (x, w_in, w_out))
    g, u = np.split(x @ w_in.T, 2, axis=1)
    h = np.maximum(g, 0) * u
    size = np.maximum(np.abs(x) @ np.abs(w_in[:F]).T, 0) * (np.abs(x) @ np.abs(w_in[F:]).T)
    bound = (np.abs(h) + 3 * 48 * U32 * size) @ (np.full_like(w_out, 3 * STEP).T) \
        + ((3 * 48 + F + 8) * U32 * size) @ np.abs(w_out).T + 8 * F * LEAST
    assert np.all(np.abs(y - h @ w_out.T) <= bound)
