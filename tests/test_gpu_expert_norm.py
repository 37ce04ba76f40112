"""yabt_layer_norm and its gradient against the formulas in float64.

Bounds: a lane adds at most 16 values one after the other, then at most 10
pairwise steps and 16 waves, so a row's sums are off by fewer than 64 rounding
units of the sum of magnitudes; what follows is a handful of roundings; then
one rounding to the output's type."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from yabt_amd import expert_ops as X

from expert_plain import TINY, U32, UNIT, norm, norm_grad

pytestmark = pytest.mark.gpu

EPS = 1e-5
TYPES = [torch.float32, torch.bfloat16, torch.float16]
# widths around the values of a 16-byte access, the lanes' limits and past the registers'
WIDTHS = [1, 2, 3, 7, 8, 9, 31, 63, 65, 100, 127, 500, 513, 1023, 2049, 4096, 5001, 8193, 16385]


def name(dt):
    return str(dt).replace("torch.", "")


def inputs(n, D, dt, seed, offset=0.3):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn((n, D), generator=gen) * 1.5 + offset).to(dt)
    dy = torch.randn((n, D), generator=gen).to(dt)
    w, b = 1.0 + 0.2 * torch.randn(D, generator=gen), 0.3 * torch.randn(D, generator=gen)
    return x, dy, w, b


def check_forward(x, w, b, out, eps=EPS):
    y, mean, rstd = (t.double().cpu().numpy() for t in out)
    dt = name(x.dtype)
    xd = x.double().cpu().numpy()
    wd, bd = (None if t is None else t.double().numpy() for t in (w, b))
    ry, rm, rr = norm(xd, wd, bd, eps)
    size = np.abs(xd).mean(axis=1)
    assert np.all(np.abs(mean - rm) <= 64 * U32 * size + 1e-38)
    # the mean's error shifts every centred value; the variance's is that of its sum
    shift = 64 * U32 * (size * rr)
    assert np.all(np.abs(rstd - rr) <= rr * (100 * U32 + 2 * shift + shift * shift))
    xh = np.abs(xd - rm[:, None]) * rr[:, None]
    tol = (shift[:, None] + (110 * U32 + 2 * shift + shift * shift)[:, None] * xh + 2 * U32 * np.abs(xd) * rr[:, None])
    tol = tol * (1.0 if wd is None else np.abs(wd)) + 4 * U32 * (np.abs(ry) + (0.0 if bd is None else np.abs(bd)))
    assert np.all(np.abs(y - ry) <= tol * 1.01 + UNIT[dt] * np.abs(ry) + TINY[dt])


def check_backward(x, dy, mean, rstd, w, out):
    dx, dw, db = (t.double().cpu().numpy() for t in out)
    n, D = x.shape
    dt = name(x.dtype)
    xd, gd = x.double().cpu().numpy(), dy.double().cpu().numpy()
    md, rd = mean.double().cpu().numpy(), rstd.double().cpu().numpy()
    wd = None if w is None else w.double().numpy()
    rx, rw, rb = norm_grad(gd, xd, md, rd, wd)
    t = np.abs(gd if wd is None else gd * wd)
    # |x| and |mean| may cancel in xh
    xh = (np.abs(xd) + np.abs(md)[:, None]) * rd[:, None]
    tol = 80 * U32 * rd[:, None] * (t + t.mean(axis=1, keepdims=True) + xh * (t * xh).mean(axis=1, keepdims=True))
    assert np.all(np.abs(dx - rx) <= tol + UNIT[dt] * np.abs(rx) + TINY[dt])
    chain = (n + 64) * U32                            # at worst one row after the other
    assert np.all(np.abs(dw - rw) <= chain * (np.abs(gd) * xh).sum(axis=0) + 1e-38)
    assert np.all(np.abs(db - rb) <= chain * np.abs(gd).sum(axis=0) + 1e-38)


@pytest.mark.parametrize("dt", TYPES, ids=name)
@pytest.mark.parametrize("D", WIDTHS)
def test_norm_and_gradient(D, dt):
    for n in (1, 5, 130) if D < 4000 else (1, 67):
        print(f"layer_norm n={n} D={D} {name(dt)}", flush=True)
        x, dy, w, b = inputs(n, D, dt, D + n)
        xg, dyg, wg, bg = (t.cuda() for t in (x, dy, w, b))
        out = X.layer_norm(xg, wg, bg, eps=EPS)
        check_forward(x, w, b, out)
        back = X.layer_norm_grad(dyg, xg, out[1], out[2], wg)
        check_backward(x, dy, out[1], out[2], w, back)
        again = X.layer_norm_grad(dyg, xg, out[1], out[2], wg)
        assert all(torch.equal(a, c) for a, c in zip(back, again))


@pytest.mark.parametrize("dt", TYPES, ids=name)
@pytest.mark.parametrize("n,D", [(4097, 20), (70_001, 28), (9_000, 500), (3_000, 1001), (2_500, 4096)])
def test_many_rows(n, D, dt):
    """More rows than blocks: the gradient's parts are added over all of them."""
    x, dy, w, b = inputs(n, D, dt, n)
    out = X.layer_norm(x.cuda(), w.cuda(), b.cuda(), eps=EPS)
    check_forward(x, w, b, out)
    check_backward(x, dy, out[1], out[2], w, X.layer_norm_grad(dy.cuda(), x.cuda(), out[1], out[2], w.cuda()))


@pytest.mark.parametrize("dt", TYPES, ids=name)
def test_strides_and_missing_parameters(dt):
    """Rows inside a wider matrix, at odd starts; transposed inputs; no weight, no bias."""
    for D, wide, start in [(100, 131, 3), (9, 11, 1), (513, 520, 7)]:
        x, dy, w, b = inputs(37, wide, dt, D)
        xv, dv = x[:, start:start + D], dy[:, start:start + D]
        wv, bv = w[:D], b[:D]
        xg, dg = x.cuda()[:, start:start + D], dy.cuda()[:, start:start + D]
        out = X.layer_norm(xg, None, bv.cuda())
        check_forward(xv, None, bv, out)
        out = X.layer_norm(xg, wv.cuda(), None)
        check_forward(xv, wv, None, out)
        check_backward(xv, dv, out[1], out[2], wv, X.layer_norm_grad(dg, xg, out[1], out[2], wv.cuda()))
        check_backward(xv, dv, out[1], out[2], None, X.layer_norm_grad(dg, xg, out[1], out[2]))
        turned = X.layer_norm(xg.t().contiguous().t(), wv.cuda(), None)
        assert all(torch.equal(a, c) for a, c in zip(out, turned))
        odd = torch.stack([wv, bv], 1).cuda()
        assert torch.equal(X.layer_norm(xg, odd[:, 0], odd[:, 1].to(torch.float64))[0],
                           X.layer_norm(xg, wv.cuda(), bv.cuda())[0])


def test_constant_rows_and_far_means():
    """A constant row has variance 0: y is the bias, dx finite.  A mean far from
    zero costs only what its rounding does (the variance is of centred values)."""
    x = torch.full((3, 257), 7.25)
    w, b = torch.rand(257) + 0.5, torch.randn(257)
    y, mean, rstd = X.layer_norm(x.cuda(), w.cuda(), b.cuda())
    assert torch.equal(y.cpu(), b.expand(3, 257)) and torch.equal(mean.cpu(), x[:, 0])
    assert torch.allclose(rstd.cpu(), torch.full((3,), float(np.float32(1e-5)) ** -0.5), rtol=1e-6)
    dx, dw, db = X.layer_norm_grad(torch.ones_like(x).cuda(), x.cuda(), mean, rstd, w.cuda())
    assert torch.isfinite(dx).all() and torch.equal(dw.cpu(), torch.zeros(257)) and torch.equal(db.cpu(), torch.full((257,), 3.0))
    x, dy, w, b = inputs(8, 1000, torch.float32, 1, offset=1000.0)
    check_forward(x, w, b, X.layer_norm(x.cuda(), w.cuda(), b.cuda()))


def test_rows_with_nan_and_infinity_stay_in_their_rows():
    x, dy, w, b = inputs(64, 96, torch.float32, 3)
    bad = x.clone()
    bad[5, 7], bad[20, 0], bad[41, 95] = float("nan"), float("inf"), float("-inf")
    good = [r for r in range(64) if r not in (5, 20, 41)]
    want, got = X.layer_norm(x.cuda(), w.cuda(), b.cuda()), X.layer_norm(bad.cuda(), w.cuda(), b.cuda())
    for a, c in zip(want, got):
        assert torch.equal(a[good], c[good]) and not torch.isfinite(c[[5, 20, 41]]).reshape(3, -1).all(1).any()


def test_gradient_against_differences():
    """The directional derivative of sum(c y) by central differences of the
    float64 formula, and by the gradients."""
    x, dy, w, b = inputs(23, 150, torch.float32, 9)
    rng = np.random.default_rng(0)
    xd, gd, wd, bd = (t.double().numpy() for t in (x, dy, w, b))
    vx, vw, vb = rng.normal(size=xd.shape), rng.normal(size=wd.shape), rng.normal(size=bd.shape)
    h = 1e-5
    up = (norm(xd + h * vx, wd + h * vw, bd + h * vb, EPS)[0] * gd).sum()
    down = (norm(xd - h * vx, wd - h * vw, bd - h * vb, EPS)[0] * gd).sum()
    _, mean, rstd = X.layer_norm(x.cuda(), w.cuda(), b.cuda(), eps=EPS)
    dx, dw, db = (t.double().cpu().numpy() for t in X.layer_norm_grad(dy.cuda(), x.cuda(), mean, rstd, w.cuda()))
    slope = (dx * vx).sum() + (dw * vw).sum() + (db * vb).sum()
    size = np.sqrt((dx ** 2).sum() + (dw ** 2).sum() + (db ** 2).sum())
    # h^2 times a third derivative of order one, and float32 gradients
    assert abs(slope - (up - down) / (2 * h)) <= 1e-5 * size


def test_no_rows():
    e = torch.empty((0, 12), device="cuda")
    y, mean, rstd = X.layer_norm(e)
    assert y.shape == (0, 12) and mean.shape == (0,) and rstd.shape == (0,)
    dx, dw, db = X.layer_norm_grad(e, e, mean, rstd)
    assert dx.shape == (0, 12) and torch.equal(dw, torch.zeros(12, device="cuda")) and torch.equal(db, dw)


def test_refusals():
    x = torch.zeros((4, 8), device="cuda")
    s = torch.zeros(4, device="cuda")
    for call in (lambda: X.layer_norm(x[0]), lambda: X.layer_norm(x.double()), lambda: X.layer_norm(x[:, :0]),
                 lambda: X.layer_norm(x, torch.zeros(7, device="cuda")), lambda: X.layer_norm(x, None, torch.zeros(8)),
                 lambda: X.layer_norm_grad(x[:3], x, s, s), lambda: X.layer_norm_grad(x.half(), x, s, s),
                 lambda: X.layer_norm_grad(x, x, s[:2], s), lambda: X.layer_norm_grad(x, x, None, s)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError, match="HIP device"):
        X.layer_norm(x.cpu())
    with pytest.raises(RuntimeError, match="bad sizes"):
        X.layer_norm(x, eps=-1.0)
