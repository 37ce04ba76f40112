"""The expert layer's operations in float64, row by row from their definitions."""

from __future__ import annotations

import numpy as np

U32 = 2.0 ** -24                                   # unit roundoff of float32 ...
UNIT = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
TINY = {"float32": 2.0 ** -149, "bfloat16": 2.0 ** -133, "float16": 2.0 ** -25}   # half the smallest step


def norm(x, w, b, eps):
    mean = x.mean(axis=1)
    xc = x - mean[:, None]
    rstd = 1.0 / np.sqrt((xc * xc).mean(axis=1) + eps)
    y = xc * rstd[:, None]
    return (y if w is None else y * w) + (0.0 if b is None else b), mean, rstd


def norm_grad(dy, x, mean, rstd, w):
    t = dy if w is None else dy * w
    xh = (x - mean[:, None]) * rstd[:, None]
    dx = rstd[:, None] * (t - t.mean(axis=1, keepdims=True) - xh * (t * xh).mean(axis=1, keepdims=True))
    return dx, (dy * xh).sum(axis=0), dy.sum(axis=0)


def scores_of(row, scores):
    """p of one row in float64; closed experts have 0."""
    is_open = row > -np.inf
    if scores == "sigmoid":
        with np.errstate(over="ignore"):
            return np.where(is_open, 1.0 / (1.0 + np.exp(-np.where(is_open, row, 0.0))), 0.0)
    p = np.zeros(row.shape)
    if is_open.any():
        e = np.exp(row[is_open] - row[is_open].max())
        p[is_open] = e / e.sum()
    return p


def choose(row, k, scores, bias, groups, keep):
    """The ids of one row, keys in float32."""
    is_open = row > -np.inf
    key = (scores_of(row, scores) if scores == "sigmoid" else row).astype(np.float32)
    if bias is not None:
        key = (key + bias.astype(np.float32)).astype(np.float32)
    key = np.where(is_open, key, -np.inf).astype(np.float64)
    size = len(row) // groups
    if keep < groups:
        best = []
        for g in range(groups):
            part = sorted((v for v in key[g * size:(g + 1) * size] if v > -np.inf), reverse=True)
            part = part[:1] if scores == "softmax" else part[:2]
            best.append((-float(np.float32(sum(part))) if part else np.inf, g))
        kept = {g for _, g in sorted(best)[:keep]}
        key = np.array([v if i // size in kept else -np.inf for i, v in enumerate(key)])
    order = [i for _, i in sorted((-v, i) for i, v in enumerate(key) if v > -np.inf)][:k]
    return order + [-1] * (k - len(order))


def weights_of(row, ids, scores, renormalise, scale):
    p = scores_of(row, scores)
    w = np.array([p[i] if i >= 0 else 0.0 for i in ids])
    if renormalise:
        if scores == "softmax":                    # over the chosen alone, so that none underflows
            on = [i for i in ids if i >= 0]
            if on:
                e = np.exp(row[on] - row[on].max())
                w[[j for j, i in enumerate(ids) if i >= 0]] = e
        w = w / w.sum() if w.sum() > 0 else w
    return scale * w


def weights_grad(row, ids, dw, scores, renormalise, scale):
    p, d = scores_of(row, scores), np.zeros(row.shape)
    w = weights_of(row, ids, scores, renormalise, 1.0)
    dw = scale * np.where(np.array(ids) >= 0, dw, 0.0)
    mean = (w * dw).sum()
    total = sum(p[i] for i in ids if i >= 0)
    for j, i in enumerate(ids):
        if i < 0:
            continue
        if scores == "softmax":
            d[i] += w[j] * (dw[j] - mean if renormalise else dw[j])
        else:
            d[i] += ((dw[j] - mean) / total if renormalise and total > 0 else 0.0 if renormalise else dw[j]) * p[i] * (1.0 - p[i])
    return d - p * mean if scores == "softmax" and not renormalise else d


def plan(ids, experts):
    flat = ids.reshape(-1)
    slots = [s for e in range(experts) for s in np.nonzero(flat == e)[0]]
    offsets = np.concatenate([[0], np.cumsum([(flat == e).sum() for e in range(experts)])])
    rest = [-1] * (flat.size - len(slots))
    return offsets, np.array(slots + rest, np.int64), np.array([s // ids.shape[1] for s in slots] + rest, np.int64)



def products(x, ids, w, w_in, w_out, dtype, dy=None, mask=None):
    """{name: (value, bound)} of the experts' products and, with dy, of their
    gradients, float64; the bounds carry every rounding of the way: sums of K
    terms in float32 in any order (K + 8 units of the magnitudes' sum), h, w h,
    dg and du to the inputs' type, the exponential and reciprocal (8 + 2 |g|
    units), one rounding of the result."""
    (n, D), k, E, F = x.shape, ids.shape[1], w_in.shape[0], w_out.shape[2]
    u, tiny = UNIT[dtype], TINY[dtype]
    gam = lambda terms: (terms + 8) * U32  # noqa: E731
    out = {name: np.zeros(shape) for name, shape in (("y", (n, D)), ("dx", (n, D)), ("dweights", (n, k)),
                                                     ("dw_in", w_in.shape), ("dw_out", w_out.shape))}
    err, size = {m: np.zeros(v.shape) for m, v in out.items()}, {m: np.zeros(v.shape) for m, v in out.items()}
    for e in range(E):
        t, j = np.nonzero(ids == e)
        if not len(t):
            continue
        xe, we, A, B = x[t], w[t, j][:, None], w_in[e], w_out[e]
        pre, epre = xe @ A.T, gam(D) * (np.abs(xe) @ np.abs(A).T)
        g, v, eg, ev = pre[:, :F], pre[:, F:], epre[:, :F], epre[:, F:]
        sig = 1.0 / (1.0 + np.exp(-g))
        silu, unit = g * sig, (8 + 2 * np.abs(g)) * U32
        esilu = 1.1 * eg + unit * np.abs(silu)
        h = silu * v
        eh = esilu * np.abs(v) + np.abs(silu) * ev + 2 * U32 * np.abs(h)
        eh16 = eh + u * (np.abs(h) + eh) + tiny
        z = h @ B.T
        ez = eh16 @ np.abs(B).T + gam(F) * (np.abs(h) @ np.abs(B).T)
        np.add.at(out["y"], t, we * z)
        np.add.at(err["y"], t, we * ez)
        np.add.at(size["y"], t, np.abs(we * z))
        if dy is None:
            continue
        de = dy[t]
        a, ea = de @ B, gam(D) * (np.abs(de) @ np.abs(B))
        out["dweights"][t, j] = (a * h).sum(axis=1)
        err["dweights"][t, j] = (np.abs(a) * eh + np.abs(h) * ea).sum(axis=1) + gam(F) * np.abs(a * h).sum(axis=1)
        slope = sig * (1.0 + g * (1.0 - sig))
        du, dg = we * a * silu, we * a * v * slope
        edu = np.abs(we) * (np.abs(silu) * ea + np.abs(a) * esilu)
        edg = np.abs(we) * (np.abs(v * slope) * ea + np.abs(a * slope) * ev
                            + np.abs(a * v) * (0.5 * eg + 1.5 * unit))
        dpre, edpre = np.concatenate([dg, du], 1), np.concatenate([edg, edu], 1)
        edpre = edpre + 4 * U32 * np.abs(dpre)
        edpre = edpre + u * (np.abs(dpre) + edpre) + tiny
        np.add.at(out["dx"], t, dpre @ A)
        np.add.at(err["dx"], t, edpre @ np.abs(A) + gam(2 * F) * (np.abs(dpre) @ np.abs(A)))
        np.add.at(size["dx"], t, np.abs(dpre @ A))
        out["dw_in"][e] = dpre.T @ xe
        err["dw_in"][e] = edpre.T @ np.abs(xe) + gam(len(t)) * (np.abs(dpre).T @ np.abs(xe))
        hw = we * h
        ehw = np.abs(we) * eh + U32 * np.abs(hw)
        ehw = ehw + u * (np.abs(hw) + ehw) + tiny
        out["dw_out"][e] = de.T @ hw
        err["dw_out"][e] = np.abs(de).T @ ehw + gam(len(t)) * (np.abs(de).T @ np.abs(hw))
    for m in ("y", "dx"):
        err[m] = err[m] + (k + 2) * U32 * size[m]
    names = ("y",) if dy is None else tuple(out)
    last = {m: U32 if m == "dweights" else u for m in names}
    return {m: (out[m], err[m] + last[m] * (np.abs(out[m]) + err[m]) + (0.0 if m == "dweights" else tiny) + 1e-38)
            for m in names}
