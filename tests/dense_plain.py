"""The dense stage's operations from their definitions: the AdamW step and its
8-bit moments in float32 steps and in float64, products and blocks in float64."""

from __future__ import annotations

import numpy as np

F32 = np.float32
LEAST = F32(2.0 ** -100)
BLOCK = 256


def fma32(a, b, c):
    """a b + c rounded once to float32: the product of two of them is exact in
    float64, and its sum with a third, in 53 bits, is rounded once more; the two
    roundings differ from one in 2^-29 of all cases, which the callers allow for."""
    return (a.astype(np.float64) * b.astype(np.float64) + c.astype(np.float64)).astype(F32)


def blocks(flat):
    return np.concatenate([flat, np.zeros(-flat.size % BLOCK, flat.dtype)]).reshape(-1, BLOCK)


def put(values, steps, signed):
    """(codes, scales) of float32 values: steps sqrt(|value| / largest), rounded to even."""
    n, b = values.size, blocks(values)
    most = np.abs(b).max(axis=1)
    some = most >= LEAST
    unit = np.where(some, F32(1.0) / np.where(some, most, F32(1.0)), F32(0.0)).astype(F32)
    code = np.rint(F32(steps) * np.sqrt(np.abs(b) * unit[:, None])).astype(np.int64)
    if not signed:
        code = np.where((b > 0) & some[:, None], np.maximum(code, 1), code)
    return np.where(b < 0, -code, code).reshape(-1)[:n], np.where(some, most, F32(0.0))


def shown(code, scale, signed):
    """The float32 values that codes stand for."""
    n, c = code.size, blocks(code.astype(F32))
    unit = (scale * F32(1.0 / (16129.0 if signed else 65025.0))).astype(F32)[:, None]
    v = c * np.abs(c) * unit
    return (v if signed else v * v).reshape(-1)[:n]


def adamw32(p, g, m, v, step, lr, b1, b2, eps, decay):
    """(p, m, v) in float32, the operations in the step's order."""
    def toward(a, b, w):
        d = (b - a).astype(F32)
        return fma32(F32(w), d, a) if F32(w) < 0.5 else fma32(-d, F32(1.0) - F32(w), b)

    left = np.sqrt(1.0 - b2 ** step)
    m, v = toward(m, g, 1.0 - b1), toward(v, g * g, 1.0 - b2)
    move = m / (np.sqrt(v) + F32(eps * left))
    return fma32(F32(-(lr * left / (1.0 - b1 ** step))), move, p * F32(1.0 - lr * decay)), m, v


def adamw64(p, g, m, v, step, lr, b1, b2, eps, decay):
    m, v = b1 * m + (1.0 - b1) * g, b2 * v + (1.0 - b2) * g * g
    with np.errstate(divide="ignore", invalid="ignore"):
        move = (m / (1.0 - b1 ** step)) / (np.sqrt(v / (1.0 - b2 ** step)) + eps)
    return p * (1.0 - lr * decay) - lr * move, m, v


# ---------------------------------------------------------------------------
# the feed-forward block in float64, with bounds of every rounding on the way
# ---------------------------------------------------------------------------

U32 = 2.0 ** -24
UNIT = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
TINY = {"float32": 2.0 ** -149, "bfloat16": 2.0 ** -133, "float16": 2.0 ** -25}   # half the smallest step


def erf(x):
    from scipy.special import erf as f
    return f(x)


def activation(act, g):
    """(value, slope) of act at g, and bounds of what float32 makes of them: of
    each value's 8 roundings, of an exponential's argument, whose rounding counts
    as often as it is large, and 1.5e-7 of the handbook's erf (7.5e-8 of the
    distribution function)."""
    a = np.abs(g)
    with np.errstate(over="ignore"):
        if act == "relu":
            return np.maximum(g, 0.0), (g > 0) * 1.0, 0.0 * a, 0.0 * a
        if act == "gelu":
            p, d = 0.5 * (1 + erf(g / np.sqrt(2))), np.exp(-0.5 * g * g) / np.sqrt(2 * np.pi)
            ep = 8e-8 + (12 + g * g) * U32 * np.minimum(p, 1 - p) + 4 * U32
            return g * p, p + g * d, a * ep + U32 * a * p, ep + (8 + g * g) * U32 * a * d + 4 * U32 * (p + a * d)
        z = 2 * np.sqrt(2 / np.pi) * (g + 0.044715 * g ** 3) if act == "gelu_tanh" else g
        dz = 2 * np.sqrt(2 / np.pi) * (1 + 3 * 0.044715 * g * g) if act == "gelu_tanh" else 1.0
        s = 1 / (1 + np.exp(-z))
        t = 1 / (1 + np.exp(z))                                  # 1 - s, not rounded to 0
        es = (8 + 10 * np.abs(z)) * U32 * s
        rest = U32 + es                                          # of 1 - s in float32, near s = 1
        return g * s, s + g * s * t * dz, a * es + U32 * a * s, \
            es * (1 + a * dz) + a * s * dz * rest + 12 * U32 * (s + a * s * t * dz)


def feed(x, w_in, w_out, act, dtype, dy=None):
    """{name: (value, bound)} of y and, with dy, dx, dw_in and dw_out: sums of K
    terms in float32 in any order (K + 8 units of the magnitudes' sum), slopes of at
    most 1.13 and curvatures of at most 1.2, h and the inner gradients rounded to the type
    (h of 16 rows or fewer to two parts of it for y), one rounding of the result."""
    n, F = x.shape[0], w_out.shape[1]
    u, tiny = UNIT[dtype], TINY[dtype]
    gam = lambda terms: (terms + 8) * U32  # noqa: E731
    pre, epre = x @ w_in.T, gam(x.shape[1]) * (np.abs(x) @ np.abs(w_in).T)
    g, v, eg, ev = pre[:, :F], pre[:, F:], epre[:, :F], epre[:, F:]
    a, slope, ea, es = activation(act, g)
    ea = ea + 1.13 * eg
    es = es + (np.where(np.abs(g) <= eg, 1.0, 0.0) if act == "relu" else 1.2 * eg)
    h = a * v
    eh = 1.01 * (ea * np.abs(v) + np.abs(a) * ev + ea * ev) + 2 * U32 * np.abs(h)
    kept = eh + u * (np.abs(h) + eh) + tiny                       # h in the type
    used = eh + (u * u * (np.abs(h) + eh) + 2 * tiny if n <= 16 else u * (np.abs(h) + eh) + tiny)
    y, ey = h @ w_out.T, (used + gam(2 * F) * (np.abs(h) + used)) @ np.abs(w_out).T
    out = {"y": (y, ey + u * (np.abs(y) + ey) + tiny)}
    if dy is None:
        return out
    dh, edh = dy @ w_out, gam(dy.shape[1]) * (np.abs(dy) @ np.abs(w_out))
    dg, du = dh * v * slope, dh * a

    def rounded(value, e):
        return e + 4 * U32 * np.abs(value) + u * (np.abs(value) + e) + tiny

    edg = rounded(dg, 1.02 * (edh * np.abs(v * slope) + np.abs(dh) * ev * np.abs(slope) + np.abs(dh * v) * es
                              + np.abs(dh) * ev * es + edh * ev * es + edh * np.abs(v) * es + edh * ev * np.abs(slope)))
    edu = rounded(du, 1.02 * (edh * np.abs(a) + np.abs(dh) * ea + edh * ea))
    d, ed = np.concatenate([dg, du], 1), np.concatenate([edg, edu], 1)
    for name, (A, eA), (B, eB) in (("dx", (d, ed), (w_in, 0 * w_in)), ("dw_in", (d.T, ed.T), (x, 0 * x)),
                                   ("dw_out", (dy.T, 0 * dy.T), (h, kept))):
        value = A @ B
        e = eA @ (np.abs(B) + eB) + np.abs(A) @ eB + gam(A.shape[1]) * ((np.abs(A) + eA) @ (np.abs(B) + eB))
        out[name] = (value, e + u * (np.abs(value) + e) + tiny)
    return out


def codes(x):
    """(codes, scales) of rows, in float32 as the definition has it."""
    x = x.astype(F32)
    most = np.abs(x).max(axis=1)
    finite = np.isfinite(most)
    some = finite & (most >= LEAST)
    safe = np.where(some, most, F32(1.0)).astype(F32)
    unit = np.where(some, F32(127.0) / safe, F32(0.0)).astype(F32)
    with np.errstate(invalid="ignore"):
        q = np.where(some[:, None], np.clip(np.rint(np.where(some[:, None], x, 0) * unit[:, None]), -127, 127), 0)
    scale = np.where(some, safe * F32(1.0 / 127.0), F32(0.0)).astype(F32)
    return q.astype(np.int64), np.where(finite, scale, F32(np.nan)).astype(F32)


def product8(a, sa, b, sb):
    """float32, rounded as the definition has it."""
    whole = (a.astype(np.float64) @ b.astype(np.float64).T).astype(np.int64)       # sums below 2^53
    return (whole.astype(F32) * sb[None, :]).astype(F32) * sa[:, None]


def feed8(x, w_in, si, w_out, so, act):
    """(y, bound) in float64: g, u and h within a few units of float32, a code of h
    off by one where that may move it over a border."""
    q, sx = codes(x)
    F = w_out.shape[1]
    pre = (q.astype(np.float64) @ w_in.astype(np.float64).T) * si.astype(np.float64) * sx.astype(np.float64)[:, None]
    g, v = pre[:, :F], pre[:, F:]
    a, _, ea, _ = activation(act, g)
    h = a * v
    eh = (ea + 1.13 * 4 * U32 * np.abs(g)) * np.abs(v) + 8 * U32 * np.abs(h)
    most = np.abs(h).max(axis=1, keepdims=True)
    at, slack = 127.0 * h / most, 127.0 * (eh + np.abs(h) / most * eh.max(axis=1, keepdims=True)) / most + 1e-4
    border = np.abs(np.abs(at - np.floor(at)) - 0.5) <= slack
    y = (np.rint(at) @ w_out.astype(np.float64).T) * so * most / 127.0
    e = (border @ np.abs(w_out.astype(np.float64)).T) * so * most / 127.0
    return y, e + 1e-5 * ((np.abs(at) @ np.abs(w_out.astype(np.float64)).T) * so * most / 127.0)
