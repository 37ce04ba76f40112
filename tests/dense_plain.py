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
