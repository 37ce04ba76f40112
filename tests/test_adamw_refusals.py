"""What an AdamW step refuses, without a device; and its plain form against
differences of the quantity that it minimises in one step."""

import ctypes

import numpy as np
import pytest
import torch

from yabt_amd import _lib, optim

from dense_plain import put, shown


def refused(rc, text):
    assert rc < 0 and text in _lib.last_error(), (rc, _lib.last_error())


def words(n=4, p=16, g=16, m=16, v=16, sm=16, sv=16, pt=0, gt=0):
    return (ctypes.c_int64 * 8)(p, g, m, v, sm, sv, n, pt | gt << 32)


def test_c_entry():
    lib = _lib.load()

    def step(table=None, count=1, bits=32, t=1, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, decay=0.0):
        return lib.yabt_adamw_step(count, words() if table is None else table, bits, t, None, lr, b1, b2, eps, decay, None)

    for args, text in [(dict(bits=16), "32 or 8"), (dict(t=0), "bad sizes"), (dict(t=2 ** 31), "bad sizes"),
                       (dict(count=-1), "bad sizes"), (dict(lr=-1.0), "0 or more"), (dict(lr=float("nan")), "0 or more"),
                       (dict(b1=1.0), "0 or more"), (dict(b2=-0.1), "0 or more"), (dict(eps=-1.0), "0 or more"),
                       (dict(decay=float("inf")), "0 or more"), (dict(table=words(pt=3)), "dtype"),
                       (dict(table=words(gt=-1)), "dtype"), (dict(table=words(n=-1)), "bad sizes"),
                       (dict(table=words(n=1 << 40)), "bad sizes"), (dict(table=words(p=0)), "null pointer"),
                       (dict(table=words(g=0)), "null pointer"), (dict(table=words(sm=0), bits=8), "null pointer")]:
        refused(step(**args), text)
    assert step(count=0) == 0
    assert step(table=words(n=0, p=0, g=0, m=0, v=0)) == 0
    refused(lib.yabt_adamw_values(1, words(sv=0), None), "null pointer")
    refused(lib.yabt_adamw_values(-1, words(), None), "bad sizes")
    refused(lib.yabt_adamw_values(1, None, None), "null pointer")
    assert lib.yabt_adamw_values(0, None, None) == 0


def test_python_entry():
    p = [torch.zeros(300)]
    g = [torch.zeros(300)]
    with pytest.raises(ValueError, match="bits"):
        optim.adamw_state(p, bits=16)
    s = optim.adamw_state(p)
    with pytest.raises(RuntimeError, match="HIP device"):
        optim.adamw_step(p, g, s, 1)
    with pytest.raises(ValueError, match="parameters"):
        optim.adamw_step(p, [], s, 1)
    for how in (dict(lr=-1.0), dict(lr=float("nan")), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1e-8),
                dict(weight_decay=-0.1)):
        with pytest.raises(ValueError, match="betas"):
            optim.adamw_step(p, g, s, 1, **how)
    with pytest.raises(ValueError, match="both scales"):
        optim.adamw_step(p, g, optim.AdamWState(s.first, s.second, [torch.zeros(2)]), 1)
    with pytest.raises(ValueError, match="both scales"):
        optim.adamw_step(p, g, optim.AdamWState(s.first, []), 1)
    with pytest.raises(ValueError, match="first moment 0"):
        optim.adamw_step(p, g, optim.AdamWState([torch.zeros(300, dtype=torch.float64)], s.second), 1)
    e = optim.adamw_state(p, bits=8)
    assert e.bits == 8 and e.first[0].dtype == torch.int8 and e.second[0].dtype == torch.uint8
    assert e.first_scale[0].shape == (2,)
    with pytest.raises(ValueError, match="first scales 0"):
        optim.adamw_step(p, g, optim.AdamWState(e.first, e.second, [torch.zeros(1)], e.second_scale), 1)
    with pytest.raises(RuntimeError, match="autograd"):
        optim.adamw_step([torch.zeros(300, requires_grad=True)], g, s, 1)


def test_codes_of_the_plain_form():
    """Codes keep a value to half a step of its root, and what they stand for is put in the same codes again."""
    rng = np.random.default_rng(0)
    v = (rng.normal(size=1000) * np.exp(-8 * rng.random(1000))).astype(np.float32)
    for signed, x, steps in ((True, v, 127), (False, np.abs(v), 255)):
        code, scale = put(x, steps, signed)
        assert np.abs(code).max() == steps and code.min() >= (-127 if signed else 0)
        back = shown(code, scale, signed)
        back = back if signed else np.sqrt(back)
        assert np.array_equal(put(back.astype(np.float32), steps, signed)[0], code)
        most = np.repeat(scale, 256)[:1000].astype(np.float64)
        root = np.sqrt(np.abs(x) / most)
        assert np.all(np.abs(np.sqrt(np.abs(back) / most) - root)[code != 1] <= 0.5001 / steps)
    assert np.all(put(np.zeros(5, np.float32), 127, True)[0] == 0)
