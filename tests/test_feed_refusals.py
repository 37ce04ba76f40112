"""What the dense stage's calls refuse, without a device; and the block's plain
form against differences."""

import numpy as np
import pytest
import torch

from yabt_amd import _lib, feed_ops as X

from dense_plain import activation, feed


def refused(rc, text):
    assert rc < 0 and text in _lib.last_error(), (rc, _lib.last_error())


BIG = 1 << 40


def test_block_entries():
    lib = _lib.load()

    def call(dt=0, act=0, ldx=8, n=4, D=8, F=4, O=6, p=4096, ws=BIG, ldy=6):
        return lib.yabt_feed_forward(dt, act, p, ldx, n, D, F, O, p, p, p, ws, 0, p, ldy, None)

    def grad(dt=0, act=0, ldx=8, n=4, D=8, F=4, O=6, p=4096, ws=BIG, ldy=6):
        return lib.yabt_feed_forward_grad(dt, act, p, ldy, p, ldx, n, D, F, O, p, p, p, p, ws, p, 8, p, p, None)

    def codes(dt=0, act=0, ldx=8, n=4, D=8, F=4, O=6, p=4096, ws=BIG, ldy=6):
        return lib.yabt_feed_forward_int8(dt, act, p, ldx, n, D, F, O, p, p, p, p, p, ws, p, ldy, None)

    for f in (call, grad, codes):
        for args, text in [(dict(dt=3), "dtype"), (dict(act=4), "activation"), (dict(act=-1), "activation"),
                           (dict(ldx=7), "bad sizes"), (dict(ldy=5), "bad sizes"), (dict(D=0), "bad sizes"),
                           (dict(F=0), "bad sizes"), (dict(O=0), "bad sizes"), (dict(n=-1), "bad sizes"),
                           (dict(n=1 << 31), "bad sizes"), (dict(F=(1 << 24) + 1), "bad sizes"), (dict(p=0), "null pointer"),
                           (dict(ws=16), "workspace")]:
            refused(f(**args), text)
    assert call(n=0, p=0) == 0 and codes(n=0, p=0) == 0
    refused(codes(D=131072, ldx=131072), "bad sizes")
    for sizes in (lib.yabt_feed_forward_workspace_bytes, lib.yabt_feed_forward_grad_workspace_bytes,
                  lib.yabt_feed_forward_inner_bytes):
        assert sizes(0, 4, 8, 0, 6) == 0 and sizes(9, 4, 8, 4, 6) == 0 and sizes(0, -1, 8, 4, 6) == 0
        assert sizes(1, 1000, 64, 32, 64) >= 1000 * 32 * 2
    assert lib.yabt_feed_forward_inner_bytes(0, 1000, 64, 33, 64) >= 1000 * 4 * (2 * 36 + 36)
    assert lib.yabt_feed_forward_int8_workspace_bytes(10, 0, 4, 4) == 0
    # 2^31 rows' tiles of 64 x 128 have 2^33 threads
    assert lib.yabt_feed_forward_workspace_bytes(0, (1 << 31) - 1000, 1, 1, 1) == 0
    refused(call(n=(1 << 31) - 1000), "bad sizes")
    refused(grad(F=1 << 24, D=1 << 24, ldx=1 << 24), "bad sizes")
    refused(codes(n=(1 << 24) - 1, O=1 << 24, ldy=1 << 24), "bad sizes")


def test_8_bit_entries():
    lib = _lib.load()
    quantize = lambda dt=0, ldx=8, n=4, D=8, ldq=8, p=4096: lib.yabt_quantize_rows(dt, p, ldx, n, D, p, ldq, p, None)  # noqa: E731
    for args, text in [(dict(dt=3), "dtype"), (dict(ldx=7), "bad sizes"), (dict(ldq=7), "bad sizes"), (dict(D=0), "bad sizes"),
                       (dict(n=1 << 24), "bad sizes"), (dict(n=-1), "bad sizes"), (dict(p=0), "null pointer")]:
        refused(quantize(**args), text)
    assert quantize(n=0, p=0) == 0

    def product(dt=0, lda=8, n=4, K=8, ldb=8, N=6, p=4096, ws=BIG, ldy=6):
        return lib.yabt_product_int8(p, lda, p, n, K, p, ldb, p, N, dt, p, ws, p, ldy, None)

    for args, text in [(dict(dt=-1), "dtype"), (dict(lda=7), "bad sizes"), (dict(ldb=7), "bad sizes"), (dict(ldy=5), "bad sizes"),
                       (dict(K=0), "bad sizes"), (dict(N=0), "bad sizes"), (dict(K=131072, lda=131072, ldb=131072), "bad sizes"),
                       (dict(n=1 << 24), "bad sizes"), (dict(p=0), "null pointer"),
                       (dict(n=100, K=2048, lda=2048, ldb=2048, ws=16), "workspace")]:
        refused(product(**args), text)
    assert product(n=0, p=0) == 0
    assert lib.yabt_product_int8_workspace_bytes(4, 0, 6) == 0


def test_python_entries():
    x, a, b = torch.zeros(4, 8), torch.zeros(6, 8), torch.zeros(5, 3)
    q, s = torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4)
    with pytest.raises(ValueError, match="activation"):
        X.feed_forward(x, a, b, activation="tanh")
    for call in (lambda: X.feed_forward(x, a, b), lambda: X.feed_forward_grad(x, x, a, b, x), lambda: X.quantize_rows(x),
                 lambda: X.product_int8(q, s, q, s), lambda: X.feed_forward_int8(x, q, s, q, s)):
        with pytest.raises(RuntimeError, match="HIP device"):
            call()
    with pytest.raises(ValueError, match="int8"):
        X.product_int8(x, s, q, s)
    with pytest.raises(ValueError, match="dtype"):
        X.product_int8(q, s, q, s, dtype=torch.float64)
    with pytest.raises(ValueError, match="matrix"):
        X.feed_forward(x[0], a, b)


def needs(which):
    def t(i, *shape):
        return torch.zeros(shape, requires_grad=i == which)

    q = torch.zeros(4, 8, dtype=torch.int8)
    return {
        "feed_forward": (3, lambda: X.feed_forward(t(0, 4, 8), t(1, 6, 8), t(2, 5, 3))),
        "feed_forward_grad": (4, lambda: X.feed_forward_grad(t(0, 4, 5), t(1, 4, 8), t(2, 6, 8), t(3, 5, 3), q)),
        "quantize_rows": (1, lambda: X.quantize_rows(t(0, 4, 8))),
        "product_int8": (2, lambda: X.product_int8(q, t(0, 4), q, t(1, 4))),
        "feed_forward_int8": (3, lambda: X.feed_forward_int8(t(0, 4, 8), q, t(1, 4), q, t(2, 4))),
    }


@pytest.mark.parametrize("name", list(needs(-1)))
def test_tensors_that_require_gradients(name):
    for which in range(needs(-1)[name][0]):
        call = needs(which)[name][1]
        with pytest.raises(RuntimeError, match="autograd"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="HIP device"):
            call()


@pytest.mark.parametrize("act", sorted(X.ACTIVATIONS))
def test_plain_form_against_differences(act):
    rng = np.random.default_rng(2)
    v = dict(x=rng.normal(size=(5, 4)), w_in=rng.normal(size=(6, 4)), w_out=rng.normal(size=(2, 3)))
    dy = rng.normal(size=(5, 2))
    loss = lambda: (feed(v["x"], v["w_in"], v["w_out"], act, "float32")["y"][0] * dy).sum()  # noqa: E731
    got = feed(v["x"], v["w_in"], v["w_out"], act, "float32", dy)
    for m, grad in (("x", "dx"), ("w_in", "dw_in"), ("w_out", "dw_out")):
        flat, ref = v[m].reshape(-1), got[grad][0].reshape(-1)
        for i in range(flat.size):
            keep, h = flat[i], 1e-6
            flat[i] = keep + h
            up = loss()
            flat[i] = keep - h
            down = loss()
            flat[i] = keep
            assert abs((up - down) / (2 * h) - ref[i]) < 1e-6


def test_slopes_and_curvatures_of_the_bounds():
    g = np.linspace(-30, 30, 600_001)
    for act in ("silu", "gelu", "gelu_tanh"):
        slope = activation(act, g)[1]
        assert np.abs(slope).max() < 1.13 and np.abs(np.diff(slope) / 1e-4).max() < 1.2
