"""The expert layer's C entry points refuse bad arguments before they touch a
device, and its plain restatement has the gradients that differences give."""

import numpy as np

from yabt_amd import _lib

from expert_plain import norm, norm_grad


def refused(rc, text):
    assert rc < 0 and text in _lib.last_error(), (rc, _lib.last_error())


def test_norm_refusals():
    lib = _lib.load()
    refused(lib.yabt_layer_norm(3, 16, 8, 4, 8, 0, 0, 1e-5, 16, 8, 0, 0, None), "dtype")
    refused(lib.yabt_layer_norm(0, 16, 7, 4, 8, 0, 0, 1e-5, 16, 8, 0, 0, None), "bad sizes")
    refused(lib.yabt_layer_norm(0, 16, 8, 4, 8, 0, 0, float("nan"), 16, 8, 0, 0, None), "bad sizes")
    refused(lib.yabt_layer_norm(0, 0, 8, 4, 8, 0, 0, 1e-5, 16, 8, 0, 0, None), "null pointer")
    assert lib.yabt_layer_norm(0, 0, 8, 0, 8, 0, 0, 1e-5, 0, 8, 0, 0, None) == 0
    refused(lib.yabt_layer_norm_grad(0, 16, 8, 16, 8, 4, 8, 0, 16, 16, 16, 8, 16, 8, 16, 16, None), "workspace")
    refused(lib.yabt_layer_norm_grad(0, 16, 8, 16, 8, 4, 8, 0, 0, 16, 16, 8, 16, 8, 16, 16, None), "null pointer")
    assert lib.yabt_layer_norm_grad_workspace_bytes(4, 0) == 0
    sizes = [lib.yabt_layer_norm_grad_workspace_bytes(n, 100) for n in range(0, 5000, 7)]
    assert sizes == sorted(sizes) and sizes[0] >= 800


def test_route_refusals():
    lib = _lib.load()

    def route(dt=0, ld=8, n=4, E=8, k=2, scores=0, groups=1, keep=1, p=16):
        return lib.yabt_route(dt, p, ld, n, E, k, scores, 0, groups, keep, 1, 1.0, p, p, None)

    for args, text in [(dict(dt=5), "dtype"), (dict(ld=7), "bad sizes"), (dict(E=2000, ld=2000), "bad sizes"),
                       (dict(k=9), "k <= min"), (dict(E=64, ld=64, k=33), "k <= min"), (dict(scores=2), "scores"),
                       (dict(groups=3), "groups"), (dict(groups=4, keep=5), "groups"), (dict(p=0), "null pointer")]:
        refused(route(**args), text)
    assert route(n=0, p=0) == 0
    refused(lib.yabt_route_grad(0, 16, 1, 16, 8, 16, 4, 8, 2, 0, 1, 1.0, 16, 8, None), "k <= min")
    refused(lib.yabt_route_grad(0, 16, 2, 16, 8, 16, 4, 8, 2, 0, 1, 1.0, 16, 7, None), "bad sizes")
    refused(lib.yabt_route_grad(0, 0, 2, 16, 8, 16, 4, 8, 2, 0, 1, 1.0, 16, 8, None), "null pointer")


def test_plan_refusals():
    lib = _lib.load()
    for n, k, E in [(-1, 1, 4), (4, 0, 4), (4, 1, 0), (4, 1, 1025), (2 ** 30, 2, 4)]:
        assert lib.yabt_expert_plan_workspace_bytes(n, k, E) == 0
        refused(lib.yabt_expert_plan(16, n, k, E, 16, 1 << 30, 16, 16, 16, None), "bad sizes")
    refused(lib.yabt_expert_plan(16, 4, 1, 4, 16, 4, 16, 16, 16, None), "workspace")
    refused(lib.yabt_expert_plan(0, 4, 1, 4, 16, 1 << 20, 16, 16, 16, None), "null pointer")


def test_plain_norm_gradient_against_differences():
    rng = np.random.default_rng(0)
    x, c, w, b = rng.normal(size=(3, 7)), rng.normal(size=(3, 7)), rng.normal(size=7), rng.normal(size=7)
    _, mean, rstd = norm(x, w, b, 1e-5)
    dx, dw, db = norm_grad(c, x, mean, rstd, w)
    for grad, arg in ((dx, x), (dw, w), (db, b)):
        flat = arg.reshape(-1)
        for i in range(flat.size):
            keep, h = flat[i], 1e-6
            flat[i] = keep + h
            up = (norm(x, w, b, 1e-5)[0] * c).sum()
            flat[i] = keep - h
            down = (norm(x, w, b, 1e-5)[0] * c).sum()
            flat[i] = keep
            assert abs((up - down) / (2 * h) - grad.reshape(-1)[i]) < 1e-7 * max(1.0, np.abs(grad).max()) + 1e-7


def test_experts_refusals():
    lib = _lib.load()
    big = 1 << 40

    def call(dt=0, ldx=8, n=4, k=2, D=8, F=4, E=3, p=4096, ws=big, ldy=8):
        return lib.yabt_experts(dt, p, ldx, n, k, D, F, E, p, p, p, p, p, p, p, p, ws, 0, p, ldy, None)

    def grad(dt=0, ldx=8, n=4, k=2, D=8, F=4, E=3, p=4096, ws=big, lddy=8, lddx=8):
        return lib.yabt_experts_grad(dt, p, lddy, p, ldx, n, k, D, F, E, p, p, p, p, p, p, p, p, p, ws, p, lddx, p, p, p,
                                     None)

    for f in (call, grad):
        for args, text in [(dict(dt=3), "dtype"), (dict(ldx=7), "bad sizes"), (dict(k=0), "bad sizes"),
                           (dict(D=0), "bad sizes"), (dict(F=0), "bad sizes"), (dict(E=0), "bad sizes"),
                           (dict(E=1025), "bad sizes"), (dict(n=-1), "bad sizes"), (dict(n=1 << 30), "bad sizes"),
                           (dict(p=0), "null pointer"), (dict(ws=16), "workspace")]:
            refused(f(**args), text)
    assert call(n=0, p=0) == 0
    for sizes in (lib.yabt_experts_workspace_bytes, lib.yabt_experts_grad_workspace_bytes):
        assert sizes(0, 4, 2, 8, 0, 3) == 0 and sizes(9, 4, 2, 8, 4, 3) == 0
        # h (or dg, du, w h) of every slot and the slots' fp32 answers
        assert sizes(1, 1000, 4, 64, 32, 8) >= 4000 * (32 * 2 + 64 * 4)
        assert sizes(1, 1000, 1, 64, 32, 8) >= 1000 * 32 * 2


def test_plain_products_gradient_against_differences():
    from expert_plain import products
    rng = np.random.default_rng(3)
    n, D, F, E, k = 6, 4, 3, 2, 2
    ids = np.array([[0, 1], [1, -1], [0, 1], [-1, -1], [1, 0], [0, -1]])
    a = dict(x=rng.normal(size=(n, D)), w=rng.random((n, k)), w_in=rng.normal(size=(E, 2 * F, D)),
             w_out=rng.normal(size=(E, D, F)))
    dy = rng.normal(size=(n, D))

    def loss():
        return (products(a["x"], ids, a["w"], a["w_in"], a["w_out"], "float32")["y"][0] * dy).sum()

    got = products(a["x"], ids, a["w"], a["w_in"], a["w_out"], "float32", dy)
    for m, grad in (("x", "dx"), ("w", "dweights"), ("w_in", "dw_in"), ("w_out", "dw_out")):
        flat, ref = a[m].reshape(-1), got[grad][0].reshape(-1)
        for i in range(flat.size):
            keep, h = flat[i], 1e-6
            flat[i] = keep + h
            up = loss()
            flat[i] = keep - h
            down = loss()
            flat[i] = keep
            assert abs((up - down) / (2 * h) - ref[i]) < 1e-6
