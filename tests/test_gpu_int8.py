"""Rows and products in 8 bits, equal to their definition in float32 steps, and
the block in 8 bits against float64."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from yabt_amd import feed_ops as X

from dense_plain import UNIT, codes, feed8, product8

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = sorted(X.ACTIVATIONS)


def name(dt):
    return str(dt).replace("torch.", "")


def rows(n, D, dt, seed):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn((n, D), generator=gen) * torch.exp(2 * torch.randn((n, 1), generator=gen))).to(dt)


def weight(N, K, seed):
    gen = torch.Generator().manual_seed(seed)
    q = torch.randint(-128, 128, (N, K), generator=gen, dtype=torch.int8)
    return q, torch.rand(N, generator=gen) * 0.01 + 1e-4


# a wave's registers hold 1024 values of fp32 and 2048 of 16 bits, a block's four times that
@pytest.mark.parametrize("dt", TYPES, ids=name)
@pytest.mark.parametrize("n,D", [(1, 1), (3, 7), (5, 16), (9, 100), (64, 513), (7, 1024), (6, 1025), (5, 2048), (5, 2049),
                                 (3, 4097), (2, 8192), (2, 8200), (2, 20_001)])
def test_quantized_rows(n, D, dt):
    x = rows(n, D, dt, n + D)
    if n > 2:
        x[1] = 0.0
    q, s = X.quantize_rows(x.cuda())
    wq, ws = codes(x.float().numpy())
    assert np.array_equal(q.cpu().numpy(), wq) and np.array_equal(s.cpu().numpy(), ws)


def test_rows_at_the_borders():
    """Ties go to even, tiny rows count as zeros, rows that are not finite are NaN and nothing else."""
    x = torch.zeros((8, 40))
    x[0, :5] = torch.tensor([127.0, 0.5, 1.5, -2.5, 126.5])
    x[1] = 2.0 ** -101
    x[2] = 2.0 ** -100
    x[3, 7] = float("nan")
    x[4, 39] = float("-inf")
    x[5] = 3e38
    x[6, 0] = -1e-42
    x[7] = torch.linspace(-1, 1, 40)
    q, s = X.quantize_rows(x.cuda())
    wq, ws = codes(x.numpy())
    assert np.array_equal(q.cpu().numpy(), wq) and np.array_equal(s.cpu().numpy(), ws, equal_nan=True)
    assert q[0, :5].tolist() == [127, 0, 2, -2, 126]
    wide = torch.full((8, 61), float("nan"), device="cuda")
    wide[:, 5:45] = x.cuda()
    q2, s2 = X.quantize_rows(wide[:, 5:45])
    assert torch.equal(q, q2) and np.array_equal(s2.cpu().numpy(), ws, equal_nan=True)


def want(a, sa, b, sb, dt):
    y = torch.from_numpy(product8(a.numpy(), sa.numpy(), b.numpy(), sb.numpy()))
    return y.to(dt)


@pytest.mark.parametrize("dt", TYPES, ids=name)
@pytest.mark.parametrize("n,K,N", [(1, 1, 1), (1, 300, 17), (15, 16, 33), (16, 128, 16), (17, 127, 40), (40, 500, 21), (64, 1000, 100),
                                   (65, 64, 64), (100, 100, 130), (300, 257, 129), (129, 2048, 64), (70, 9000, 30), (400, 1104, 8000)])
def test_products(n, K, N, dt):
    gen = torch.Generator().manual_seed(K)
    a = torch.randint(-128, 128, (n, K), generator=gen, dtype=torch.int8)
    sa = torch.rand(n, generator=gen) + 0.01
    b, sb = weight(N, K, N)
    y = X.product_int8(a.cuda(), sa.cuda(), b.cuda(), sb.cuda(), dtype=dt)
    assert y.dtype == dt and torch.equal(y.cpu(), want(a, sa, b, sb, dt))


@pytest.mark.parametrize("n,K,N", [(2048, 768, 4096), (2100, 784, 4100), (4096, 801, 2050)])
def test_large_products(n, K, N):
    gen = torch.Generator().manual_seed(K)
    a = torch.randint(-127, 128, (n, K), generator=gen, dtype=torch.int8)
    sa = torch.rand(n, generator=gen) + 0.01
    b, sb = weight(N, K, N)
    y = X.product_int8(a.cuda(), sa.cuda(), b.cuda(), sb.cuda(), dtype=torch.bfloat16)
    assert torch.equal(y.cpu(), want(a, sa, b, sb, torch.bfloat16))


@pytest.mark.parametrize("n", [2, 80])
def test_the_longest_sums(n):
    """131 071 terms of 128 x 128: the sum is 2^31 - 2^14."""
    K = X.MAX_INT8_TERMS
    a = torch.full((n, K), -128, dtype=torch.int8, device="cuda")
    b = torch.full((3, K), -128, dtype=torch.int8, device="cuda")
    b[1] = 127
    one = torch.ones(3, device="cuda")
    y = X.product_int8(a, torch.ones(n, device="cuda"), b, one)
    assert torch.equal(y, torch.tensor([128.0 * 128 * K, -128.0 * 127 * K, 128.0 * 128 * K], device="cuda").expand(n, 3))


def test_codes_of_other_pitch_and_address():
    for n, K, N in ((5, 100, 30), (90, 64, 70), (200, 333, 65)):
        gen = torch.Generator().manual_seed(n)
        a = torch.randint(-128, 128, (n, K + 11), generator=gen, dtype=torch.int8).cuda()
        b = torch.randint(-128, 128, (N, K + 3), generator=gen, dtype=torch.int8).cuda()
        sa, sb = torch.rand(n, generator=gen).cuda(), torch.rand(N, generator=gen).cuda()
        p, q = a[:, 5:5 + K], b[:, 1:1 + K]
        assert torch.equal(X.product_int8(p, sa, q, sb), X.product_int8(p.contiguous(), sa, q.contiguous(), sb))
        t = p.t().contiguous().t()
        assert torch.equal(X.product_int8(p, sa, q, sb), X.product_int8(t, sa, q, sb))


def test_rows_that_are_nan_stay_alone():
    for n in (20, 200):
        x = rows(n, 96, torch.bfloat16, 1).cuda()
        w = X.quantize_rows(rows(50, 96, torch.float32, 2).cuda())
        y = X.product_int8(*X.quantize_rows(x), *w)
        x[3, 4] = float("inf")
        z = X.product_int8(*X.quantize_rows(x), *w)
        keep = torch.arange(n, device="cuda") != 3
        assert torch.equal(y[keep], z[keep]) and bool(torch.isnan(z[3]).all())


def block(n, D, F, O, dt, seed):
    gen = torch.Generator().manual_seed(seed)
    w_in, w_out = torch.randn((2 * F, D), generator=gen) / D ** 0.5, torch.randn((O, F), generator=gen) / F ** 0.5
    return rows(n, D, dt, seed), *X.quantize_rows(w_in.cuda()), *X.quantize_rows(w_out.cuda())


# few rows whose values every block puts in 8 bits itself (to 16384 of them), more, and tiles
@pytest.mark.parametrize("dt", TYPES, ids=name)
@pytest.mark.parametrize("n,D,F,O", [(1, 1, 1, 1), (1, 1000, 300, 40), (5, 33, 17, 20), (16, 1024, 64, 32), (17, 1025, 50, 64),
                                     (64, 256, 257, 30), (64, 250, 255, 30), (33, 100, 700, 100), (65, 64, 64, 64),
                                     (130, 100, 61, 100), (300, 72, 400, 33), (70, 40, 5000, 16), (100, 1040, 130, 50)])
def test_block_in_8_bits(n, D, F, O, dt):
    act = ACTS[(n + D) % 4]
    print(f"feed8 n={n} D={D} F={F} O={O} {act} {name(dt)}", flush=True)
    x, *w = block(n, D, F, O, dt, n + D)
    y = X.feed_forward_int8(x.cuda(), *w, activation=act)
    value, bound = feed8(x.float().numpy(), *(t.cpu().numpy() for t in w), act)
    got, most = y.double().cpu().numpy(), torch.finfo(dt).max
    bound = bound + UNIT[name(dt)] * (np.abs(value) + bound) + (2.0 ** -25 if dt == torch.float16 else 2.0 ** -133)
    # rounding to the type makes what is half a step past its largest value infinite
    past = np.isinf(got) & (np.sign(got) * value + bound > most)
    off = np.where(past, 0.0, np.abs(got - value))
    assert np.all(off <= bound), f"{np.max(off / bound):.3g} of the bound"
    assert torch.equal(y, X.feed_forward_int8(x.cuda(), *w, activation=act))


def test_large_block_in_8_bits():
    """The same as its parts, made one by one."""
    x, *w = block(2048, 768, 2048, 4096, torch.bfloat16, 3)
    y = X.feed_forward_int8(x.cuda(), *w)
    pre = X.product_int8(*X.quantize_rows(x.cuda()), w[0], w[1])
    g, u = pre.chunk(2, dim=1)
    h = torch.nn.functional.silu(g) * u
    z = X.product_int8(*X.quantize_rows(h), w[2], w[3], dtype=torch.bfloat16)
    # codes at a border: one of 127 steps in a few of 2048 places
    assert float((y.float() - z.float()).norm() / z.float().norm()) < 2.0 ** -8


def test_8_bits_are_near_the_block_itself():
    """Codes of rows and weights are off by half a 127th of the largest at most, some 4 standard deviations of
    normal values: 4 / 254 / sqrt(3) of a factor, two factors a product and three products' worth."""
    gen = torch.Generator().manual_seed(0)
    x, w_in, w_out = (torch.randn(s, generator=gen).cuda() for s in ((200, 256), (512, 256), (64, 256)))
    w_in, w_out = w_in / 16, w_out / 16
    y = X.feed_forward(x, w_in, w_out)
    z = X.feed_forward_int8(x, *X.quantize_rows(w_in), *X.quantize_rows(w_out))
    assert float((y - z).norm() / y.norm()) < 0.06


@pytest.mark.parametrize("n", [4, 300])
def test_captured_and_replayed(n):
    x, *w = block(n, 128, 96, 64, torch.float16, 7)
    x = x.cuda()
    X.feed_forward_int8(x, *w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, s = X.quantize_rows(x)
        p = X.product_int8(q, s, w[0], w[1])
        y = X.feed_forward_int8(x, *w)
    for _ in range(4):
        x.mul_(1.1)
        graph.replay()
        want_p, want_y = X.product_int8(*X.quantize_rows(x), w[0], w[1]), X.feed_forward_int8(x, *w)
        torch.cuda.synchronize()
        assert torch.equal(p, want_p) and torch.equal(y, want_y)


def test_no_rows():
    x, *w = block(0, 24, 10, 12, torch.bfloat16, 1)
    q, s = X.quantize_rows(x.cuda())
    assert q.shape == (0, 24) and s.shape == (0,)
    assert X.product_int8(q, s, w[0], w[1]).shape == (0, 20)
    assert X.feed_forward_int8(x.cuda(), *w).shape == (0, 12)


# few tiles over a long sum: [g u] is made in parts
@pytest.mark.parametrize("dt", TYPES, ids=name)
@pytest.mark.parametrize("n,D,F,O", [(65, 9000, 17, 30), (83, 2520, 256, 40), (300, 8192, 130, 33), (100, 4096, 1021, 16)])
def test_block_of_few_tiles_over_long_sums(n, D, F, O, dt):
    x, *w = block(n, D, F, O, dt, n + D)
    y = X.feed_forward_int8(x.cuda(), *w, activation="gelu_tanh")
    value, bound = feed8(x.float().numpy(), *(t.cpu().numpy() for t in w), "gelu_tanh")
    # feed8 bounds the value before it is rounded to the type: half a step of it, or of the type's least values
    bound = bound + UNIT[name(dt)] * (np.abs(value) + bound) + (2.0 ** -25 if dt == torch.float16 else 2.0 ** -133)
    got, most = y.double().cpu().numpy(), torch.finfo(dt).max
    # rounding to the type makes what is half a step past its largest value infinite
    past = np.isinf(got) & (np.sign(got) * value + bound > most)
    off = np.where(past, 0.0, np.abs(got - value))
    assert np.all(off <= bound), f"{np.max(off / bound):.3g} of the bound"
