"""Every form of the block's kernels that sizes choose, held to the form that the
size is there for: 128 x 256 tiles of fp32 for each product, 256 x 256 tiles of 8-bit
codes with ragged edges and with operands through registers, 16 rows or fewer of a wide block."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from yabt_amd import _lib, feed_ops as X

from dense_plain import UNIT, feed

TYPES = [torch.float32, torch.bfloat16, torch.float16]
(FEW, FEW_OUT, H, Y, INNER_GRAD, GRADS, H_PARTS, Y_PARTS, INNER_GRAD_PARTS, GRADS_PARTS, WHOLE) = (1 << i for i in range(11))
X_CODES, H_CODES = 1 << 10, 1 << 11
U32 = 2.0 ** -24

# whole tiles; odd widths throughout; rows' and gradients' sums in parts beside them; dh of large tiles beside gradients of small ones
FP32 = [((2560, 256, 2560, 2560), H | Y | INNER_GRAD | GRADS), ((2571, 261, 2565, 2563), H | Y | INNER_GRAD | GRADS),
        ((2571, 101, 2565, 2563), Y | INNER_GRAD), ((2571, 1027, 1301, 801), H | GRADS)]
INT8 = [((2048, 768, 2048, 300), H), ((2050, 784, 2052, 300), H), ((2050, 784, 2051, 300), H), ((2050, 801, 2051, 300), H),
        ((2050, 801, 2052, 4100), H | Y)]
WIDE = [(16, 60, 2050, 2100), (16, 64, 2048, 2304), (5, 33, 4101, 4100), (9, 40, 3001, 2999)]


def name(dt):
    return str(dt).replace("torch.", "")


def test_sizes_lead_to_their_forms():
    lib = _lib.load()
    mask = H | Y | INNER_GRAD | GRADS
    for size, want in FP32:
        assert lib.yabt_feed_forward_forms(0, *size) & mask == want, size
    for size, want in INT8:
        assert lib.yabt_feed_forward_int8_forms(*size) & (FEW | H | Y) == want, size
    for size in WIDE:
        for dt in range(3):
            assert lib.yabt_feed_forward_forms(dt, *size) & (FEW | FEW_OUT | Y_PARTS | WHOLE) == FEW | Y_PARTS, size


def test_forms_of_few_rows_and_of_bad_sizes():
    forms, forms8 = _lib.load().yabt_feed_forward_forms, _lib.load().yabt_feed_forward_int8_forms
    assert forms(1, 1, 1024, 4096, 1024) & 0xFF == FEW | FEW_OUT and forms(1, 1, 1024, 4096, 1024) & WHOLE
    assert forms(2, 48, 2048, 5632, 2048) & 0xCF == FEW | Y_PARTS
    assert forms(1, 8192, 2048, 5632, 2048) & 0xFF == H | Y | INNER_GRAD | GRADS
    assert forms(0, 83, 2520, 256, 2520) & H_PARTS and forms(0, 300, 40, 64, 3100) & INNER_GRAD_PARTS
    assert forms8(64, 256, 257, 30) == FEW | FEW_OUT | X_CODES and forms8(64, 250, 255, 30) == FEW | FEW_OUT | X_CODES | H_CODES
    assert forms8(83, 2520, 256, 40) & H_PARTS
    assert forms(3, 8, 8, 8, 8) == -1 and forms(0, 8, 0, 8, 8) == -1 and forms8(8, 8, 131072, 8) == -1


def inputs(n, D, F, O, dt, seed):
    gen = torch.Generator().manual_seed(seed)
    return ((1.5 * torch.randn((n, D), generator=gen)).to(dt), (torch.randn((2 * F, D), generator=gen) / D ** 0.5).to(dt),
            (torch.randn((O, F), generator=gen) / F ** 0.5).to(dt), torch.randn((n, O), generator=gen).to(dt))


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("size", [s for s, _ in FP32])
def test_large_tiles_of_float32(size, act):
    """Against float64 on the device.  A sum of K terms in any order, each partial sum rounded by 2^-24 / sqrt(3)
    of itself (times 0.7, the mean of a value over its power of two), has an error of 0.4 sqrt(K / 2) units of its
    own rms: 21 for K = 5130, 15 for 2571, and an output has two such sums, slopes' 4 and the parts'
    left-out products' 1 behind it: 26, and 40 allows for partial sums that do not grow evenly.  A product of parts
    that is lost makes 160 (the least of the six)."""
    print(f"feed forms {size} {act}", flush=True)
    n, D, F, O = size
    args = [t.cuda() for t in inputs(n, D, F, O, torch.float32, n + D)]
    y, inner = X.feed_forward(*args[:3], activation=act, keep_inner=True)
    got = (y,) + tuple(X.feed_forward_grad(args[3], *args[:3], inner, activation=act))
    x, w_in, w_out, dy = (t.double().requires_grad_(i < 3) for i, t in enumerate(args))
    g, u = (x @ w_in.t()).chunk(2, dim=1)
    want = ((torch.nn.functional.silu if act == "silu" else torch.nn.functional.gelu)(g) * u) @ w_out.t()
    want = (want.detach(),) + torch.autograd.grad(want, [x, w_in, w_out], dy)
    for m, a, b in zip(("y", "dx", "dw_in", "dw_out"), got, want):
        off, rms = a.double() - b, float(b.square().mean().sqrt())
        assert float(off.square().mean().sqrt()) <= 40 * U32 * rms, (m, float(off.square().mean().sqrt()) / rms / U32)
        # and every value within 8 standard deviations of that: no tile, row or column is wrong
        assert bool((off.abs() <= 8 * 40 * U32 * rms).all()), m
    assert torch.equal(X.feed_forward(*args[:3], activation=act), y)


def gates(act, g):
    """act(g) in float64 and what float32 may make of it (yabt_feed_forward_int8 in the C header)."""
    f = torch.nn.functional
    if act == "gelu":
        return f.gelu(g), (20 + 2 * g * g) * U32
    return f.silu(g), (8 + 10 * g.abs()) * U32


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dt", TYPES, ids=name)
@pytest.mark.parametrize("size", [s for s, _ in INT8])
def test_large_tiles_of_the_block_in_8_bits(size, dt, act):
    """Element by element, from the codes' products (exact): where the float32 of h may move a code
    over a border, the code may be off by one."""
    n, D, F, O = size
    print(f"feed8 forms {size} {act} {name(dt)}", flush=True)
    gen = torch.Generator().manual_seed(n + D)
    x = (torch.randn((n, D), generator=gen) * torch.exp(torch.randn((n, 1), generator=gen))).to(dt).cuda()
    w_in = X.quantize_rows((torch.randn((2 * F, D), generator=gen) / D ** 0.5).cuda())
    w_out = X.quantize_rows((torch.randn((O, F), generator=gen) / F ** 0.5).cuda())
    y = X.feed_forward_int8(x, *w_in, *w_out, activation=act)
    g, u = X.product_int8(*X.quantize_rows(x), *w_in).double().chunk(2, dim=1)
    a, ea = gates(act, g)
    h = a * u
    eh = (ea + 4 * U32) * h.abs() + 2.0 ** -126 * u.abs()
    most = h.abs().amax(dim=1, keepdim=True)
    at = 127.0 * h / most
    slack = 127.0 * (eh + h.abs() / most * eh.amax(dim=1, keepdim=True)) / most + 127 * 4 * U32
    border = ((at - at.floor()).sub_(0.5).abs_() <= slack).double()
    w, scale = w_out[0].double().t(), w_out[1].double() * most / 127.0
    value = (at.round() @ w) * scale
    # the row's largest h, the code's scale and y's two products in float32
    e = (border @ w.abs()) * scale + (8 * U32 + float((eh / most).max())) * ((at.abs() @ w.abs()) * scale)
    unit = UNIT[name(dt)]
    bound = e + unit * (value.abs() + e) + (2.0 ** -25 if dt == torch.float16 else 2.0 ** -133)
    off = (y.double() - value).abs()
    assert bool((off <= bound).all()), float((off / bound).max())
    assert float(border.mean()) < 2e-3                     # the bound leaves the codes' errors nothing to hide in
    assert torch.equal(y, X.feed_forward_int8(x, *w_in, *w_out, activation=act))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES, ids=name)
@pytest.mark.parametrize("size", WIDE)
def test_few_rows_of_a_wide_block(size, dt):
    """h is rounded to the type, as of more rows: y's bound is that of the rows among others."""
    print(f"feed wide {size} {name(dt)}", flush=True)
    n = size[0]
    args = inputs(*size, dt, n)
    x, w_in, w_out, dy = (t.cuda() for t in args)
    y, inner = X.feed_forward(x, w_in, w_out, keep_inner=True)
    got = dict(zip(("dx", "dw_in", "dw_out"), X.feed_forward_grad(dy, x, w_in, w_out, inner)), y=y)
    assert torch.equal(X.feed_forward(x, w_in, w_out), y)
    x, w_in, w_out, dy = (t.double().numpy() for t in args)
    want = feed(x, w_in, w_out, "silu", name(dt), dy)
    more = feed(np.concatenate([x, np.zeros((17 - n, x.shape[1]))]), w_in, w_out, "silu", name(dt))["y"]
    want["y"] = more[0][:n], more[1][:n]
    for m, (value, bound) in want.items():
        off = np.abs(got[m].double().cpu().numpy() - value)
        assert np.all(off <= bound), f"{m}: {np.max(off / bound):.3g} of the bound"
