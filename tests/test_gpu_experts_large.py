"""The 256 x 256 tiles of every product, in both ways that operands reach LDS
(whole 16-byte pieces of rows, or any width through registers) and in both ways
that answers leave (one slot a row, or the slots' fp32 answers added), against
the formulas in float64.  The sizes are held to lead there."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from yabt_amd import _lib, expert_ops as X

from expert_plain import products

TYPES = [torch.bfloat16, torch.float16]
INNER_FEW, ANSWER_FEW, H, Y, INNER_GRAD, GRADS = (1 << i for i in range(6))
# 15 of 16 experts with about 850 slots: four row tiles, the last one a third full
SIZES = [(6400, 400, 400, 16, 2), (6400, 397, 395, 16, 2), (12_800, 400, 408, 16, 1), (12_800, 395, 397, 16, 1),
         (4300, 520, 392, 16, 3)]


def name(dt):
    return str(dt).replace("torch.", "")


@pytest.mark.parametrize("n,D,F,E,k", SIZES)
def test_sizes_lead_to_large_tiles(n, D, F, E, k):
    for dt in TYPES:
        assert _lib.load().yabt_experts_forms(X.DTYPES[dt], n, k, D, F, E) == H | Y | INNER_GRAD | GRADS
    assert _lib.load().yabt_experts_forms(0, n, k, D, F, E) == 0           # fp32 has none


def test_forms_of_few_rows_and_of_bad_sizes():
    forms = _lib.load().yabt_experts_forms
    assert forms(1, 1, 6, 1024, 512, 64) == INNER_FEW | ANSWER_FEW
    assert forms(2, 48, 4, 2048, 1024, 32) == INNER_FEW
    assert forms(0, 500, 2, 64, 64, 16) == 0 and forms(0, 100, 2, 64, 64, 16) == INNER_FEW
    assert forms(3, 1, 6, 1024, 512, 64) == -1 and forms(1, 1, 6, 0, 512, 64) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES, ids=name)
@pytest.mark.parametrize("n,D,F,E,k", SIZES)
def test_large_tiles_of_all_products(n, D, F, E, k, dt):
    print(f"large n={n} D={D} F={F} E={E} k={k} {name(dt)}", flush=True)
    gen = torch.Generator().manual_seed(n + D)
    x, dy = torch.randn((n, D), generator=gen).to(dt), torch.randn((n, D), generator=gen).to(dt)
    w_in = (torch.randn((E, 2 * F, D), generator=gen) / D ** 0.5).to(dt)
    w_out = (torch.randn((E, D, F), generator=gen) / F ** 0.5).to(dt)
    gate = torch.randn((n, E), generator=gen)
    gate[:, E - 1] = -1e9                                                 # an expert without rows
    ids = gate.topk(k, dim=1).indices.to(torch.int32)
    weights = torch.rand((n, k), generator=gen) + 0.1
    off = torch.rand((n, k), generator=gen) < 0.03                        # slots without an expert
    ids[off], weights[off] = -1, 0.0
    d = [t.double().numpy() for t in (x, weights, w_in, w_out, dy)]
    want = products(d[0], ids.numpy(), d[1], d[2], d[3], name(dt), d[4])
    xc, wc, ic, oc, dc = (t.cuda() for t in (x, weights, w_in, w_out, dy))
    plan = X.expert_plan(ids.cuda(), E)
    y, inner = X.expert_products(xc, plan, wc, ic, oc, keep_inner=True)
    got = dict(zip(("y", "dx", "dweights", "dw_in", "dw_out"),
                   (y,) + tuple(X.expert_products_grad(dc, xc, plan, wc, ic, oc, inner))))
    assert torch.equal(X.expert_products(xc, plan, wc, ic, oc), y)
    for m, (value, bound) in want.items():
        off = np.abs(got[m].double().cpu().numpy() - value)
        assert np.all(off <= bound), f"{m}: {np.max(off / bound):.3g} of the bound"
