"""silu of float32 rows, by the tiles and by the kernels for few rows."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from yabt_amd import expert_ops as X

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [7, 4096])
def test_silu_of_gates_far_from_zero(n):
    """One column, one inner value, gate row 1 and u row 1.5: y = g silu'd times
    1.5 g, no sum to round.  In units of 2^-24 relative: the exponential 2 (one
    unit in the last place), 1 + e, its reciprocal and the products g s and h
    one each, u = 1.5 g one: 7 of first order, one more for the rest."""
    g = np.concatenate([np.linspace(-60, 30, n - 4), [-20.0, -5.0, 5.0, 20.0]]).astype(np.float32)
    x = torch.as_tensor(g[:, None], device="cuda")
    plan = X.expert_plan(torch.zeros((n, 1), dtype=torch.int32, device="cuda"), 1)
    ones = torch.ones((n, 1), device="cuda")
    w_in = torch.tensor([[[1.0], [1.5]]], device="cuda")
    w_out = torch.ones((1, 1, 1), device="cuda")
    y, inner = X.expert_products(x, plan, ones, w_in, w_out, keep_inner=True)
    _, dweights, _, _ = X.expert_products_grad(ones, x, plan, ones, w_in, w_out, inner)
    d = g.astype(np.float64)
    want = d / (1.0 + np.exp(-d)) * 1.5 * d
    for got in (y, dweights):
        off = np.abs(got[:, 0].double().cpu().numpy() - want)
        assert np.all(off <= 8 * 2.0 ** -24 * np.abs(want)), np.max(off / np.maximum(np.abs(want), 1e-300)) * 2 ** 24
