"""Autograd does not see the expert layer's calls: a tensor that requires a
gradient is refused while it records, and taken as it is under no_grad (where
these tensors, on the CPU, meet the next check)."""

import pytest
import torch

from yabt_amd import expert_ops as X


def calls(which):
    """Every call with the which-th of its tensors requiring a gradient."""
    def t(i, *shape):
        return torch.zeros(shape, requires_grad=i == which)

    plan = X.ExpertPlan(*(torch.zeros(s, dtype=torch.int32) for s in ((4, 2), (3,), (8,), (8,))))
    return {
        "layer_norm": (3, lambda: X.layer_norm(t(0, 4, 8), t(1, 8), t(2, 8))),
        "layer_norm_grad": (5, lambda: X.layer_norm_grad(t(0, 4, 8), t(1, 4, 8), t(2, 4), t(3, 4), t(4, 8))),
        "route": (2, lambda: X.route(t(0, 4, 8), 2, bias=t(1, 8))),
        "route_grad": (2, lambda: X.route_grad(t(0, 4, 2), t(1, 4, 8), plan.ids)),
        "expert_products": (4, lambda: X.expert_products(t(0, 4, 8), plan, t(1, 4, 2), t(2, 2, 6, 8), t(3, 2, 8, 3))),
        "expert_products_grad": (6, lambda: X.expert_products_grad(
            t(0, 4, 8), t(1, 4, 8), plan, t(2, 4, 2), t(3, 2, 6, 8), t(4, 2, 8, 3), t(5, 8, 8))),
    }


@pytest.mark.parametrize("name", list(calls(-1)))
def test_tensors_that_require_gradients(name):
    for which in range(calls(-1)[name][0]):
        call = calls(which)[name][1]
        with pytest.raises(RuntimeError, match="autograd"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="HIP device"):
            call()
    with pytest.raises(RuntimeError, match="HIP device"):
        calls(-1)[name][1]()
