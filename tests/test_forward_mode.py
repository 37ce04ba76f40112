"""Autograd's forward mode does not see the expert layer's, the dense stage's and
the optimiser's calls: a tensor with a tangent is refused, also under no_grad, which
leaves tangents on; without one, or with forward mode off, it is taken as it is
(and meets the next check: these tensors are on the CPU)."""

import pytest
import torch
from torch.autograd import forward_ad

from yabt_amd import expert_ops as E, feed_ops as X, optim


def calls(which):
    """Every call with the which-th of its tensors dual."""
    def t(i, *shape):
        z = torch.zeros(shape)
        return forward_ad.make_dual(z, torch.ones(shape)) if i == which else z

    plan = E.ExpertPlan(*(torch.zeros(s, dtype=torch.int32) for s in ((4, 2), (3,), (8,), (8,))))
    q = torch.zeros(4, 8, dtype=torch.int8)
    return {
        "layer_norm": (3, lambda: E.layer_norm(t(0, 4, 8), t(1, 8), t(2, 8))),
        "layer_norm_grad": (5, lambda: E.layer_norm_grad(t(0, 4, 8), t(1, 4, 8), t(2, 4), t(3, 4), t(4, 8))),
        "route": (2, lambda: E.route(t(0, 4, 8), 2, bias=t(1, 8))),
        "route_grad": (2, lambda: E.route_grad(t(0, 4, 2), t(1, 4, 8), plan.ids)),
        "expert_products": (4, lambda: E.expert_products(t(0, 4, 8), plan, t(1, 4, 2), t(2, 2, 6, 8), t(3, 2, 8, 3))),
        "expert_products_grad": (6, lambda: E.expert_products_grad(
            t(0, 4, 8), t(1, 4, 8), plan, t(2, 4, 2), t(3, 2, 6, 8), t(4, 2, 8, 3), t(5, 8, 8))),
        "feed_forward": (3, lambda: X.feed_forward(t(0, 4, 8), t(1, 6, 8), t(2, 5, 3))),
        "feed_forward_grad": (4, lambda: X.feed_forward_grad(t(0, 4, 5), t(1, 4, 8), t(2, 6, 8), t(3, 5, 3), q)),
        "quantize_rows": (1, lambda: X.quantize_rows(t(0, 4, 8))),
        "product_int8": (2, lambda: X.product_int8(q, t(0, 4), q, t(1, 4))),
        "feed_forward_int8": (3, lambda: X.feed_forward_int8(t(0, 4, 8), q, t(1, 4), q, t(2, 4))),
        "adamw_step": (4, lambda: optim.adamw_step([t(0, 9)], [t(1, 9)], optim.AdamWState([t(2, 9)], [t(3, 9)]), 1)),
    }


@pytest.mark.parametrize("name", list(calls(-1)))
def test_tensors_with_tangents(name):
    with forward_ad.dual_level():
        for which in range(calls(-1)[name][0]):
            call = calls(which)[name][1]
            with pytest.raises(RuntimeError, match="forward mode"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward mode"):
                call()
            with torch.inference_mode(), pytest.raises(RuntimeError, match="HIP device"):
                call()
        with pytest.raises(RuntimeError, match="HIP device"):
            calls(-1)[name][1]()
