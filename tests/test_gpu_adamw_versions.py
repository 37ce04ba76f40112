"""What a step writes in place has a new version, so that autograd refuses a
backward pass that needs the values from before."""

import pytest
import torch

from yabt_amd import optim

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
def test_tensors_that_a_backward_pass_kept(bits):
    p, g = torch.ones(300, device="cuda"), torch.ones(300, device="cuda")
    s = optim.adamw_state([p], bits)
    kept = [p, s.first[0], s.second[0]] + ([s.first_scale[0], s.second_scale[0]] if bits == 8 else [])
    before = [t._version for t in kept]
    x = torch.ones(300, device="cuda", requires_grad=True)
    y = (x * p).sum()
    optim.adamw_step([p], [g], s, 1)
    assert all(t._version > v for t, v in zip(kept, before)) and g._version == 0
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()


def test_one_without_a_gradient_stays():
    p = [torch.ones(300, device="cuda") for _ in range(2)]
    s = optim.adamw_state(p)
    optim.adamw_step(p, [None, torch.ones(300, device="cuda")], s, 1)
    assert p[0]._version == 0 and s.first[0]._version == 0 and p[1]._version > 0


def test_inference_tensors_have_no_versions():
    with torch.inference_mode():
        p = torch.ones(300, device="cuda")
    q = torch.ones(300, device="cuda")
    s = optim.adamw_state([p, q])
    before = q._version
    optim.adamw_step([p, q], [torch.ones(300, device="cuda")] * 2, s, 1)
    assert torch.equal(p, q) and bool((p < 1.0).all()) and q._version > before
    with torch.inference_mode():
        optim.adamw_step([p, q], [torch.ones(300, device="cuda")] * 2, optim.adamw_state([p, q]), 1)
