"""An ExpertStage's parameters of the dense kind, without a device."""

import pickle

import numpy as np
import pytest
import torch

from yabt_amd import ExpertParams, ExpertStage, MSELoss


@pytest.mark.parametrize("bad,text", [(dict(shared=-1), "shared"), (dict(state_bits=16), "state_bits"),
                                      (dict(weight_decay=-0.1), "weight_decay"), (dict(weight_decay=float("nan")), "weight_decay")])
def test_refused(bad, text):
    with pytest.raises(ValueError, match=text):
        ExpertStage(ExpertParams(**bad), MSELoss()).fit(np.zeros((4, 2), np.float32), np.zeros(4, np.float32))


def test_8_bits_without_a_block():
    with pytest.raises(ValueError, match="shared block"):
        ExpertStage(ExpertParams(), MSELoss()).predict_margin(np.zeros((4, 2), np.float32), int8=True)


def test_parameters_saved_before_there_was_a_block():
    p = ExpertParams(experts=4)
    for m in ("shared", "weight_decay", "state_bits"):
        del p.__dict__[m]
    again = pickle.loads(pickle.dumps(p))
    assert (again.shared, again.weight_decay, again.state_bits, again.experts) == (0, 0.0, 32, 4)
    ExpertStage(again, MSELoss())._check()


def test_the_order_of_the_parameters_is_kept():
    p = ExpertParams(4, 1, 8, 8, "softmax", 0.0, 1, 16, 1e-3, "bfloat16", 3, "cuda:0")
    assert (p.random_state, p.device, p.shared) == (3, "cuda:0", 0)
