"""A stage that was fitted and saved before answers had a unit."""

import pickle

import torch

from yabt_amd import ExpertParams, ExpertStage, MSELoss


def test_a_saved_stage_without_a_unit():
    stage = ExpertStage(ExpertParams(), MSELoss())
    stage.weights_ = dict(head=torch.arange(3.0))
    assert "unit_" not in vars(stage)
    again = pickle.loads(pickle.dumps(stage))
    assert torch.equal(again._head(), torch.arange(3.0))
