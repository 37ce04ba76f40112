"""The shape of the margin that a stage is given."""

import numpy as np
import pytest

from yabt_amd import ExpertParams, ExpertStage, MSELoss

pytestmark = pytest.mark.gpu


def test_margin_of_another_shape_is_refused():
    rng = np.random.default_rng(0)
    X = rng.normal(size=(60, 3)).astype(np.float32)
    stage = ExpertStage(ExpertParams(experts=2, k=1, width=8, inner=8, epochs=1), MSELoss()).fit(X, X[:, 0])
    for bad in (np.zeros((60, 1)), np.zeros(59), np.zeros((2, 60))):
        with pytest.raises(ValueError):
            stage.predict_margin(X, bad)
    assert np.array_equal(stage.predict_margin(X, np.full(1, 0.5)), stage.predict_margin(X, 0.5))
