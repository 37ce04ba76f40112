"""What the stage does with columns that the fit could learn nothing from."""

from __future__ import annotations

import numpy as np
import pytest

from yabt_amd import ExpertParams, ExpertStage, MSELoss

pytestmark = pytest.mark.gpu


def table(n=2000, F=6, seed=0):
    rng = np.random.default_rng(seed)
    X = rng.normal(size=(n, F)).astype(np.float32)
    return X, (X[:, 0] - np.abs(X[:, 1])).astype(np.float32)


def fitted(X, y):
    return ExpertStage(ExpertParams(experts=4, k=2, width=16, inner=16, epochs=3), MSELoss()).fit(X, y)


@pytest.mark.parametrize("constant,later", [(0.0, 1.0), (0.1, 0.11), (-7.5, np.nan), (np.nan, 1.0), (np.nan, -1e30),
                                            (1e30, -1e30)])
def test_columns_without_spread_add_nothing(constant, later):
    X, y = table()
    X[:, 4] = constant
    stage = fitted(X, y)
    rows = X[:8].copy()
    rows[:, 4] = later
    assert np.array_equal(stage.predict_margin(rows), stage.predict_margin(X[:8]))


def test_spread_of_the_last_bits_is_none():
    """A column whose values differ by one unit in the last place holds no scale to divide by."""
    X, y = table()
    X[:, 4] = np.float32(0.1)
    X[::2, 4] = np.nextafter(np.float32(0.1), np.float32(1))
    stage = fitted(X, y)
    rows = X[:8].copy()
    rows[:, 4] = 0.11
    assert np.array_equal(stage.predict_margin(rows), stage.predict_margin(X[:8]))


@pytest.mark.parametrize("unit", [1e-12, 1e25])
def test_the_unit_of_a_column_does_not_matter(unit):
    """A column measured in another unit is standardised to the same inputs: as
    many units in the last place as the product by the unit, its mean and its
    spread have roundings."""
    X, y = table()
    want = fitted(X, y)._inputs(X).cpu().numpy()
    X[:, 2] = X[:, 2] * np.float32(unit)
    stage = ExpertStage(ExpertParams(experts=4, k=2, width=16, inner=16, epochs=0), MSELoss()).fit(X, y)
    got = stage._inputs(X).cpu().numpy()
    assert np.max(np.abs(got - want)) < 1e-5
