"""Infinite and huge inputs of the stage, in the fit and at prediction."""

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


@pytest.mark.parametrize("bad", [np.inf, -np.inf])
def test_infinite_inputs_are_missing_ones(bad):
    X, y = table()
    X[3, 0], X[1999, 2] = np.nan, np.nan
    want = fitted(X, y)
    Z = X.copy()
    Z[3, 0], Z[1999, 2] = bad, bad
    got = fitted(Z, y)
    assert np.array_equal(got.predict_margin(Z), want.predict_margin(X))
    rows = X[:5].copy()
    rows[:, 1] = np.nan
    other = rows.copy()
    other[:, 1] = bad
    assert np.array_equal(got.predict_margin(other), got.predict_margin(rows))


def test_huge_inputs_leave_a_finite_margin():
    X, y = table()
    stage = fitted(X, y)
    rows = X[:4].copy()
    rows[0, 0], rows[1, 1], rows[2] = 3e38, -3e38, 3e38
    m = stage.predict_margin(rows)
    assert np.isfinite(m).all() and m[3] == stage.predict_margin(X[3:4])[0]


def test_an_infinite_value_in_a_column_without_spread():
    X, y = table()
    X[:, 4] = 0.0
    stage = fitted(X, y)
    rows = X[:8].copy()
    rows[::2, 4], rows[1::2, 4] = np.inf, -np.inf
    assert np.array_equal(stage.predict_margin(rows), stage.predict_margin(X[:8]))
