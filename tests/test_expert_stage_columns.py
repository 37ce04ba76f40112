"""The stage's column statistics on the CPU: those of the finite values, the same
bits as plain sums for ordinary columns, and no spread where there is none."""

import torch

from yabt_amd.expert_stage import _statistics

INF = float("inf")


def test_ordinary_columns_have_plain_statistics():
    raw = torch.randn((3000, 9), generator=torch.Generator().manual_seed(0)) * 3 + 1
    raw[5, 2] = float("nan")
    seen = ~torch.isnan(raw)
    count = seen.sum(dim=0)
    mean = torch.where(seen, raw, 0.0).sum(dim=0) / count
    spread = torch.where(seen, raw - mean, 0.0).square().sum(dim=0) / count
    got_mean, got_std = _statistics(raw)
    assert torch.equal(got_mean, mean) and torch.equal(got_std, spread.sqrt())
    raw[7, 3], raw[8, 3] = INF, -INF
    clean = raw.clone()
    clean[7, 3], clean[8, 3] = float("nan"), float("nan")
    assert all(torch.equal(a, b) for a, b in zip(_statistics(raw), _statistics(clean)))


def test_columns_without_spread():
    raw = torch.randn((400, 7), generator=torch.Generator().manual_seed(1))
    raw[:, 0], raw[:, 1], raw[:, 2], raw[:, 3] = 0.0, 0.1, float("nan"), INF
    raw[:, 4] = torch.tensor([1.0, 1.0 + 2.0 ** -23]).repeat(200)
    raw[:, 5] = torch.tensor([1e6, 1e6 + 1.0]).repeat(200)          # small beside its values, and real
    mean, std = _statistics(raw)
    assert std[:5].tolist() == [INF] * 5 and torch.isfinite(std[5:]).all() and torch.isfinite(mean).all()
    assert abs(std[5].item() - 0.5) < 0.1
    assert _statistics(raw[:0])[1].tolist() == [INF] * 7 and _statistics(raw[:1])[1].tolist() == [INF] * 7


def test_columns_in_any_unit():
    raw = torch.randn((400, 3), generator=torch.Generator().manual_seed(2))
    mean, std = _statistics(raw)
    for power in (-100, 100):
        m, s = _statistics(raw * 2.0 ** power)
        assert torch.equal(m, mean * 2.0 ** power) and torch.equal(s, std * 2.0 ** power)
