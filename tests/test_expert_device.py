"""The device that the expert layer's calls are launched on, without a device."""

from __future__ import annotations

import contextlib

import pytest
import torch

from yabt_amd import ExpertParams, ExpertStage, MSELoss, _lib, expert_ops


def test_launches_on_the_tensors_device(monkeypatch):
    """A call whose tensors lie on another device than the current one runs with
    theirs current; one on the current device is called as it is."""
    now, seen = [0], []

    @contextlib.contextmanager
    def device(dev):
        before, now[0] = now[0], torch.device(dev).index
        yield
        now[0] = before

    class Lib:
        @staticmethod
        def yabt_layer_norm(*args):
            seen.append((now[0], args))
            return 0

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: now[0], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 100 + index, raising=False)
    monkeypatch.setattr(_lib, "load", lambda: Lib)
    expert_ops._call("yabt_layer_norm", torch.device("cuda:1"), 5, 6)
    expert_ops._call("yabt_layer_norm", torch.device("cuda:0"), 7)
    assert seen == [(1, (5, 6, 101)), (0, (7, 100))] and now == [0]


def test_a_failed_launch_raises_and_leaves_the_device(monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)
    with pytest.raises(RuntimeError, match="bad sizes"):
        expert_ops._call("yabt_layer_norm", torch.device("cuda:0"), 0, 16, 7, 4, 8, 0, 0, 1e-5, 16, 8, 0, 0)


def test_the_stage_works_on_its_own_device(monkeypatch):
    now, seen = [0], []

    @contextlib.contextmanager
    def device(dev):
        before, now[0] = now[0], torch.device(dev).index
        yield
        now[0] = before

    class Stage(ExpertStage):
        def _fit(self, *args):
            seen.append(("fit", now[0]))

        def _inputs(self, X):
            seen.append(("inputs", now[0]))
            return torch.zeros(0, 3)

    monkeypatch.setattr(torch.cuda, "device", device)
    stage = Stage(ExpertParams(device="cuda:2"), MSELoss()).fit([[1.0]], [1.0])
    stage.predict_margin([[1.0]])
    assert seen == [("fit", 2), ("inputs", 2)] and now == [0] and stage.device_ == torch.device("cuda:2")
