"""Sizes whose launches would have 2^32 threads or more are refused before
anything is launched, and those below are not."""

import pytest

from yabt_amd import _lib


def forward(lib, dt, n, k, D, F, E):
    return lib.yabt_experts(dt, 4096, D, n, k, D, F, E, *[4096] * 8, 1 << 62, 0, 4096, D, None)


def backward(lib, dt, n, k, D, F, E):
    return lib.yabt_experts_grad(dt, 4096, D, 4096, D, n, k, D, F, E, *[4096] * 9, 1 << 62, 4096, D, *[4096] * 3, None)


# 64 x 128 tiles of 256 threads, h's 64 columns of each half; 256 x 256 of 512
@pytest.mark.parametrize("dt,n,k,D,F,E", [(0, 1 << 26, 8, 256, 256, 4), (1, 1 << 26, 8, 256, 256, 4),
                                          (1, 1 << 26, 8, 2048, 2048, 8), (0, 1 << 20, 4, 300, 1 << 20, 2)])
def test_too_many_threads(dt, n, k, D, F, E):
    lib = _lib.load()
    assert lib.yabt_experts_workspace_bytes(dt, n, k, D, F, E) == 0
    assert lib.yabt_experts_grad_workspace_bytes(dt, n, k, D, F, E) == 0
    for call in (forward, backward):
        assert call(lib, dt, n, k, D, F, E) == -1 and "bad sizes" in _lib.last_error()


@pytest.mark.parametrize("dt,n,k,D,F,E", [(0, 1 << 24, 8, 256, 256, 4), (1, 1 << 23, 8, 2048, 2048, 8),
                                          (1, 1 << 20, 2, 2048, 2048, 1024)])
def test_as_many_as_a_launch_takes(dt, n, k, D, F, E):
    lib = _lib.load()
    assert lib.yabt_experts_workspace_bytes(dt, n, k, D, F, E) > 0
    assert lib.yabt_experts_grad_workspace_bytes(dt, n, k, D, F, E) > 0


def test_wide_weights_for_few_rows():
    """The weights' gradients alone need so many tiles: the forward pass of the same sizes runs."""
    lib = _lib.load()
    assert lib.yabt_experts_workspace_bytes(0, 4, 1, 1 << 18, 1 << 18, 4) > 0
    assert lib.yabt_experts_grad_workspace_bytes(0, 4, 1, 1 << 18, 1 << 18, 4) == 0
    assert backward(lib, 0, 4, 1, 1 << 18, 1 << 18, 4) == -1 and "bad sizes" in _lib.last_error()
