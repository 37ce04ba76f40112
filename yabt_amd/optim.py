"""One AdamW step over all tensors of a model (csrc/adamw.hip).

``adamw_state`` makes the moments of a list of parameters, in 32 bits or in 8
(about 2 bytes a value in place of 8), and ``adamw_step`` moves parameters and
moments by one step, in one launch for up to 48 tensors.  ``ExpertStage`` fits
its parameters with it.

Parameters and gradients are float32, bfloat16 or float16, the step's arithmetic
float32.  A call runs on the current stream and neither waits nor reads anything
back; with the step's number in a device tensor it can be captured into a HIP
graph.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from . import expert_ops
from .expert_ops import DTYPES

BLOCK = 256                    # consecutive values of 8-bit moments that share a scale


@dataclass
class AdamWState:
    """Moments, a tensor of each for every parameter, flat or of its shape:
    float32, or int8 (first) and uint8 (second) with a float32 scale for each
    256 values.  In a block with largest magnitude s a code c stands for
    sign(c) (c / 127)^2 s (first) and ((c / 255)^2 s)^2 (second, s being the
    largest square root)."""
    first: list[torch.Tensor]
    second: list[torch.Tensor]
    first_scale: list[torch.Tensor] | None = None
    second_scale: list[torch.Tensor] | None = None

    @property
    def bits(self) -> int:
        return 32 if self.first_scale is None else 8

    def values(self) -> tuple[list[torch.Tensor], list[torch.Tensor]]:
        """The moments as float32: with 32 bits the tensors themselves, with 8
        what they stand for now, in new ones."""
        if self.bits == 32:
            return self.first, self.second
        dev = _state_device(self)
        sizes = [t.numel() for t in self.first]
        held = [(n + 63) // 64 * 64 for n in sizes]
        both = [torch.empty(sum(held), dtype=torch.float32, device=dev).split(held) for _ in range(2)]
        first, second = ([v[:n].view(t.shape) for v, n, t in zip(part, sizes, old)]
                         for part, old in zip(both, (self.first, self.second)))
        rows = [(a.data_ptr(), b.data_ptr(), c.data_ptr(), d.data_ptr(), e.data_ptr(), f.data_ptr(), n, 0)
                for a, b, c, d, e, f, n in zip(first, second, self.first, self.second, self.first_scale,
                                               self.second_scale, sizes)]
        if rows:
            expert_ops._call("yabt_adamw_values", dev, len(rows), _table(rows))
        return first, second


def _table(rows: list[tuple]) -> ctypes.Array:
    """yabt_adamw_tensor's fields, eight 64-bit words a tensor."""
    return (ctypes.c_int64 * (8 * len(rows)))(*[w for row in rows for w in row])


def _state_device(state: AdamWState) -> torch.device:
    """The device of a state whose tensors fit each other."""
    lists = (state.first, state.second, state.first_scale, state.second_scale)
    if state.second_scale is None and state.first_scale is not None or state.first_scale is None and \
            state.second_scale is not None or len({len(part) for part in lists if part is not None}) != 1:
        raise ValueError("an AdamWState has a tensor of every moment (and of both scales, or of none) for each parameter")
    dev = None
    types = (torch.float32, torch.float32) if state.first_scale is None else (torch.int8, torch.uint8)
    for i, m in enumerate(state.first):
        v, n = state.second[i], m.numel()
        if m.dtype != types[0] or v.dtype != types[1] or v.numel() != n:
            raise ValueError(f"moments {i} must be {types[0]} and {types[1]} of one size, got {m.dtype} {tuple(m.shape)} "
                             f"and {v.dtype} {tuple(v.shape)}")
        parts = [m, v]
        if state.first_scale is not None:
            parts += [state.first_scale[i], state.second_scale[i]]
            if any(t.dtype != torch.float32 or t.numel() != -(-n // BLOCK) for t in parts[2:]):
                raise ValueError(f"scales {i} must be {-(-n // BLOCK)} float32 values, one for each {BLOCK}")
        for t in parts:
            if not t.is_cuda:
                raise RuntimeError("moments must be on a HIP device: the step has no CPU form")
            if not t.is_contiguous():
                raise ValueError(f"moments {i} and their scales must be contiguous: they are written in place")
            if dev is None:
                dev = t.device
            elif t.device != dev:
                raise ValueError(f"all tensors must be on {dev}")
    return dev


def adamw_state(params: list[torch.Tensor], bits: int = 32) -> AdamWState:
    """The moments before the first step, zeros, on the parameters' devices."""
    if bits not in (32, 8):
        raise ValueError(f"bits must be 32 or 8, got {bits}")

    def zeros(dtype, size=lambda n: n):
        return [torch.zeros(size(p.numel()), dtype=dtype, device=p.device) for p in params]

    if bits == 32:
        return AdamWState(zeros(torch.float32), zeros(torch.float32))
    blocks = lambda n: -(-n // BLOCK)  # noqa: E731
    return AdamWState(zeros(torch.int8), zeros(torch.uint8), zeros(torch.float32, blocks), zeros(torch.float32, blocks))


def adamw_step(params: list[torch.Tensor], grads: list[torch.Tensor | None], state: AdamWState,
               step: int | torch.Tensor, *, lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999),
               eps: float = 1e-8, weight_decay: float = 0.01) -> None:
    """Step number ``step`` (the first is 1), in place:

        m = m + (1 - b1) (g - m),   v = v + (1 - b2) (g^2 - v)
        p = p (1 - lr weight_decay) - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)

    A parameter whose gradient is None stays as it is, with its moments.  The
    same arithmetic, bit for bit, as torch's lerp_ and addcdiv_ in float32 where
    m / (sqrt(v) + eps sqrt(1 - b2^t)) is scaled by lr sqrt(1 - b2^t) / (1 - b1^t).

    ``step`` may be a device tensor of one int32: it is read when the step runs,
    so that a captured graph that adds one to it counts on (a plain number would
    stay what it was, and is refused while a graph is captured).  With 8-bit
    moments p moves by the moments before they are rounded; a gradient that is
    not finite makes the moments of its 256 values NaN."""
    if not len(params) == len(grads) == len(state.first):
        raise ValueError(f"{len(params)} parameters, {len(grads)} gradients and {len(state.first)} moments")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for part in (params, grads) for t in part):
        expert_ops._unrecorded()
    b1, b2 = betas
    if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0 and 0.0 <= lr <= 1e30 and 0.0 <= eps <= 1e30
            and 0.0 <= weight_decay <= 1e30):
        raise ValueError(f"betas must be in [0, 1), lr, eps and weight_decay 0 to 1e30, got {betas}, {lr}, {eps}, "
                         f"{weight_decay}")
    dev = _state_device(state)
    at, number = 0, 1
    if isinstance(step, torch.Tensor):
        if step.dtype != torch.int32 or step.numel() != 1 or not step.is_cuda or dev is not None and step.device != dev:
            raise ValueError("step must be a number or one int32 on the parameters' device")
        at = step.data_ptr()
    else:
        number = int(step)
        if not 1 <= number < 2 ** 31:
            raise ValueError(f"steps are counted from 1 to 2^31 - 1, got {step}")
        if dev is not None and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a captured step would keep its number: pass step as an int32 device tensor")
    rows, scales, seen, kept = [], state.bits == 8, set(), []
    for i, (p, g) in enumerate(zip(params, grads)):
        if g is None:
            continue
        n = p.numel()
        m, v = state.first[i], state.second[i]
        if p.dtype not in DTYPES or g.dtype not in DTYPES:
            raise ValueError(f"parameter and gradient {i} must be float32, bfloat16 or float16, got {p.dtype}, {g.dtype}")
        if g.shape != p.shape or m.numel() != n:
            raise ValueError(f"parameter {i} has shape {tuple(p.shape)}, its gradient {tuple(g.shape)} and {m.numel()} "
                             "moments")
        if p.device != dev or g.device != dev:
            raise ValueError(f"all tensors must be on {dev}")
        if not p.is_contiguous():
            raise ValueError(f"parameter {i} must be contiguous: it is written in place")
        if not g.is_contiguous():
            g = g.contiguous()
            kept.append(g)                   # until the step is on its way
        where = p.data_ptr()
        if n and (where in seen or seen.add(where)):
            raise ValueError(f"parameter {i} is in the list twice")
        rows.append((where, g.data_ptr(), m.data_ptr(), v.data_ptr(),
                     state.first_scale[i].data_ptr() if scales else 0,
                     state.second_scale[i].data_ptr() if scales else 0, n, DTYPES[p.dtype] | DTYPES[g.dtype] << 32))
    if rows:
        expert_ops._call("yabt_adamw_step", dev, len(rows), _table(rows), state.bits, number, at, float(lr), float(b1),
                         float(b2), float(eps), float(weight_decay))
    for p in params:
        if p.requires_grad:
            torch.autograd.graph.increment_version(p)
