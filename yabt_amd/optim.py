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

from array import array
from contextlib import nullcontext
from dataclasses import dataclass
from itertools import chain
from operator import attrgetter

import torch
from torch.autograd import forward_ad

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
        sizes = list(map(_numel, self.first))
        if not sizes:
            return [], []
        lists, dev = _checked(self, sizes)
        held = [(n + 63) // 64 * 64 for n in sizes]
        # both moments' tensors in one buffer, each at a multiple of 256 bytes, all of a size next to its rest
        parts = torch.empty(2 * sum(held), dtype=torch.float32, device=dev).split_with_sizes(
            [m for n, h in zip(sizes, held) for m in (n, h - n)] * 2)[::2]
        flat = parts[:len(sizes)], parts[len(sizes):]
        table = _table(zip(*(map(_pointer, part) for part in (*flat, *lists)), sizes, [0] * len(sizes)))
        expert_ops._call("yabt_adamw_values", dev, len(sizes), table.buffer_info()[0])
        return tuple([v if t.dim() == 1 else v.view(t.shape) for v, t in zip(part, self.first)] for part in flat)


def _table(rows) -> array:
    """yabt_adamw_tensor's fields, eight 64-bit words a tensor, to be held while their address is in use."""
    return array("q", chain.from_iterable(rows))


_TYPES = {32: (torch.float32, torch.float32), 8: (torch.int8, torch.uint8)}
_DTYPE, _SHAPE, _NEEDS = (attrgetter(m) for m in ("dtype", "shape", "requires_grad"))
_numel, _contiguous, _device_number, _pointer = (getattr(torch.Tensor, m) for m in
                                                 ("numel", "is_contiguous", "get_device", "data_ptr"))


def _moments(state: AdamWState) -> list[list[torch.Tensor]]:
    """The state's lists, if they fit each other."""
    lists = [state.first, state.second]
    if (state.first_scale is None) != (state.second_scale is None):
        lists.append([])
    elif state.first_scale is not None:
        lists += [state.first_scale, state.second_scale]
    if any(len(part) != len(state.first) for part in lists):
        raise ValueError("an AdamWState has a tensor of every moment (and of both scales, or of none) for each parameter")
    return lists


def _checked(state: AdamWState, sizes: list[int]) -> tuple[list[list[torch.Tensor]], torch.device]:
    """The moments' lists and their device: of these sizes, contiguous, on one device."""
    lists = _moments(state)
    types = _TYPES[state.bits] + (torch.float32, torch.float32)
    blocks = [-(-n // BLOCK) for n in sizes]
    # over whole lists, as a loop over the tensors takes as long as a step of small ones
    every = list(chain.from_iterable(lists))
    if any(set(map(_DTYPE, part)) != {dt} for part, dt in zip(lists, types)) or \
            any(list(map(_numel, part)) != want for part, want in zip(lists, (sizes, sizes, blocks, blocks))) or \
            not all(map(_contiguous, every)) or len(numbers := set(map(_device_number, every))) != 1 or -1 in numbers:
        _refuse(lists, types, sizes, blocks)
    return lists, every[0].device


def _refuse(lists, types, sizes, blocks) -> None:
    """What is wrong with the moments."""
    for name, part, dt, want in zip(("first moment", "second moment", "first scales", "second scales"), lists, types,
                                    (sizes, sizes, blocks, blocks)):
        for i, (t, n) in enumerate(zip(part, want)):
            if t.dtype != dt or t.numel() != n:
                raise ValueError(f"{name} {i} must be {n} values of {dt}, got {t.numel()} of {t.dtype}")
    for t in chain.from_iterable(lists):
        if not t.is_cuda:
            raise RuntimeError("moments must be on a HIP device: the step has no CPU form")
        if not t.is_contiguous():
            raise ValueError("moments and their scales must be contiguous: they are written in place")
    raise ValueError("all tensors must be on one device")


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
    not finite makes the moments of its 256 values NaN.

    Parameters, moments and scales may not overlap, nor a gradient any of them but its
    own parameter or moment, from the same place on in values of the same width."""
    if not len(params) == len(grads) == len(state.first):
        raise ValueError(f"{len(params)} parameters, {len(grads)} gradients and {len(state.first)} moments")
    b1, b2 = betas
    if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0 and 0.0 <= lr <= 1e30 and 0.0 <= eps <= 1e30
            and 0.0 <= weight_decay <= 1e30):
        raise ValueError(f"betas must be in [0, 1), lr, eps and weight_decay 0 to 1e30, got {betas}, {lr}, {eps}, "
                         f"{weight_decay}")
    if any(g is None for g in grads):
        on = [i for i, g in enumerate(grads) if g is not None]
        some = lambda part: None if part is None else [part[i] for i in on]  # noqa: E731
        _moments(state)
        state = AdamWState(*map(some, (state.first, state.second, state.first_scale, state.second_scale)))
        params, grads = some(params), some(grads)
    if not params:
        _moments(state)
        return
    if torch.is_grad_enabled() and (any(map(_NEEDS, params)) or any(map(_NEEDS, grads))):
        expert_ops._unrecorded()
    if forward_ad._current_level >= 0:
        expert_ops._no_tangents(*params, *grads, *chain.from_iterable(_moments(state)))
    sizes = list(map(_numel, params))
    lists, dev = _checked(state, sizes)
    at, number = 0, 1
    if isinstance(step, torch.Tensor):
        if step.dtype != torch.int32 or step.numel() != 1 or step.device != dev:
            raise ValueError("step must be a number or one int32 on the parameters' device")
        at = step.data_ptr()
    else:
        number = int(step)
        if not 1 <= number < 2 ** 31:
            raise ValueError(f"steps are counted from 1 to 2^31 - 1, got {step}")
        with torch.cuda.device(dev) if torch._C._cuda_getDevice() != dev.index else nullcontext():
            capturing = torch.cuda.is_current_stream_capturing()
        if capturing:
            raise RuntimeError("a captured step would keep its number: pass step as an int32 device tensor")
    if list(map(_SHAPE, params)) != list(map(_SHAPE, grads)):
        raise ValueError(f"gradients must have their parameters' shapes, got {[tuple(g.shape) for g in grads]} for "
                         f"{[tuple(p.shape) for p in params]}")
    if set(map(_device_number, chain(params, grads))) != {dev.index}:
        raise ValueError(f"all tensors must be on {dev}")
    if not all(map(_contiguous, params)):
        raise ValueError("parameters must be contiguous: they are written in place")
    if not all(map(_contiguous, grads)):
        grads = [g.contiguous() for g in grads]          # held until the step is on its way
    try:
        types = [DTYPES[p] | DTYPES[g] << 32 for p, g in zip(map(_DTYPE, params), map(_DTYPE, grads))]
    except KeyError as e:
        raise ValueError(f"parameters and gradients must be float32, bfloat16 or float16, got {e.args[0]}") from None
    where = list(map(_pointer, params))
    none = [0] * len(params)
    first, second, *scales = (list(map(_pointer, part)) for part in lists)
    table = _table(zip(where, map(_pointer, grads), first, second, *(scales or (none, none)), sizes, types))
    try:
        expert_ops._call("yabt_adamw_step", dev, len(params), table.buffer_info()[0], state.bits, number, at, float(lr),
                         float(b1), float(b2), float(eps), float(weight_decay))
    except RuntimeError as e:
        if "tensors overlap" in str(e):
            raise ValueError("a parameter or a moment is in the lists twice, overlaps another, or is overlapped by a "
                             "gradient that is not all its own") from None
        raise
    # also of tensors without a gradient of their own: a backward pass may have kept them
    torch.autograd.graph.increment_version(list(chain(params, *lists)))
