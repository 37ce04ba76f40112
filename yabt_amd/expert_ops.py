"""The expert layer's operations on torch tensors (csrc/norm.hip, route.hip,
experts.hip).

Rows are normalised, a gate's scores route each row to k of E experts, and the
experts' weighted answers are added up: the learned, soft form of a tree with
models in its leaves (yabt/neural_leaves.py:93-184), which sends a row to one
leaf.

* ``layer_norm`` / ``layer_norm_grad``: rows to zero mean and unit variance,
  times a weight, plus a bias;
* ``route`` / ``route_grad``: the k best experts of each row and their weights;
* ``expert_plan``: the (row, expert) slots sorted by expert;
* ``expert_products`` / ``expert_products_grad``: what the experts answer.

Values are float32, bfloat16 or float16; statistics, weights, parameters of
the norm and all sums are float32.  Every call runs on the current stream and
neither waits nor reads anything back, so it can be captured into a HIP graph.

Autograd does not see these calls: a program takes the gradients from the
``_grad`` functions itself.  A tensor that requires a gradient is therefore
refused while autograd records; under ``torch.no_grad()``, as in a backward pass
of one's own, it is taken as it is.  A dual tensor with a tangent (forward mode) is refused too.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch
from torch.autograd import forward_ad

from . import _lib

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
SCORES = {"softmax": 0, "sigmoid": 1}
MAX_EXPERTS, MAX_K, MAX_GROUPS = 1024, 32, 64


def _call(name: str, dev: torch.device, *args) -> None:
    """The library's ``name`` with args and dev's current stream, dev being the
    current device meanwhile: the default stream's handle is 0 on every device,
    and a launch on it goes to the current one.  ``torch.cuda.current_stream``
    takes 2 us to make an object of the handle and ``torch.cuda.device`` more,
    which a call for one row would notice."""
    call, index = getattr(_lib.load(), name), dev.index
    if torch._C._cuda_getDevice() == index:
        rc = call(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(dev):
            rc = call(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check(rc, name)


def _unrecorded() -> None:
    """A call's tensor requires a gradient, which autograd would silently not get."""
    if torch.is_grad_enabled():
        raise RuntimeError("these calls are not recorded by autograd, and a tensor requires a gradient: "
                           "call them under torch.no_grad() and take the gradients from the _grad functions, or "
                           "detach it")


def _no_tangents(*tensors: torch.Tensor | None) -> None:
    """The same for forward mode, whose dual tensors require no gradient: called while a level of it is open."""
    if torch._C._is_fwd_grad_enabled() and any(t is not None and forward_ad.unpack_dual(t).tangent is not None
                                               for t in tensors):
        raise RuntimeError("these calls are not seen by autograd's forward mode, and a tensor has a tangent: pass the "
                           "primal (torch.autograd.forward_ad.unpack_dual), and make the tangent from the formulas")


def _matrix(t: torch.Tensor, what: str, dtype: torch.dtype | None = None) -> torch.Tensor:
    """t as a device matrix with unit column stride."""
    if t.dim() != 2:
        raise ValueError(f"{what} must be a matrix, got shape {tuple(t.shape)}")
    if not t.is_cuda:
        raise RuntimeError(f"{what} must be on a HIP device: this call has no CPU form")
    if t.dtype not in DTYPES or (dtype is not None and t.dtype != dtype):
        raise ValueError(f"{what} must be {dtype or 'float32, bfloat16 or float16'}, got {t.dtype}")
    rows, cols = t.shape
    if rows > 1 and t.stride(0) < cols or cols > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t


def _ld(t: torch.Tensor) -> int:
    return max(t.stride(0), t.shape[1]) if t.shape[0] > 1 else t.shape[1]


def _vector(t: torch.Tensor | None, size: int, dev: torch.device, what: str) -> torch.Tensor | None:
    """t as a contiguous float32 vector on dev."""
    if t is None:
        return None
    if t.dim() != 1 or t.shape[0] != size:
        raise ValueError(f"{what} must have shape ({size},), got {tuple(t.shape)}")
    if t.device != dev:
        raise ValueError(f"{what} must be on {dev}")
    return t if t.dtype == torch.float32 and t.is_contiguous() else t.float().contiguous()


def _at(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, mean, rstd) of the rows of x (n, D): y = (x - mean) * rstd * weight
    + bias in x's type, mean and rstd (n,) float32 for the backward pass."""
    if x.requires_grad or weight is not None and weight.requires_grad or bias is not None and bias.requires_grad:
        _unrecorded()
    if forward_ad._current_level >= 0:
        _no_tangents(x, weight, bias)
    x = _matrix(x, "x")
    (n, D), dev = x.shape, x.device
    if D == 0:
        raise ValueError("layer_norm needs at least one column")
    w, b = _vector(weight, D, dev, "weight"), _vector(bias, D, dev, "bias")
    y = torch.empty((n, D), dtype=x.dtype, device=dev)
    mean, rstd = torch.empty((2, n), dtype=torch.float32, device=dev).unbind()
    _call("yabt_layer_norm", dev, DTYPES[x.dtype], x.data_ptr(), _ld(x), n, D, _at(w), _at(b), float(eps),
          y.data_ptr(), D, mean.data_ptr(), rstd.data_ptr())
    return y, mean, rstd


def layer_norm_grad(dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                    weight: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dweight, dbias) of ``layer_norm`` at x, from dy and the mean and
    rstd it returned: dx in x's type, dweight and dbias (D,) float32."""
    if any(t is not None and t.requires_grad for t in (dy, x, mean, rstd, weight)):
        _unrecorded()
    if forward_ad._current_level >= 0:
        _no_tangents(dy, x, mean, rstd, weight)
    x = _matrix(x, "x")
    dy = _matrix(dy, "dy", x.dtype)
    (n, D), dev = x.shape, x.device
    if dy.shape != x.shape or dy.device != dev:
        raise ValueError(f"dy must be like x, {tuple(x.shape)} on {dev}")
    w, mu, rs = _vector(weight, D, dev, "weight"), _vector(mean, n, dev, "mean"), _vector(rstd, n, dev, "rstd")
    if mu is None or rs is None:
        raise ValueError("layer_norm_grad needs the mean and rstd of the forward pass")
    lib = _lib.load()
    nbytes = int(lib.yabt_layer_norm_grad_workspace_bytes(n, D))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    dx = torch.empty((n, D), dtype=x.dtype, device=dev)
    dw, db = torch.empty((2, D), dtype=torch.float32, device=dev).unbind()
    _call("yabt_layer_norm_grad", dev, DTYPES[x.dtype], dy.data_ptr(), _ld(dy), x.data_ptr(), _ld(x), n, D, _at(w),
          mu.data_ptr(), rs.data_ptr(), ws.data_ptr(), nbytes, dx.data_ptr(), D, dw.data_ptr(), db.data_ptr())
    return dx, dw, db


def _scores(scores: str) -> int:
    if scores not in SCORES:
        raise ValueError(f"scores must be one of {sorted(SCORES)}, got {scores!r}")
    return SCORES[scores]


def route(logits: torch.Tensor, k: int, *, scores: str = "softmax", bias: torch.Tensor | None = None,
          groups: int = 1, keep_groups: int = 1, renormalise: bool = True,
          scale: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """(ids, weights), (n, k) int32 and float32: the k best of each row's E
    experts, best first, equal keys by the lower index.

    An expert's key is logit + bias ("softmax") or sigmoid(logit) + bias
    ("sigmoid"), in float32; the bias (for balance) changes the choice alone.
    A logit of -inf or NaN closes the expert to the row; a slot that no expert
    is left for has id -1 and weight 0.  With groups > 1 only the best
    ``keep_groups`` groups of E / groups consecutive experts stay, by their
    largest key ("softmax") or the sum of their two largest ("sigmoid").
    Weights are scale * score, with ``renormalise`` divided by the sum of the
    row's chosen scores."""
    if logits.requires_grad or bias is not None and bias.requires_grad:
        _unrecorded()
    if forward_ad._current_level >= 0:
        _no_tangents(logits, bias)
    logits = _matrix(logits, "logits")
    (n, E), dev = logits.shape, logits.device
    how = _scores(scores)
    if not 1 <= E <= MAX_EXPERTS:
        raise ValueError(f"route takes 1 to {MAX_EXPERTS} experts, got {E}")
    if not 1 <= k <= min(E, MAX_K):
        raise ValueError(f"k must be 1 to {min(E, MAX_K)}, got {k}")
    if not 1 <= groups <= MAX_GROUPS or E % groups or not 1 <= keep_groups <= groups:
        raise ValueError(f"groups must divide {E} and be at most {MAX_GROUPS}, keep_groups 1 to groups; "
                         f"got {groups}, {keep_groups}")
    b = _vector(bias, E, dev, "bias")
    ids = torch.empty((n, k), dtype=torch.int32, device=dev)
    weights = torch.empty((n, k), dtype=torch.float32, device=dev)
    _call("yabt_route", dev, DTYPES[logits.dtype], logits.data_ptr(), _ld(logits), n, E, int(k), how, _at(b),
          int(groups), int(keep_groups), int(bool(renormalise)), float(scale), ids.data_ptr(), weights.data_ptr())
    return ids, weights


def route_grad(dweights: torch.Tensor, logits: torch.Tensor, ids: torch.Tensor, *, scores: str = "softmax",
               renormalise: bool = True, scale: float = 1.0) -> torch.Tensor:
    """Gradient of ``route``'s weights in the logits, (n, E) in their type, the
    choice (ids) held fixed; a balancing bias has none."""
    if dweights.requires_grad or logits.requires_grad:
        _unrecorded()
    if forward_ad._current_level >= 0:
        _no_tangents(dweights, logits)
    logits = _matrix(logits, "logits")
    (n, E), dev = logits.shape, logits.device
    how = _scores(scores)
    ids = _ids(ids, dev)
    k = ids.shape[1]
    if ids.shape[0] != n or not 1 <= E <= MAX_EXPERTS or not 1 <= k <= min(E, MAX_K):
        raise ValueError(f"ids must be route's, (n, k) for logits {tuple(logits.shape)}; got {tuple(ids.shape)}")
    if tuple(dweights.shape) != (n, k) or dweights.device != dev:
        raise ValueError(f"dweights must have shape {(n, k)} on {dev}")
    dweights = _matrix(dweights if dweights.dtype == torch.float32 else dweights.float(), "dweights")
    out = torch.empty((n, E), dtype=logits.dtype, device=dev)
    _call("yabt_route_grad", dev, DTYPES[logits.dtype], dweights.data_ptr(), _ld(dweights), logits.data_ptr(),
          _ld(logits), ids.data_ptr(), n, E, k, how, int(bool(renormalise)), float(scale), out.data_ptr(), E)
    return out


def _ids(ids: torch.Tensor, dev: torch.device | None = None) -> torch.Tensor:
    if ids.dim() != 2 or ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"ids must be an (n, k) integer matrix, got {tuple(ids.shape)} {ids.dtype}")
    if not ids.is_cuda or dev is not None and ids.device != dev:
        raise RuntimeError("ids must be on the other tensors' HIP device")
    # a wider id names no expert: it must not come out as one
    return (ids if ids.dtype == torch.int32 else ids.clamp(-1, 2 ** 31 - 1).to(torch.int32)).contiguous()


@dataclass
class ExpertPlan:
    """Slots (row * k + j) sorted by expert.  Expert e's are ``slots[offsets[e]
    : offsets[e + 1]]``, in row order, and ``rows`` their rows; the places
    after the last hold -1, as many as there are ids that name no expert.  ids
    are kept, not copied: they stay as they are while the plan is in use."""
    ids: torch.Tensor       # (n, k) int32
    offsets: torch.Tensor   # (E + 1,) int32
    slots: torch.Tensor     # (n k,) int32
    rows: torch.Tensor      # (n k,) int32

    @property
    def experts(self) -> int:
        return self.offsets.shape[0] - 1


def expert_plan(ids: torch.Tensor, experts: int) -> ExpertPlan:
    """The plan of ids (n, k); ids outside [0, experts) belong to no expert."""
    ids = _ids(ids)
    (n, k), dev = ids.shape, ids.device
    lib, experts = _lib.load(), int(experts)
    nbytes = lib.yabt_expert_plan_workspace_bytes(n, k, experts)
    if nbytes == 0:
        raise ValueError(f"expert_plan takes 1 to {MAX_EXPERTS} experts, k >= 1 and n k < 2^31; got {experts} "
                         f"experts, ids {(n, k)}")
    # one allocation: the plan's three arrays and the call's workspace behind them
    sizes = (experts + 1, n * k, n * k, nbytes // 4)
    offsets, slots, rows, ws = torch.empty(sum(sizes), dtype=torch.int32, device=dev).split_with_sizes(sizes)
    _call("yabt_expert_plan", dev, ids.data_ptr(), n, k, experts, ws.data_ptr(), nbytes, offsets.data_ptr(),
          slots.data_ptr(), rows.data_ptr())
    return ExpertPlan(ids, offsets, slots, rows)


def _expert_args(x, plan, weights, w_in, w_out):
    """Checked sizes and tensors of the products: (x, weights, w_in, w_out, n, k, D, F, E)."""
    x = _matrix(x, "x")
    (n, D), dev, dt = x.shape, x.device, x.dtype
    if w_in.dim() != 3 or w_out.dim() != 3 or w_in.shape[0] != w_out.shape[0] or w_out.shape[1] != D or D < 1 \
            or w_in.shape[2] != D or w_out.shape[2] < 1 or w_in.shape[1] != 2 * w_out.shape[2]:
        raise ValueError(f"w_in and w_out must be (E, 2 F, {D}) and (E, {D}, F), got {tuple(w_in.shape)}, "
                         f"{tuple(w_out.shape)}")
    E, _, F = w_out.shape
    if w_in.dtype != dt or w_out.dtype != dt:
        raise ValueError(f"x, w_in and w_out must have one type, got {dt}, {w_in.dtype}, {w_out.dtype}")
    ids = plan.ids
    k = ids.shape[1]
    if plan.offsets.shape[0] != E + 1 or ids.shape[0] != n:
        raise ValueError(f"the plan is for {plan.experts} experts and {ids.shape[0]} rows, not {E} and {n}")
    if weights.shape != ids.shape:
        raise ValueError(f"weights must have shape {(n, k)}, got {tuple(weights.shape)}")
    if w_in.device != dev or w_out.device != dev or weights.device != dev or ids.device != dev:
        raise ValueError(f"all tensors must be on {dev}")
    if weights.dtype != torch.float32:
        weights = weights.float()
    return x, weights.contiguous(), w_in.contiguous(), w_out.contiguous(), n, k, D, F, E


def _inner_width(F: int) -> int:
    return 2 * ((F + 3) // 4 * 4)


def expert_products(x: torch.Tensor, plan: ExpertPlan, weights: torch.Tensor, w_in: torch.Tensor,
                    w_out: torch.Tensor, keep_inner: bool = False):
    """y (n, D) in x's type: y_t = sum over row t's slots of weights * w_out[e]
    (silu(g) * u) with [g u] = w_in[e] x_t, e the slot's expert.

    w_in (E, 2 F, D) holds each expert's F gate rows, then its F rows of u;
    w_out (E, D, F); both of x's type.  weights (n, k) as ``route`` gives them.
    A row none of whose slots has an expert gets zeros.  With ``keep_inner``
    returns (y, inner), inner (n k, 2 G) float32, G being F up to a multiple of
    4: g and u by the plan's places, which the backward pass takes.

    16-bit types round silu(g) * u to theirs before w_out, which float32 does
    not; in float16 one beyond 65504 makes its row infinite or NaN."""
    if x.requires_grad or weights.requires_grad or w_in.requires_grad or w_out.requires_grad:
        _unrecorded()
    if forward_ad._current_level >= 0:
        _no_tangents(x, weights, w_in, w_out)
    x, weights, w_in, w_out, n, k, D, F, E = _expert_args(x, plan, weights, w_in, w_out)
    dev, dt, lib = x.device, DTYPES[x.dtype], _lib.load()
    nbytes = lib.yabt_experts_workspace_bytes(dt, n, k, D, F, E)
    if nbytes == 0:
        raise ValueError("expert_products: sizes out of range (D, F <= 2^24, n k < 2^31)")
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    y = torch.empty((n, D), dtype=x.dtype, device=dev)
    inner = torch.empty((n * k, _inner_width(F)), dtype=torch.float32, device=dev) if keep_inner else None
    _call("yabt_experts", dev, dt, x.data_ptr(), _ld(x), n, k, D, F, E, plan.ids.data_ptr(), plan.offsets.data_ptr(),
          plan.slots.data_ptr(), plan.rows.data_ptr(), weights.data_ptr(), w_in.data_ptr(), w_out.data_ptr(),
          ws.data_ptr(), nbytes, _at(inner), y.data_ptr(), D)
    return (y, inner) if keep_inner else y


def expert_products_grad(dy: torch.Tensor, x: torch.Tensor, plan: ExpertPlan, weights: torch.Tensor,
                         w_in: torch.Tensor, w_out: torch.Tensor, inner: torch.Tensor):
    """(dx, dweights, dw_in, dw_out) of ``expert_products`` from dy (n, D) and
    the inner it kept: dx, dw_in and dw_out in x's type, dweights (n, k)
    float32, 0 for slots without an expert.  In float16 the inner gradients have
    its range too: scale dy for them and the results back."""
    if dy.requires_grad or x.requires_grad or weights.requires_grad or w_in.requires_grad or w_out.requires_grad or \
            inner.requires_grad:
        _unrecorded()
    if forward_ad._current_level >= 0:
        _no_tangents(dy, x, weights, w_in, w_out, inner)
    x, weights, w_in, w_out, n, k, D, F, E = _expert_args(x, plan, weights, w_in, w_out)
    dy = _matrix(dy, "dy", x.dtype)
    dev, dt, lib = x.device, DTYPES[x.dtype], _lib.load()
    if dy.shape != x.shape or dy.device != dev:
        raise ValueError(f"dy must be like x, {tuple(x.shape)} on {dev}")
    if tuple(inner.shape) != (n * k, _inner_width(F)) or inner.dtype != torch.float32 or not inner.is_contiguous() \
            or inner.device != dev or inner.data_ptr() % 16:
        raise ValueError(f"inner must be what expert_products kept, {(n * k, _inner_width(F))} float32 on {dev}")
    nbytes = int(lib.yabt_experts_grad_workspace_bytes(dt, n, k, D, F, E))
    if nbytes == 0:
        raise ValueError("expert_products_grad: sizes out of range (D, F <= 2^24, n k < 2^31)")
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    dx = torch.empty((n, D), dtype=x.dtype, device=dev)
    dweights = torch.empty((n, k), dtype=torch.float32, device=dev)
    dw_in, dw_out = torch.empty_like(w_in), torch.empty_like(w_out)
    _call("yabt_experts_grad", dev, dt, dy.data_ptr(), _ld(dy), x.data_ptr(), _ld(x), n, k, D, F, E,
          plan.ids.data_ptr(), plan.offsets.data_ptr(), plan.slots.data_ptr(), plan.rows.data_ptr(),
          weights.data_ptr(), w_in.data_ptr(), w_out.data_ptr(), inner.data_ptr(), ws.data_ptr(), nbytes,
          dx.data_ptr(), D, dweights.data_ptr(), dw_in.data_ptr(), dw_out.data_ptr())
    return dx, dweights, dw_in, dw_out
