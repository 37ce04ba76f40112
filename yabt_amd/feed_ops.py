"""The dense stage's operations on torch tensors (csrc/feed.hip).

Beside its routed experts a layer may have a block that every row passes.

* ``feed_forward`` / ``feed_forward_grad``: that block, gated, and its gradients;
* ``quantize_rows``: rows in 8 bits with a scale each;
* ``product_int8``: rows in 8 bits times a weight in 8 bits;
* ``feed_forward_int8``: the block with both its weights in 8 bits.

Values are float32, bfloat16 or float16, sums float32, those of 8-bit codes exact.
Every call runs on the current stream and neither waits nor reads anything back, so
it can be captured into a HIP graph.  Autograd does not see these calls: a tensor
that requires a gradient is refused while it records, and one with a tangent, as in ``expert_ops``.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _lib
from .expert_ops import DTYPES, _at, _call, _ld, _matrix, _no_tangents, _unrecorded, _vector

ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2, "relu": 3}
MAX_INT8_TERMS = 131071        # of a sum of 8-bit products that stays in 32 bits


def _activation(activation: str) -> int:
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    return ACTIVATIONS[activation]


def _weight(t: torch.Tensor, what: str, dtype: torch.dtype, dev: torch.device) -> torch.Tensor:
    """t as a contiguous device matrix."""
    if t.dim() != 2:
        raise ValueError(f"{what} must be a matrix, got shape {tuple(t.shape)}")
    if t.dtype != dtype:
        raise ValueError(f"{what} must be {dtype}, got {t.dtype}")
    if t.device != dev:
        raise ValueError(f"{what} must be on {dev}")
    return t.contiguous()


def _block(x, w_in, w_out, dtype):
    """Checked tensors and sizes of a block: (x, w_in, w_out, n, D, F, O)."""
    x = _matrix(x, "x")
    (n, D), dev = x.shape, x.device
    w_in = _weight(w_in, "w_in", dtype or x.dtype, dev)
    w_out = _weight(w_out, "w_out", dtype or x.dtype, dev)
    O, F = w_out.shape
    if min(D, F, O) < 1 or tuple(w_in.shape) != (2 * F, D):
        raise ValueError(f"w_in and w_out must be (2 F, {D}) and (O, F), got {tuple(w_in.shape)}, {tuple(w_out.shape)}")
    return x, w_in, w_out, n, D, F, O


def feed_forward(x: torch.Tensor, w_in: torch.Tensor, w_out: torch.Tensor, *, activation: str = "silu",
                 keep_inner: bool = False):
    """y (n, O) = (act(g) * u) w_out^T with [g u] = x w_in^T, in x's type.

    x (n, D), w_in (2 F, D): F gate rows, then F rows of u, w_out (O, F), all of x's
    type.  ``activation``: "silu", "gelu" (by the normal distribution function),
    "gelu_tanh" (its usual approximation) or "relu".  With ``keep_inner`` returns
    (y, inner), inner a buffer for the backward pass: g and u in float32 and act(g) * u.

    16-bit types round act(g) * u to theirs before w_out, and the inner gradients; small
    blocks (24 / F + 6 / min(D, O) > n / 128) keep 16 bits of them, and y of 16 rows or fewer
    (n F O <= 2^26) of act(g) * u; what they are multiplied by there, a weight, x or dy, counts
    as NaN where it is infinite.  In float16 an act(g) * u beyond 65504 makes its row infinite or NaN.
    In float32 an infinite x or weight may count as NaN, and of more than 64 rows x, weights
    and act(g) * u below 2^-110 are taken to 2^-133 (their gradients' factors too)."""
    if x.requires_grad or w_in.requires_grad or w_out.requires_grad:
        _unrecorded()
    if forward_ad._current_level >= 0:
        _no_tangents(x, w_in, w_out)
    act = _activation(activation)
    x, w_in, w_out, n, D, F, O = _block(x, w_in, w_out, None)
    dev, dt, lib = x.device, DTYPES[x.dtype], _lib.load()
    nbytes = lib.yabt_feed_forward_workspace_bytes(dt, n, D, F, O)
    if nbytes == 0:
        raise ValueError("feed_forward: sizes out of range (D, F, O <= 2^24, n < 2^31 - 256, tiles of fewer than 2^32 "
                         "threads)")
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    y = torch.empty((n, O), dtype=x.dtype, device=dev)
    inner = None
    if keep_inner:
        inner = torch.empty(lib.yabt_feed_forward_inner_bytes(dt, n, D, F, O), dtype=torch.uint8, device=dev)
    _call("yabt_feed_forward", dev, dt, act, x.data_ptr(), _ld(x), n, D, F, O, w_in.data_ptr(), w_out.data_ptr(),
          ws.data_ptr(), nbytes, _at(inner), y.data_ptr(), O)
    return (y, inner) if keep_inner else y


def feed_forward_grad(dy: torch.Tensor, x: torch.Tensor, w_in: torch.Tensor, w_out: torch.Tensor,
                      inner: torch.Tensor, *, activation: str = "silu"):
    """(dx, dw_in, dw_out) of ``feed_forward`` from dy (n, O) and the inner it
    kept, all in x's type.  In float16 the inner gradients have its range too:
    scale dy for them and the results back."""
    if dy.requires_grad or x.requires_grad or w_in.requires_grad or w_out.requires_grad:
        _unrecorded()
    if forward_ad._current_level >= 0:
        _no_tangents(dy, x, w_in, w_out)
    act = _activation(activation)
    x, w_in, w_out, n, D, F, O = _block(x, w_in, w_out, None)
    dy = _matrix(dy, "dy", x.dtype)
    dev, dt, lib = x.device, DTYPES[x.dtype], _lib.load()
    if tuple(dy.shape) != (n, O) or dy.device != dev:
        raise ValueError(f"dy must have shape {(n, O)} on {dev}, got {tuple(dy.shape)}")
    nbytes = int(lib.yabt_feed_forward_grad_workspace_bytes(dt, n, D, F, O))
    if nbytes == 0:
        raise ValueError("feed_forward_grad: sizes out of range (D, F, O <= 2^24, n < 2^31 - 256, tiles of fewer than 2^32 "
                         "threads)")
    size = int(lib.yabt_feed_forward_inner_bytes(dt, n, D, F, O))
    if inner.dtype != torch.uint8 or tuple(inner.shape) != (size,) or inner.device != dev or \
            not inner.is_contiguous() or inner.data_ptr() % 256:
        raise ValueError(f"inner must be what feed_forward kept, {size} bytes on {dev} from a multiple of 256 on")
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    dx = torch.empty((n, D), dtype=x.dtype, device=dev)
    dw_in, dw_out = torch.empty_like(w_in), torch.empty_like(w_out)
    _call("yabt_feed_forward_grad", dev, dt, act, dy.data_ptr(), _ld(dy), x.data_ptr(), _ld(x), n, D, F, O,
          w_in.data_ptr(), w_out.data_ptr(), inner.data_ptr(), ws.data_ptr(), nbytes, dx.data_ptr(), D,
          dw_in.data_ptr(), dw_out.data_ptr())
    return dx, dw_in, dw_out


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scale), (n, D) int8 and (n,) float32: x's rows in steps of a 127th
    of the row's largest magnitude m, codes round(x * (127 / m)) with ties to even,
    scale m / 127.  Rows below 2^-100 become zeros; a row that is not finite has
    scale NaN.  Of a weight (O, D), its rows are the output's channels."""
    if x.requires_grad:
        _unrecorded()
    if forward_ad._current_level >= 0:
        _no_tangents(x)
    x = _matrix(x, "x")
    (n, D), dev = x.shape, x.device
    if D < 1 or n >= 1 << 24 or D > 1 << 24:
        raise ValueError(f"quantize_rows takes less than 2^24 rows of 1 to 2^24 values, got {(n, D)}")
    codes = torch.empty((n, D), dtype=torch.int8, device=dev)
    scale = torch.empty(n, dtype=torch.float32, device=dev)
    _call("yabt_quantize_rows", dev, DTYPES[x.dtype], x.data_ptr(), _ld(x), n, D, codes.data_ptr(), D, scale.data_ptr())
    return codes, scale


def _codes(t: torch.Tensor, what: str) -> torch.Tensor:
    if t.dim() != 2 or t.dtype != torch.int8:
        raise ValueError(f"{what} must be an int8 matrix, got {tuple(t.shape)} {t.dtype}")
    if not t.is_cuda:
        raise RuntimeError(f"{what} must be on a HIP device: the dense stage has no CPU form")
    rows, cols = t.shape
    if rows > 1 and t.stride(0) < cols or cols > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t


def product_int8(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor,
                 dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """y (n, N) in ``dtype``: y_io = a_scale_i (b_scale_o sum_k a_ik b_ok).

    a (n, K) int8 with a scale for each row, as ``quantize_rows`` gives them, b
    (N, K) int8 with one for each output channel.  The sums are exact (K up to
    131071) and rounded to float32 once."""
    if a_scale.requires_grad or b_scale.requires_grad:
        _unrecorded()
    if forward_ad._current_level >= 0:
        _no_tangents(a_scale, b_scale)
    if dtype not in DTYPES:
        raise ValueError(f"dtype must be float32, bfloat16 or float16, got {dtype}")
    a, b = _codes(a, "a"), _codes(b, "b")
    (n, K), N, dev = a.shape, b.shape[0], a.device
    if b.shape[1] != K or b.device != dev:
        raise ValueError(f"b must be (N, {K}) on {dev}, got {tuple(b.shape)} on {b.device}")
    sa, sb = _vector(a_scale, n, dev, "a_scale"), _vector(b_scale, N, dev, "b_scale")
    lib = _lib.load()
    nbytes = lib.yabt_product_int8_workspace_bytes(n, K, N)
    if nbytes == 0:
        raise ValueError(f"product_int8: sizes out of range (K 1 to {MAX_INT8_TERMS}, N 1 to 2^24, n < 2^24), got "
                         f"{(n, K)} and {(N, K)}")
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes > 1 else None
    y = torch.empty((n, N), dtype=dtype, device=dev)
    _call("yabt_product_int8", dev, a.data_ptr(), _ld(a), sa.data_ptr(), n, K, b.data_ptr(), _ld(b), sb.data_ptr(), N,
          DTYPES[dtype], _at(ws), nbytes, y.data_ptr(), N)
    return y


def feed_forward_int8(x: torch.Tensor, w_in: torch.Tensor, in_scale: torch.Tensor, w_out: torch.Tensor,
                      out_scale: torch.Tensor, *, activation: str = "silu") -> torch.Tensor:
    """``feed_forward`` with its weights in 8 bits, each ``quantize_rows`` of the
    weight: x's rows are put in 8 bits, g, u and h = act(g) * u are float32, act(g) off
    by up to (20 + 2 g^2) 2^-24 of itself (gelu) or (8 + 10 |z|) 2^-24, z the sigmoid's
    argument, and h's rows are put in 8 bits before w_out.  y (n, O) in x's type."""
    if x.requires_grad or in_scale.requires_grad or out_scale.requires_grad:
        _unrecorded()
    if forward_ad._current_level >= 0:
        _no_tangents(x, in_scale, out_scale)
    act = _activation(activation)
    x, w_in, w_out, n, D, F, O = _block(x, w_in, w_out, torch.int8)
    dev, lib = x.device, _lib.load()
    si, so = _vector(in_scale, 2 * F, dev, "in_scale"), _vector(out_scale, O, dev, "out_scale")
    nbytes = lib.yabt_feed_forward_int8_workspace_bytes(n, D, F, O)
    if nbytes == 0:
        raise ValueError(f"feed_forward_int8: sizes out of range (D, F <= {MAX_INT8_TERMS}, n < 2^24)")
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    y = torch.empty((n, O), dtype=x.dtype, device=dev)
    _call("yabt_feed_forward_int8", dev, DTYPES[x.dtype], act, x.data_ptr(), _ld(x), n, D, F, O, w_in.data_ptr(),
          si.data_ptr(), w_out.data_ptr(), so.data_ptr(), ws.data_ptr(), nbytes, y.data_ptr(), O)
    return y
