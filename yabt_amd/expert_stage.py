"""One more stage on a booster's margin: a layer of routed experts.

Boosting adds stages to a margin, each fitted to the loss's gradient where the
margin stands.  ``ExpertStage`` is such a stage whose model is not a tree with
a model in each leaf (yabt/neural_leaves.py:93-184) but its learned, soft form:
a gate routes every row to k of E experts, small gated networks, whose weighted
answers are added.  It starts as zero, so a stage that learns nothing leaves
the booster's predictions as they are:

    margin = booster.predict_margin(X)
    stage = ExpertStage(ExpertParams(experts=16, k=2), LogLoss()).fit(X, y, margin)
    stage.predict_margin(X_new, booster.predict_margin(X_new))

Per row, with x the standardised inputs (missing ones, NaN or infinite, at their
mean, 0, and columns that the fit saw no spread in always 0):

    r = x A;  a = layer_norm(r);  ids, weights = route(a G, k);
    out = (r + sum_j weights_j expert_{ids_j}(a)) h

The passes are the operations of ``expert_ops`` and torch's plain matrix
products; g comes from the booster's own losses (``boost_ops.grad_hess``);
the parameters are fitted by Adam on mini-batches.  The gate's choice is
balanced by a bias per expert that moves against its share of the rows, by a
constant step, and takes no part in the weights.
"""

from __future__ import annotations

from dataclasses import dataclass

import numpy as np
import torch

from . import boost_ops, expert_ops


@dataclass
class ExpertParams:
    experts: int = 16
    k: int = 2
    width: int = 64               # of a row inside the stage
    inner: int = 64               # of an expert
    scores: str = "sigmoid"
    balance_step: float = 1e-3
    epochs: int = 10
    batch_rows: int = 512
    learning_rate: float = 3e-3
    dtype: str = "float32"        # of the rows and the experts' weights in the passes; parameters are float32
                                  # ("float16" ends at 65504: a fit or an answer that leaves it is an error)
    random_state: int = 0
    device: str = "cuda"


_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


# Standardised inputs are held to +-2^40: the squares of a row of them, which the
# layer norm adds, stay in float32 (a row past that is no row of the fit's table).
_FAR = 2.0 ** 40

# What the rows' gradients are made to add up to before they become float16.  No
# column of a weight's gradient is larger than that times an inner value and an
# input, which leaves those 2^10 below the type's 2^16; and of 65536 rows with
# equal gradients each has 2^-10, which leaves 14 bits above its smallest step 2^-24.
_HALF_SUM = 2.0 ** 6

# An answer in float16 ends at 65504: the answers are counted in a unit in which
# the median gradient before the first step is about this, if it is larger.
_HALF_ANSWER = 2.0 ** 4


def _power_of_two(t: torch.Tensor) -> torch.Tensor:
    """The power of two below each of t's positive normal float32 values."""
    return (t.view(torch.int32) & 0x7F800000).view(torch.float32)


def _half_unit(g: torch.Tensor, head: torch.Tensor) -> torch.Tensor:
    """The power of two, as a 0-d tensor, that the rows' gradients g head are
    multiplied by for float16 (any, where they are all 0)."""
    total = torch.linalg.vector_norm(g, 1) * torch.linalg.vector_norm(head, float("inf"))
    return _power_of_two((_HALF_SUM / total).clamp_(2.0 ** -100, 2.0 ** 100))


def _statistics(raw: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Mean and spread of the finite values of each column of raw (n, F).  A
    column whose values differ by their last bits alone, or that has none, has an
    infinite spread: whatever comes later, its input is 0, as in the fit, which
    learned nothing about it.  Sums are taken in units of the power of two below
    a column's largest value, so that no square leaves float32."""
    if raw.shape[0] == 0:
        return raw.new_zeros(raw.shape[1]), raw.new_full((raw.shape[1],), float("inf"))
    seen = torch.isfinite(raw)
    count = seen.sum(dim=0).clamp_min(1)
    high = torch.where(seen, raw, float("-inf")).amax(dim=0)
    low = torch.where(seen, raw, float("inf")).amin(dim=0)
    most = torch.where(seen, raw.abs(), 0.0).amax(dim=0)
    unit = _power_of_two(most).clamp_min(2.0 ** -126)
    mean = torch.where(seen, raw / unit, 0.0).sum(dim=0) / count
    spread = torch.where(seen, raw / unit - mean, 0.0).square().sum(dim=0) / count
    std = spread.sqrt() * unit
    flat = ~(high - low > 2.0 ** -22 * most) | (std == 0.0)
    return mean * unit, torch.where(flat, float("inf"), std)


class ExpertStage:
    """See the module's text; ``loss`` as a ``Booster`` takes it."""

    unit_: torch.Tensor | None = None     # of the answers, where it may not be 1

    def __init__(self, params: ExpertParams, loss):
        self.p, self.loss = params, loss

    def _check(self) -> None:
        p = self.p
        if p.dtype not in _DTYPES:
            raise ValueError(f"dtype must be one of {sorted(_DTYPES)}, got {p.dtype!r}")
        if p.scores not in expert_ops.SCORES:
            raise ValueError(f"scores must be one of {sorted(expert_ops.SCORES)}, got {p.scores!r}")
        if not 1 <= p.k <= min(p.experts, expert_ops.MAX_K) or p.experts > expert_ops.MAX_EXPERTS:
            raise ValueError(f"{p.k} of {p.experts} experts: at most {expert_ops.MAX_K} of {expert_ops.MAX_EXPERTS}")
        if min(p.width, p.inner, p.batch_rows) < 1 or p.epochs < 0:
            raise ValueError("width, inner and batch_rows must be positive, epochs not negative")

    def _inputs(self, X: np.ndarray) -> torch.Tensor:
        Xt = torch.as_tensor(np.asarray(X, dtype=np.float32), device=self.device_)
        if Xt.dim() != 2 or Xt.shape[1] != self.mean_.shape[0]:
            raise ValueError(f"X must be (n, {self.mean_.shape[0]}), got {tuple(Xt.shape)}")
        known = torch.isfinite(Xt) & torch.isfinite(self.std_)
        return torch.where(known, (Xt - self.mean_) / self.std_, 0.0).clamp_(-_FAR, _FAR)

    def _head(self) -> torch.Tensor:
        return self.weights_["head"] if self.unit_ is None else self.weights_["head"] * self.unit_

    def _forward(self, x: torch.Tensor, keep: bool):
        """(out (n,), what the backward pass needs)."""
        w, p, dt = self.weights_, self.p, _DTYPES[self.p.dtype]
        r = x @ w["embed"]
        a, mean, rstd = expert_ops.layer_norm(r, w["norm"], w["shift"])
        logits = a @ w["gate"].t()
        ids, weights = expert_ops.route(logits, p.k, scores=p.scores, bias=self.bias_)
        plan = expert_ops.expert_plan(ids, p.experts)
        ac, w_in, w_out = a.to(dt), w["w_in"].to(dt), w["w_out"].to(dt)
        if not keep:
            y = expert_ops.expert_products(ac, plan, weights, w_in, w_out)
            return (r + y) @ self._head(), None
        y, inner = expert_ops.expert_products(ac, plan, weights, w_in, w_out, keep_inner=True)
        s = r + y
        return s @ self._head(), (x, r, mean, rstd, a, logits, ids, plan, weights, ac, w_in, w_out, inner, s)

    def _backward(self, g: torch.Tensor, kept) -> dict[str, torch.Tensor]:
        """Gradients of sum_t L_t / n, g = dL/dout, in every parameter."""
        x, r, mean, rstd, a, logits, ids, plan, weights, ac, w_in, w_out, inner, s = kept
        w = self.weights_
        g = g / g.shape[0]
        if self.unit_ is not None:
            g = g * self.unit_
        ds = g[:, None] * w["head"]
        if ac.dtype == torch.float16:
            # float16 has too few powers of two for gradients as they come
            unit = _half_unit(g, w["head"])
            grads = expert_ops.expert_products_grad((ds * unit).half(), ac, plan, weights, w_in, w_out, inner)
            dac, dweights, dw_in, dw_out = (t.float() / unit for t in grads)
        else:
            dac, dweights, dw_in, dw_out = expert_ops.expert_products_grad(ds.to(ac.dtype), ac, plan, weights, w_in,
                                                                           w_out, inner)
        dlogits = expert_ops.route_grad(dweights, logits, ids, scores=self.p.scores)
        da = dac.float() + dlogits @ w["gate"]
        dr, dnorm, dshift = expert_ops.layer_norm_grad(da, r, mean, rstd, w["norm"])
        return dict(embed=x.t() @ (ds + dr), norm=dnorm, shift=dshift, gate=dlogits.t() @ a, w_in=dw_in.float(),
                    w_out=dw_out.float(), head=s.t() @ g)

    def fit(self, X: np.ndarray, y: np.ndarray, margin: np.ndarray | float = 0.0) -> "ExpertStage":
        """Fit to the loss at margin + out; margin (n,), the booster's on these rows, or one number."""
        self._check()
        p = self.p
        # "cuda" is the current device, any other is made current while the stage works
        dev = torch.device(p.device if p.device != "cuda" else f"cuda:{torch.cuda.current_device()}")
        if dev.type != "cuda":
            raise RuntimeError("ExpertStage needs a HIP device: the expert layer has no CPU form")
        self.device_ = dev
        with torch.cuda.device(dev):
            self._fit(np.asarray(X, dtype=np.float32), y, margin)
        return self

    def _fit(self, X: np.ndarray, y: np.ndarray, margin: np.ndarray | float) -> None:
        p, dev = self.p, self.device_
        n, F = X.shape
        self.mean_, self.std_ = _statistics(torch.as_tensor(X, device=dev))
        x = self._inputs(X)
        yt = torch.as_tensor(np.asarray(y, dtype=np.float32), device=dev)
        base = torch.as_tensor(np.broadcast_to(np.asarray(margin, dtype=np.float32), (n,)).copy(), device=dev)
        if yt.shape != (n,):
            raise ValueError(f"y must have shape {(n,)}, got {tuple(yt.shape)}")
        gen = torch.Generator().manual_seed(p.random_state)

        def normal(*shape, scale):
            return (torch.randn(shape, generator=gen) * scale).to(dev)

        self.weights_ = dict(embed=normal(F, p.width, scale=F ** -0.5), norm=torch.ones(p.width, device=dev),
                             shift=torch.zeros(p.width, device=dev),
                             gate=normal(p.experts, p.width, scale=p.width ** -0.5),
                             w_in=normal(p.experts, 2 * p.inner, p.width, scale=p.width ** -0.5),
                             w_out=normal(p.experts, p.width, p.inner, scale=p.inner ** -0.5),
                             head=torch.zeros(p.width, device=dev))
        self.bias_ = torch.zeros(p.experts, device=dev)
        self.unit_ = None
        if p.dtype == "float16" and n:
            g, _ = boost_ops.grad_hess(self.loss, base, yt)
            self.unit_ = _power_of_two((g.abs().median() / _HALF_ANSWER).clamp(1.0, 2.0 ** 100))
        first = {m: torch.zeros_like(t) for m, t in self.weights_.items()}
        second = {m: torch.zeros_like(t) for m, t in self.weights_.items()}
        step = 0
        for _ in range(p.epochs):
            order = torch.randperm(n, generator=gen).to(dev)
            for lo in range(0, n, p.batch_rows):
                rows = order[lo:lo + p.batch_rows]
                out, kept = self._forward(x[rows], keep=True)
                g, _ = boost_ops.grad_hess(self.loss, base[rows] + out, yt[rows])
                step += 1
                scale = p.learning_rate * (1 - 0.999 ** step) ** 0.5 / (1 - 0.9 ** step)
                for m, grad in self._backward(g, kept).items():
                    first[m].lerp_(grad, 0.1)
                    second[m].lerp_(grad.square(), 0.001)
                    self.weights_[m].addcdiv_(first[m], second[m].sqrt() + 1e-8, value=-scale)
                # experts with more than their share become a little less likely
                share = kept[7].offsets.diff().float()
                self.bias_ -= p.balance_step * torch.sign(share - share.mean())
        if not all(bool(torch.isfinite(t).all()) for t in self.weights_.values()):
            raise RuntimeError(f"the fit's parameters are not finite: y or margin are not, or passes in {p.dtype} "
                               "left the type's range")

    def predict_margin(self, X: np.ndarray, margin: np.ndarray | float = 0.0) -> np.ndarray:
        """margin + the stage's answer for each row; margin (n,) or one number."""
        with torch.cuda.device(self.device_):
            x = self._inputs(X)
            base = np.broadcast_to(np.asarray(margin, dtype=np.float32), (x.shape[0],))
            parts = [self._forward(x[lo:lo + (1 << 18)], keep=False)[0] for lo in range(0, x.shape[0], 1 << 18)]
            out = torch.cat(parts) if parts else x.new_zeros(0)
        if not bool(torch.isfinite(out).all()):
            raise RuntimeError(f"answers are not finite: passes in {self.p.dtype} left the type's range")
        return base + out.cpu().numpy()

    def loads(self, X: np.ndarray) -> np.ndarray:
        """How many of X's slots each expert gets."""
        with torch.cuda.device(self.device_):
            x, w = self._inputs(X), self.weights_
            a = expert_ops.layer_norm(x @ w["embed"], w["norm"], w["shift"])[0]
            ids, _ = expert_ops.route(a @ w["gate"].t(), self.p.k, scores=self.p.scores, bias=self.bias_)
            return expert_ops.expert_plan(ids, self.p.experts).offsets.diff().cpu().numpy()
