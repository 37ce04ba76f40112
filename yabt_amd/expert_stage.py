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
    random_state: int = 0
    device: str = "cuda"


_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


# Standardised inputs are held to +-2^40: the squares of a row of them, which the
# layer norm adds, stay in float32 (a row past that is no row of the fit's table).
_FAR = 2.0 ** 40


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
    unit = (most.view(torch.int32) & 0x7F800000).view(torch.float32).clamp_min(2.0 ** -126)
    mean = torch.where(seen, raw / unit, 0.0).sum(dim=0) / count
    spread = torch.where(seen, raw / unit - mean, 0.0).square().sum(dim=0) / count
    std = spread.sqrt() * unit
    flat = ~(high - low > 2.0 ** -22 * most) | (std == 0.0)
    return mean * unit, torch.where(flat, float("inf"), std)


class ExpertStage:
    """See the module's text; ``loss`` as a ``Booster`` takes it."""

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
            return (r + y) @ w["head"], None
        y, inner = expert_ops.expert_products(ac, plan, weights, w_in, w_out, keep_inner=True)
        s = r + y
        return s @ w["head"], (x, r, mean, rstd, a, logits, ids, plan, weights, ac, w_in, w_out, inner, s)

    def _backward(self, g: torch.Tensor, kept) -> dict[str, torch.Tensor]:
        """Gradients of sum_t L_t / n, g = dL/dout, in every parameter."""
        x, r, mean, rstd, a, logits, ids, plan, weights, ac, w_in, w_out, inner, s = kept
        w = self.weights_
        g = g / g.shape[0]
        ds = g[:, None] * w["head"]
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
        dev = torch.device(p.device if p.device != "cuda" else f"cuda:{torch.cuda.current_device()}")
        if dev.type != "cuda":
            raise RuntimeError("ExpertStage needs a HIP device: the expert layer has no CPU form")
        X = np.asarray(X, dtype=np.float32)
        n, F = X.shape
        self.device_ = dev
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
        return self

    def predict_margin(self, X: np.ndarray, margin: np.ndarray | float = 0.0) -> np.ndarray:
        """margin + the stage's answer for each row; margin (n,) or one number."""
        x = self._inputs(X)
        base = np.broadcast_to(np.asarray(margin, dtype=np.float32), (x.shape[0],))
        parts = [self._forward(x[lo:lo + (1 << 18)], keep=False)[0] for lo in range(0, x.shape[0], 1 << 18)]
        out = torch.cat(parts) if parts else x.new_zeros(0)
        return base + out.cpu().numpy()

    def loads(self, X: np.ndarray) -> np.ndarray:
        """How many of X's slots each expert gets."""
        x, w = self._inputs(X), self.weights_
        a = expert_ops.layer_norm(x @ w["embed"], w["norm"], w["shift"])[0]
        ids, _ = expert_ops.route(a @ w["gate"].t(), self.p.k, scores=self.p.scores, bias=self.bias_)
        return expert_ops.expert_plan(ids, self.p.experts).offsets.diff().cpu().numpy()
