"""What is timed of the expert layer: row normalisation, routing and the experts' products.

Rows of a table (or of a batch of requests) pass through a layer norm, a gate
scores E experts for each, the best k of them answer, and the weighted answers
are added up.  Six kinds of work:

* ``norm``: the layer norm of n rows, as scoring runs it;
* ``norm_grad``: forward and backward, with the gradients of weight and bias;
* ``route``: logits to expert ids and weights, and the plan that sorts the
  slots by expert;
* ``route_grad``: the same, and the logits' gradient;
* ``experts``: the plan and the experts' products, as scoring runs them;
* ``experts_grad``: forward and backward, with every gradient.

``own`` chooses between the framework's kernels and the plain form: elementary
torch operations in 32 bits.  ``exact`` restates each in 64 bits.
"""

from __future__ import annotations

import math
import random

import torch

own = False

EPS = 1e-5
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # one request: the launch is what costs
        dict(name="norm_1x512_bf16", kind="norm", rows=1, width=512, type="bf16"),
        # training on a sample of the widest benchmark table (500 columns), in its own type
        dict(name="norm_grad_20000x500_f32", kind="norm_grad", rows=20_000, width=500, type="f32"),
        # a large training batch of a wide layer
        dict(name="norm_grad_16384x4096_bf16", kind="norm_grad", rows=16_384, width=4096, type="bf16"),
        # one request through the gate
        dict(name="route_1x64_top6", kind="route", rows=1, experts=64, k=6, type="f32", scores="softmax", bias=False,
             groups=1, keep=1, renormalise=True, scale=1.0, masked=0.0),
        # a large batch: sigmoid scores with a balancing bias, 4 of 8 groups, 8 of 256 experts
        dict(name="route_65536x256_top8", kind="route", rows=65_536, experts=256, k=8, type="bf16", scores="sigmoid",
             bias=True, groups=8, keep=4, renormalise=True, scale=2.5, masked=0.0),
        # training, an odd number of rows and experts, some experts closed to some rows
        dict(name="route_grad_8191x60_top4", kind="route_grad", rows=8_191, experts=60, k=4, type="f32",
             scores="softmax", bias=False, groups=1, keep=1, renormalise=False, scale=1.0, masked=0.1),
        # one request: six experts' weights are read for a single row
        dict(name="experts_1x1024_64e_top6", kind="experts", rows=1, width=1024, inner=512, experts=64, k=6,
             type="bf16", unused=0.0),
        # a batch of requests: every expert is read for a few rows
        dict(name="experts_48x2048_32e_top4", kind="experts", rows=48, width=2048, inner=1024, experts=32, k=4,
             type="f16", unused=0.0),
        # scoring a large batch
        dict(name="experts_16384x2048_16e_top2", kind="experts", rows=16_384, width=2048, inner=2048, experts=16, k=2,
             type="bf16", unused=0.0),
        # training on the benchmark table's 100 columns as they are: fp32, nothing a multiple of a tile
        dict(name="experts_grad_20000x100_7e_top1", kind="experts_grad", rows=20_000, width=100, inner=60, experts=7,
             k=1, type="f32", unused=0.02),
        # training, many small experts
        dict(name="experts_grad_8192x1024_64e_top6", kind="experts_grad", rows=8_192, width=1024, inner=704,
             experts=64, k=6, type="bf16", unused=0.02),
        # training, few large experts: the largest
        dict(name="experts_grad_16384x2048_8e_top2", kind="experts_grad", rows=16_384, width=2048, inner=2048,
             experts=8, k=2, type="bf16", unused=0.0),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], evenly spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A width: odd, a multiple of 40 or a power of two."""
    w, sort = _log(rng, lo, hi), rng.choice(["odd", "forties", "power"])
    if sort == "odd":
        return min(w | 1, hi - 1)
    return max(40, w // 40 * 40) if sort == "forties" else 1 << max(5, w.bit_length() - 1)


def draw(rng: random.Random):
    kind = rng.choice(["norm", "norm_grad", "route", "route_grad", "experts", "experts", "experts_grad"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if kind in ("norm", "norm_grad"):
        width = _width(rng, 16, 8192)
        return dict(kind=kind, rows=min(_log(rng, 1, 100_000), 67_000_000 // width), width=width, type=dtype)
    if kind in ("route", "route_grad"):
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * _log(rng, max(2, 8 // groups), 256 // groups)
        keep = rng.randint(1, groups)
        scores = rng.choice(["softmax", "sigmoid"])
        return dict(kind=kind, rows=_log(rng, 1, 65_536), experts=experts,
                    k=rng.randint(1, min(8, keep * (experts // groups))), type=dtype, scores=scores,
                    bias=scores == "sigmoid" and rng.random() < 0.7, groups=groups, keep=keep,
                    renormalise=rng.random() < 0.6, scale=rng.choice([1.0, 2.5]),
                    masked=rng.choice([0.0, 0.0, 0.1, 0.6]))
    experts, k = _log(rng, 2, 64), 1
    k = rng.randint(1, min(8, experts))
    width, inner = _width(rng, 24, 2048), _width(rng, 16, 2048)
    most = 60_000_000_000 if dtype == "f32" else 130_000_000_000     # rows * k * width * inner
    return dict(kind=kind, rows=max(1, min(_log(rng, 1, 16_384), most // (k * width * inner))), width=width,
                inner=inner, experts=experts, k=k, type=dtype, unused=rng.choice([0.0, 0.0, 0.02, 0.3]))


# ---------------------------------------------------------------------------
# inputs, from the seed alone
# ---------------------------------------------------------------------------

def _dev():
    return torch.device("cuda", torch.cuda.current_device())


def _gen(seed):
    return torch.Generator(device=_dev()).manual_seed(seed)


def _normal(gen, *shape):
    return torch.randn(shape, device=_dev(), generator=gen)


def prepare(case, seed):
    gen, kind, dt, n = _gen(seed), case["kind"], TYPES[case["type"]], case["rows"]
    if kind in ("norm", "norm_grad"):
        D = case["width"]
        x = _normal(gen, n, D) * (0.5 + torch.rand((n, 1), device=_dev(), generator=gen)) + 0.3 * _normal(gen, n, 1)
        return dict(case=case, x=x.to(dt), weight=1.0 + 0.1 * _normal(gen, D), bias=0.1 * _normal(gen, D),
                    dy=_normal(gen, n, D).to(dt))
    if kind in ("route", "route_grad"):
        E = case["experts"]
        logits = (_normal(gen, n, E) + 0.5 * _normal(gen, E)).to(dt)      # some experts are asked for more often
        if case["masked"]:
            logits[torch.rand((n, E), device=_dev(), generator=gen) < case["masked"]] = float("-inf")
        return dict(case=case, logits=logits, bias=0.05 * _normal(gen, E) if case["bias"] else None,
                    dweights=_normal(gen, n, case["k"]))
    D, F, E, k = case["width"], case["inner"], case["experts"], case["k"]
    gate = _normal(gen, n, E) + 0.5 * _normal(gen, E)
    score, ids = gate.topk(k, dim=1)
    weights = torch.softmax(score, dim=1)
    off = torch.rand((n, k), device=_dev(), generator=gen) < case["unused"]  # a slot that no expert was left for
    ids = torch.where(off, -1, ids).to(torch.int32)
    weights = torch.where(off, 0.0, weights)
    counts = torch.bincount(ids.flatten()[ids.flatten() >= 0].long(), minlength=E)
    return dict(case=case, x=_normal(gen, n, D).to(dt), ids=ids, weights=weights, most=max(1, int(counts.max())),
                w_in=(_normal(gen, E, 2 * F, D) / math.sqrt(D)).to(dt),
                w_out=(_normal(gen, E, D, F) / math.sqrt(F)).to(dt), dy=_normal(gen, n, D).to(dt))


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    kind = state["case"]["kind"]
    if kind in ("norm", "norm_grad"):
        return (_norm if own else _norm_plain)(state, kind == "norm_grad")
    if kind in ("route", "route_grad"):
        return (_route if own else _route_plain)(state, kind == "route_grad")
    return (_experts if own else _experts_plain)(state, kind == "experts_grad")


def _norm(s, grad):
    from yabt_amd import expert_ops

    y, mean, rstd = expert_ops.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS)
    out = dict(y=y, mean=mean, rstd=rstd)
    if grad:
        out["dx"], out["dweight"], out["dbias"] = expert_ops.layer_norm_grad(s["dy"], s["x"], mean, rstd, s["weight"])
    return out


def _route(s, grad):
    from yabt_amd import expert_ops

    c = s["case"]
    how = dict(scores=c["scores"], renormalise=c["renormalise"], scale=c["scale"])
    ids, weights = expert_ops.route(s["logits"], c["k"], bias=s["bias"], groups=c["groups"], keep_groups=c["keep"],
                                    **how)
    plan = expert_ops.expert_plan(ids, c["experts"])
    out = dict(ids=ids, weights=weights, offsets=plan.offsets, slots=plan.slots)
    if grad:
        out["dlogits"] = expert_ops.route_grad(s["dweights"], s["logits"], ids, **how)
    return out


def _experts(s, grad):
    from yabt_amd import expert_ops

    plan = expert_ops.expert_plan(s["ids"], s["case"]["experts"])
    if not grad:
        return dict(y=expert_ops.expert_products(s["x"], plan, s["weights"], s["w_in"], s["w_out"]))
    y, inner = expert_ops.expert_products(s["x"], plan, s["weights"], s["w_in"], s["w_out"], keep_inner=True)
    dx, dweights, dw_in, dw_out = expert_ops.expert_products_grad(s["dy"], s["x"], plan, s["weights"], s["w_in"],
                                                                  s["w_out"], inner)
    return dict(y=y, dx=dx, dweights=dweights, dw_in=dw_in, dw_out=dw_out)


def _norm_plain(s, grad):
    x, w = s["x"].float(), s["weight"]
    mean = x.mean(dim=1, keepdim=True)
    rstd = ((x - mean).square().mean(dim=1, keepdim=True) + EPS).rsqrt()
    xh = (x - mean) * rstd
    out = dict(y=(xh * w + s["bias"]).to(s["x"].dtype), mean=mean[:, 0], rstd=rstd[:, 0])
    if grad:
        dy = s["dy"].float()
        t = dy * w
        dx = rstd * (t - t.mean(dim=1, keepdim=True) - xh * (t * xh).mean(dim=1, keepdim=True))
        out.update(dx=dx.to(s["x"].dtype), dweight=(dy * xh).sum(dim=0), dbias=dy.sum(dim=0))
    return out


def _route_plain(s, grad):
    c, k, E = s["case"], s["case"]["k"], s["case"]["experts"]
    low = float("-inf")
    x = s["logits"].float()
    n = x.shape[0]
    live = x > low
    x = torch.where(live, x, low)
    if c["scores"] == "softmax":
        top = x.amax(dim=1, keepdim=True).clamp_min(-3.0e38)
        p = (x - top).exp()
        p = p / p.sum(dim=1, keepdim=True).clamp_min(1e-30)
        key = x
    else:
        p = (1.0 + (-x).exp()).reciprocal()
        key = p
    if s["bias"] is not None:
        key = key + s["bias"]
    key = torch.where(live, key, low)
    if c["groups"] > 1:
        parts = key.view(n, c["groups"], E // c["groups"])
        best = parts.sort(dim=2, descending=True).values
        if c["scores"] == "softmax":
            score = best[:, :, 0]
        else:
            two = best[:, :, 1] if E // c["groups"] > 1 else torch.full_like(best[:, :, 0], low)
            score = best[:, :, 0] + torch.where(two > low, two, 0.0)
        order = score.sort(dim=1, descending=True, stable=True).indices
        kept = torch.zeros((n, c["groups"]), dtype=torch.bool, device=x.device)
        kept.scatter_(1, order[:, :c["keep"]], True)
        key = torch.where(kept[:, :, None], parts, low).view(n, E)
    best, ids = key.sort(dim=1, descending=True, stable=True)
    ids, taken = ids[:, :k], best[:, :k] > low
    ps = torch.where(taken, p.gather(1, ids), 0.0)
    total = ps.sum(dim=1, keepdim=True).clamp_min(1e-30)
    v = ps / total if c["renormalise"] else ps
    out_ids = torch.where(taken, ids, -1).to(torch.int32)
    # the plan: slots by expert, those without one last and not listed
    flat = out_ids.flatten().long()
    by, slots = torch.where(flat >= 0, flat, E).sort(stable=True)
    offsets = torch.searchsorted(by, torch.arange(E + 1, device=x.device)).to(torch.int32)
    slots = torch.where(by < E, slots, -1).to(torch.int32)
    out = dict(ids=out_ids, weights=c["scale"] * v, offsets=offsets, slots=slots)
    if grad:
        dw = torch.where(taken, s["dweights"], 0.0) * c["scale"]
        mean = (v * dw).sum(dim=1, keepdim=True)
        if c["scores"] == "softmax" and c["renormalise"]:
            d = v * (dw - mean)
        elif c["scores"] == "softmax":
            d = v * dw
        elif c["renormalise"]:
            d = torch.where(taken, (dw - mean) / total, 0.0) * ps * (1.0 - ps)
        else:
            d = dw * ps * (1.0 - ps)
        dl = torch.zeros_like(p).scatter_(1, ids, d)
        if c["scores"] == "softmax" and not c["renormalise"]:
            dl = dl - p * mean
        out["dlogits"] = dl.to(s["logits"].dtype)
    return out


def _experts_plain(s, grad):
    x, ids, w, w_in, w_out = s["x"], s["ids"], s["weights"], s["w_in"], s["w_out"]
    (n, D), k, E, F = x.shape, ids.shape[1], w_in.shape[0], w_out.shape[2]
    flat = ids.flatten().long()
    live = flat >= 0
    rows = torch.arange(n * k, device=x.device) // k
    if grad or n * k > E:
        # the experts side by side, each with as many places as the busiest has rows
        G, C = E, s["most"]
        by, order = torch.where(live, flat, E).sort(stable=True)
        first = torch.searchsorted(by, torch.arange(E + 1, device=x.device))
        rank = torch.empty_like(order).scatter_(0, order, torch.arange(n * k, device=x.device) - first[by])
        place = torch.where(live, flat * C + rank, G * C)
        a, b = w_in.float(), w_out.float()
    else:
        # fewer slots than experts: their own experts' weights
        G, C = n * k, 1
        place = torch.where(live, torch.arange(n * k, device=x.device), G)
        a, b = w_in[flat.clamp_min(0)].float(), w_out[flat.clamp_min(0)].float()

    def spread(values):
        return torch.zeros((G * C + 1, D), device=x.device).index_copy_(0, place, values)[:-1].view(G, C, D)

    def collect(values):
        return torch.cat([values.reshape(G * C, -1), values.new_zeros((1, values.shape[2]))])[place]

    xs = spread(x.float()[rows])
    pre = torch.bmm(xs, a.transpose(1, 2))
    g, u = pre[:, :, :F], pre[:, :, F:]
    sig = (1.0 + (-g).exp()).reciprocal()
    h = g * sig * u
    z = collect(torch.bmm(h, b.transpose(1, 2)))
    y = (z * w.flatten()[:, None]).view(n, k, D).sum(dim=1).to(x.dtype)
    if not grad:
        return dict(y=y)
    dys = s["dy"].float()[rows]
    dweights = (dys * z).sum(dim=1).view(n, k)
    dz = spread(dys * w.flatten()[:, None])
    dh = torch.bmm(dz, b)
    dpre = torch.cat([dh * u * sig * (1.0 + g * (1.0 - sig)), dh * g * sig], dim=2)
    dx = collect(torch.bmm(dpre, a)).view(n, k, D).sum(dim=1)
    return dict(y=y, dx=dx.to(x.dtype), dweights=dweights, dw_in=torch.bmm(dpre.transpose(1, 2), xs).to(x.dtype),
                dw_out=torch.bmm(dz.transpose(1, 2), h).to(x.dtype))


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind in ("norm", "norm_grad"):
        return _norm_exact(s, kind == "norm_grad")
    if kind in ("route", "route_grad"):
        return _route_exact(s, kind == "route_grad")
    return _experts_exact(s, kind == "experts_grad")


def _norm_exact(s, grad):
    x, w, b, dy = (s[name].double() for name in ("x", "weight", "bias", "dy"))
    var, mean = torch.var_mean(x, dim=1, correction=0)
    rstd = 1.0 / torch.sqrt(var + EPS)
    y = torch.addcmul(b, (x - mean[:, None]) * rstd[:, None], w)
    out = dict(y=y, mean=mean, rstd=rstd)
    if grad:
        # y = w z + b with z = A x / sqrt(...): dx by the chain through the centred row and its length
        t, xc, D = dy * w, x - mean[:, None], x.shape[1]
        along = (t * xc).sum(dim=1) * rstd ** 3 / D
        dxc = t * rstd[:, None] - xc * along[:, None]
        out["dx"] = dxc - dxc.sum(dim=1, keepdim=True) / D
        out["dweight"] = torch.einsum("nd,nd,n->d", dy, xc, rstd)
        out["dbias"] = dy.sum(dim=0)
    return out


def _route_exact(s, grad):
    """ids as the definition has them: keys are compared in 32 bits."""
    c, x = s["case"], s["logits"].double()
    n, E = x.shape
    k, G = c["k"], c["groups"]
    low = float("-inf")
    none = ~(x > low)
    x = x.masked_fill(none, low)
    if c["scores"] == "softmax":
        p = torch.softmax(x, dim=1).nan_to_num(0.0)
        key = x.float()
    else:
        p = torch.special.expit(x)
        key = p.float()
    key = key if s["bias"] is None else key + s["bias"]
    key = key.masked_fill(none, low)
    index = torch.arange(E, device=x.device)
    if G > 1:
        grouped, score = key.view(n, G, E // G), torch.zeros((n, G), device=x.device)
        rest = grouped.clone()
        for step in range(1 if c["scores"] == "softmax" else 2):
            if step < E // G:
                top, at = rest.max(dim=2)
                score = top if step == 0 else torch.where(top > low, score + top, score)
                rest.scatter_(2, at[:, :, None], low)
        kept = torch.zeros((n, G), dtype=torch.bool, device=x.device)
        for _ in range(c["keep"]):
            left = score.masked_fill(kept, low)
            best = left.amax(dim=1, keepdim=True)
            first = torch.where((left == best) & ~kept, torch.arange(G, device=x.device), G).amin(dim=1)
            kept |= torch.arange(G, device=x.device) == first[:, None]
        key = grouped.masked_fill(~kept[:, :, None], low).reshape(n, E)
    ids = torch.full((n, k), -1, dtype=torch.int64, device=x.device)
    for j in range(k):
        best = key.amax(dim=1)
        at = torch.where(key == best[:, None], index, E).amin(dim=1)
        ids[:, j] = torch.where(best > low, at, -1)
        key = key.scatter(1, at[:, None], low)
    taken = ids >= 0
    ps = torch.gather(p, 1, ids.clamp_min(0)) * taken
    weights = c["scale"] * (ps / ps.sum(dim=1, keepdim=True).clamp_min(1e-300) if c["renormalise"] else ps)
    flat = ids.flatten()
    offsets = torch.cat([flat.new_zeros(1), torch.bincount(flat[flat >= 0], minlength=E).cumsum(0)])
    listed_slots = torch.argsort(torch.where(flat >= 0, flat, E), stable=True)
    listed_slots[int(offsets[-1]):] = -1
    out = dict(ids=ids.to(torch.int32), weights=weights, offsets=offsets.to(torch.int32),
               slots=listed_slots.to(torch.int32))
    if grad:
        # by torch's own differentiation of the weights, the choice held fixed
        leaf = x.masked_fill(none, -1e30).requires_grad_(True)
        q = torch.softmax(leaf, dim=1) if c["scores"] == "softmax" else torch.special.expit(leaf)
        qs = q.gather(1, ids.clamp_min(0)) * taken
        wq = c["scale"] * (qs / qs.sum(dim=1, keepdim=True).clamp_min(1e-300) if c["renormalise"] else qs)
        (wq * s["dweights"].double()).sum().backward()
        out["dlogits"] = leaf.grad
    return out


def _experts_exact(s, grad):
    x, w = s["x"].double(), s["weights"].double()
    (n, D), (k, E) = x.shape, (s["case"]["k"], s["case"]["experts"])
    F = s["case"]["inner"]
    dy = s["dy"].double()
    y, dx = torch.zeros_like(x), torch.zeros_like(x)
    dweights = torch.zeros_like(w)
    dw_in = torch.zeros(s["w_in"].shape, dtype=torch.float64, device=x.device) if grad else None
    dw_out = torch.zeros(s["w_out"].shape, dtype=torch.float64, device=x.device) if grad else None
    for e in range(E):
        t, j = torch.nonzero(s["ids"] == e, as_tuple=True)
        if not t.numel():
            continue
        a, b, xe, we = s["w_in"][e].double(), s["w_out"][e].double(), x[t], w[t, j][:, None]
        g, u = xe @ a[:F].T, xe @ a[F:].T
        sig = torch.special.expit(g)
        h = g * sig * u
        z = h @ b.T
        y.index_add_(0, t, we * z)
        if grad:
            de = dy[t]
            dweights[t, j] = (de * z).sum(dim=1)
            dh = we * (de @ b)
            dg, du = dh * u * (sig + g * sig * (1.0 - sig)), dh * g * sig
            dx.index_add_(0, t, dg @ a[:F] + du @ a[F:])
            dw_in[e, :F], dw_in[e, F:] = dg.T @ xe, du.T @ xe
            dw_out[e] = de.T @ (we * h)
    return dict(y=y, dx=dx, dweights=dweights, dw_in=dw_in, dw_out=dw_out) if grad else dict(y=y)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    kind, n, b = case["kind"], case["rows"], BYTES[case["type"]]
    if kind in ("norm", "norm_grad"):
        D, grad = case["width"], kind == "norm_grad"
        # x and dy in, y and dx out, the statistics, the parameters and their gradients
        return dict(bytes=n * D * b * (4 if grad else 2) + 8 * n + 4 * D * (4 if grad else 2),
                    flops=n * D * (22 if grad else 8))
    if kind in ("route", "route_grad"):
        E, k, grad = case["experts"], case["k"], kind == "route_grad"
        return dict(bytes=n * E * b * (2 if grad else 1) + n * k * (16 if grad else 12) + 4 * E * (2 if case["bias"] else 1),
                    flops=n * E * (10 if grad else 5))
    D, F, E, k, grad = case["width"], case["inner"], case["experts"], case["k"], kind == "experts_grad"
    slots = n * k * (1.0 - case["unused"])
    touched = E * (1.0 - (1.0 - min(1.0, k * (1.0 - case["unused"]) / E)) ** n)
    return dict(bytes=n * D * b * (4 if grad else 2) + touched * 3 * D * F * b + (E * 3 * D * F * b if grad else 0)
                + n * k * (12 if grad else 8),
                flops=slots * D * F * (18 if grad else 6))
