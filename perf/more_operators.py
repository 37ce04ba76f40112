"""What is timed of the dense stage: gated feed-forward blocks, their fit and their answers in 8 bits.

Beside its routed experts a layer has a block that every row passes.  It is
fitted by AdamW, whose states take 8 bits where memory is short, and answers
by 8-bit integer products where requests are many.  Five kinds of work:

* ``feed``: y = (act(x Wg^T) * (x Wu^T)) Wo^T of n rows, as scoring runs it;
* ``feed_grad``: forward and backward, with every gradient;
* ``adamw``: one step over all tensors of a model, states in 32 or 8 bits;
* ``product8``: rows put in 8 bits with a scale each, times a weight in 8 bits
  with a scale for each of its rows;
* ``feed8``: the block with both weights in 8 bits.

``own`` chooses between the framework's kernels and the plain form: elementary
torch operations in 32 bits.  ``exact`` restates each in 64 bits.

What is put in 8 bits is defined by operations in 32 bits, each rounded, in the
order of ``_codes`` and ``_step_plain``: two programs that keep to it hold the
same codes.
"""

from __future__ import annotations

import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
BETAS, EPS, BLOCK = (0.9, 0.999), 1e-8, 256
LEAST = 2.0 ** -100                    # rows and blocks whose largest magnitude is below count as zeros


def listed():
    return [
        # one request: the weights' bytes and two launches
        dict(name="feed_1x1024_f4096_bf16", kind="feed", rows=1, width=1024, inner=4096, type="bf16", act="silu"),
        # a batch of requests
        dict(name="feed_48x2048_f5632_f16", kind="feed", rows=48, width=2048, inner=5632, type="f16", act="gelu"),
        # scoring the benchmark table's 100 columns in their own type, an odd inner width
        dict(name="feed_20000x100_f61_f32", kind="feed", rows=20_000, width=100, inner=61, type="f32", act="silu"),
        # training on a batch of the widest benchmark table (500 columns): fp32, nothing a multiple of a tile
        dict(name="feed_grad_777x500_f1333_f32", kind="feed_grad", rows=777, width=500, inner=1333, type="f32",
             act="gelu_tanh"),
        # training, a large batch of a wide layer
        dict(name="feed_grad_8192x2048_f5632_bf16", kind="feed_grad", rows=8_192, width=2048, inner=5632, type="bf16",
             act="silu"),
        # the parameters of a stage of 16 experts on 100 columns: the launch is what costs
        dict(name="adamw_7_of_204k_f32", kind="adamw", tensors=7, values=204_000, type="f32", grads="f32", bits=32,
             step=17, decay=0.0),
        # a model with 32-bit states, gradients in the type of the passes
        dict(name="adamw_12_of_40m_f32", kind="adamw", tensors=12, values=40_000_001, type="f32", grads="bf16",
             bits=32, step=1000, decay=0.01),
        # a larger one with 8-bit states
        dict(name="adamw_16_of_120m_8bit", kind="adamw", tensors=16, values=120_000_007, type="f32", grads="bf16",
             bits=8, step=1000, decay=0.01),
        # one request through one weight
        dict(name="product8_1x4096x4096", kind="product8", rows=1, width=4096, cols=4096, type="bf16"),
        # a large batch
        dict(name="product8_8192x4096x4096", kind="product8", rows=8_192, width=4096, cols=4096, type="bf16"),
        # a batch of requests through the block
        dict(name="feed8_24x2048_f5632", kind="feed8", rows=24, width=2048, inner=5632, type="bf16", act="silu"),
        # scoring a large batch: the largest
        dict(name="feed8_16384x2048_f5632", kind="feed8", rows=16_384, width=2048, inner=5632, type="bf16",
             act="silu"),
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
    kind = rng.choice(["feed", "feed_grad", "adamw", "product8", "feed8"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    act = rng.choice(["silu", "silu", "gelu", "gelu_tanh", "relu"])
    if kind == "adamw":
        return dict(kind=kind, tensors=rng.randint(1, 16), values=_log(rng, 1000, 120_000_000), type=dtype,
                    grads=rng.choice([dtype, "f32", "bf16"]), bits=rng.choice([32, 8]), step=_log(rng, 1, 100_000),
                    decay=rng.choice([0.0, 0.01, 0.1]))
    width = _width(rng, 24, 4096)
    if kind == "product8":
        cols = _width(rng, 24, 8192)
        return dict(kind=kind, rows=max(1, min(_log(rng, 1, 16_384), 130_000_000_000 // (width * cols))), width=width,
                    cols=cols, type=dtype)
    inner = _width(rng, 24, 8192)
    most = 11_000_000_000 if dtype == "f32" else 90_000_000_000           # rows * width * inner
    return dict(kind=kind, rows=max(1, min(_log(rng, 1, 16_384), most // (width * inner))), width=width, inner=inner,
                type=dtype if kind != "feed8" or dtype != "f32" else "bf16", act=act)


# ---------------------------------------------------------------------------
# inputs, from the seed alone
# ---------------------------------------------------------------------------

def _dev():
    return torch.device("cuda", torch.cuda.current_device())


def _normal(gen, *shape):
    return torch.randn(shape, device=_dev(), generator=gen)


def _uniform(gen, *shape):
    return torch.rand(shape, device=_dev(), generator=gen)


def _sizes(case):
    """The tensors' sizes: of very different ones, the last takes what is left."""
    if case["tensors"] == 7 and case["values"] == 204_000:
        return [6400, 64, 64, 1024, 131_072, 65_536, 64]     # the stage's own
    rng, left = random.Random(case["tensors"] * 7919 + case["values"]), case["values"]
    sizes = [max(1, int(left / case["tensors"] * math.exp(rng.uniform(-5.0, 0.5)))) for _ in range(case["tensors"] - 1)]
    return sizes + [max(1, left - sum(sizes))]


def prepare(case, seed):
    gen, kind, dt = torch.Generator(device=_dev()).manual_seed(seed), case["kind"], TYPES[case["type"]]
    if kind == "adamw":
        sizes, gt = _sizes(case), TYPES[case["grads"]]
        params = [(0.02 * _normal(gen, n)).to(dt) for n in sizes]
        # gradients of a fit on its way: rows of very different spread, their averages a little apart from them
        grads = [(1e-3 * _normal(gen, n) * (-3.0 * _uniform(gen, n)).exp()).to(gt) for n in sizes]
        first = [0.3 * g.float() + 1e-4 * _normal(gen, g.numel()) for g in grads]
        second = [0.5 * g.float().square() + 1e-7 * _uniform(gen, g.numel()) for g in grads]
        s = dict(case=case, params=params, grads=grads)
        if case["bits"] == 32:
            s.update(first=first, second=second, first_scale=None, second_scale=None)
        else:
            # a state as earlier steps left it
            a, b = [_put_first(m) for m in first], [_put_second(v) for v in second]
            s.update(first=[c for c, _ in a], second=[c for c, _ in b], first_scale=[t for _, t in a],
                     second_scale=[t for _, t in b])
        return s
    n, D = case["rows"], case["width"]
    if kind == "product8":
        # activations: some channels are larger than the others
        x = (_normal(gen, n, D) * (0.7 * _normal(gen, D)).exp()).to(dt)
        weight = _codes(_normal(gen, case["cols"], D) / math.sqrt(D))
        return dict(case=case, x=x, weight=weight[0], scale=weight[1])
    F = case["inner"]
    x = _normal(gen, n, D).to(dt)
    w_in, w_out = _normal(gen, 2 * F, D) / math.sqrt(D), _normal(gen, D, F) / math.sqrt(F)
    if kind == "feed8":
        (a, sa), (b, sb) = _codes(w_in), _codes(w_out)
        return dict(case=case, x=x, w_in=a, in_scale=sa, w_out=b, out_scale=sb)
    return dict(case=case, x=x, w_in=w_in.to(dt), w_out=w_out.to(dt), dy=_normal(gen, n, D).to(dt))


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    kind = state["case"]["kind"]
    if kind == "adamw":
        return (_step if own else _step_plain)(state)
    if kind == "product8":
        return (_product8 if own else _product8_plain)(state)
    if kind == "feed8":
        return (_feed8 if own else _feed8_plain)(state)
    return (_feed if own else _feed_plain)(state, kind == "feed_grad")


def _feed(s, grad):
    from yabt_amd import feed_ops

    act = s["case"]["act"]
    if not grad:
        return dict(y=feed_ops.feed_forward(s["x"], s["w_in"], s["w_out"], activation=act))
    y, inner = feed_ops.feed_forward(s["x"], s["w_in"], s["w_out"], activation=act, keep_inner=True)
    dx, dw_in, dw_out = feed_ops.feed_forward_grad(s["dy"], s["x"], s["w_in"], s["w_out"], inner, activation=act)
    return dict(y=y, dx=dx, dw_in=dw_in, dw_out=dw_out)


def _product8(s):
    from yabt_amd import feed_ops

    q, scale = feed_ops.quantize_rows(s["x"])
    return feed_ops.product_int8(q, scale, s["weight"], s["scale"], dtype=s["x"].dtype)


def _feed8(s):
    from yabt_amd import feed_ops

    return feed_ops.feed_forward_int8(s["x"], s["w_in"], s["in_scale"], s["w_out"], s["out_scale"],
                                      activation=s["case"]["act"])


def _step(s):
    """The step writes into the program's own parameters and states."""
    from yabt_amd import optim

    c = s["case"]
    state = optim.AdamWState(s["first"], s["second"], s["first_scale"], s["second_scale"])
    optim.adamw_step(s["params"], s["grads"], state, c["step"], lr=1e-3, betas=BETAS, eps=EPS,
                     weight_decay=c["decay"])
    first, second = state.values()
    return dict(params=s["params"], first=first, second=second)


def _act_plain(name, g):
    """act(g) and its derivative."""
    if name == "silu":
        p = (1.0 + (-g).exp()).reciprocal()
        return g * p, p * (1.0 + g * (1.0 - p))
    if name == "relu":
        return torch.where(g > 0.0, g, 0.0), torch.where(g > 0.0, 1.0, 0.0)
    if name == "gelu":
        p = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * p, p + g * (-0.5 * g * g).exp() * (1.0 / math.sqrt(2.0 * math.pi))
    a, b = math.sqrt(2.0 / math.pi), 0.044715
    t = torch.tanh(a * (g + b * g * g * g))
    return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * a * (1.0 + 3.0 * b * g * g)


def _feed_plain(s, grad):
    x, a, b, F, dt = s["x"].float(), s["w_in"].float(), s["w_out"].float(), s["case"]["inner"], s["x"].dtype
    pre = x @ a.t()
    g, u = pre[:, :F], pre[:, F:]
    act, slope = _act_plain(s["case"]["act"], g)
    h = act * u
    y = (h @ b.t()).to(dt)
    if not grad:
        return dict(y=y)
    dy = s["dy"].float()
    dh = dy @ b
    dpre = torch.cat([dh * u * slope, dh * act], dim=1)
    return dict(y=y, dx=(dpre @ a).to(dt), dw_in=(dpre.t() @ x).to(dt), dw_out=(dy.t() @ h).to(dt))


def _codes(x):
    """(codes, scale) of x's rows: codes from -127 to 127 that count a 127th of the row's largest magnitude."""
    x = x.float()
    most = x.abs().amax(dim=1)
    some = most >= LEAST
    unit = torch.where(some, torch.full_like(most, 127.0) / most, 0.0)
    codes = torch.round(x * unit[:, None]).clamp(-127.0, 127.0)
    return codes.to(torch.int8), torch.where(some, most * (1.0 / 127.0), 0.0)


def _product_codes(q, scale, w, w_scale):
    return (q.float() @ w.float().t()) * w_scale * scale[:, None]


def _product8_plain(s):
    q, scale = _codes(s["x"])
    return _product_codes(q, scale, s["weight"], s["scale"]).to(s["x"].dtype)


def _feed8_plain(s):
    F = s["case"]["inner"]
    pre = _product_codes(*_codes(s["x"]), s["w_in"], s["in_scale"])
    h = _act_plain(s["case"]["act"], pre[:, :F])[0] * pre[:, F:]
    return _product_codes(*_codes(h), s["w_out"], s["out_scale"]).to(s["x"].dtype)


def _blocks(flat):
    """flat by blocks, the last filled up with zeros."""
    return torch.cat([flat, flat.new_zeros(-flat.numel() % BLOCK)]).view(-1, BLOCK)


def _put_first(m):
    """(codes, scale by block): sign * (|code| / 127)^2 of the block's largest magnitude."""
    n, m = m.numel(), _blocks(m)
    most = m.abs().amax(dim=1)
    some = most >= LEAST
    unit = torch.where(some, 1.0 / most, 0.0)
    code = torch.round(127.0 * (m.abs() * unit[:, None]).sqrt())
    return torch.where(m < 0.0, -code, code).to(torch.int8).flatten()[:n], torch.where(some, most, 0.0)


def _put_second(v):
    """(codes, scale by block): (code / 255)^4 of the block's largest, its fourth root in steps of a 255th, no code 0
    for a value above 0."""
    n, root = v.numel(), _blocks(v).sqrt()
    most = root.amax(dim=1)
    some = most >= LEAST
    unit = torch.where(some, 1.0 / most, 0.0)
    code = torch.round(255.0 * (root * unit[:, None]).sqrt())
    code = torch.where((root > 0.0) & some[:, None], code.clamp_min(1.0), code)
    return code.to(torch.uint8).flatten()[:n], torch.where(some, most, 0.0)


def _first_values(code, scale):
    n, c = code.numel(), _blocks(code.float())
    return (c * c.abs() * (scale * (1.0 / 16129.0))[:, None]).flatten()[:n]


def _second_values(code, scale):
    n, c = code.numel(), _blocks(code.float())
    return (c * c * (scale * (1.0 / 65025.0))[:, None]).square().flatten()[:n]


def _step_plain(s):
    """In 32 bits: m + w (g - m), v + w (g^2 - v) and p - s (m / (sqrt(v) + eps)) with each operation rounded but the
    last product of the three, which is rounded with its sum.  The tensors lie one behind the other, each filled up to
    whole blocks."""
    c, bits = s["case"], s["case"]["bits"]
    sizes = [p.numel() for p in s["params"]]
    held = [-(-n // BLOCK) * BLOCK for n in sizes]

    def join(parts):
        return torch.cat([_blocks(t.float()) for t in parts]).flatten()

    def split(flat):
        return [t[:n] for t, n in zip(flat.split(held), sizes)]

    p, g = join(s["params"]), join(s["grads"])
    if bits == 8:
        m = join([_first_values(q, t) for q, t in zip(s["first"], s["first_scale"])])
        v = join([_second_values(q, t) for q, t in zip(s["second"], s["second_scale"])])
    else:
        m, v = join(s["first"]), join(s["second"])
    m = torch.lerp(m, g, 1.0 - BETAS[0])
    v = torch.lerp(v, g * g, 1.0 - BETAS[1])
    left = math.sqrt(1.0 - BETAS[1] ** c["step"])
    p = torch.addcdiv(p * (1.0 - 1e-3 * c["decay"]), m, v.sqrt() + EPS * left,
                      value=-(1e-3 * left / (1.0 - BETAS[0] ** c["step"])))
    new = [t.to(q.dtype) for t, q in zip(split(p), s["params"])]
    torch._foreach_copy_(s["params"], new)
    if bits == 32:
        torch._foreach_copy_(s["first"], split(m))
        torch._foreach_copy_(s["second"], split(v))
        return dict(params=s["params"], first=s["first"], second=s["second"])
    (qm, sm), (qv, sv) = _put_first(m), _put_second(v)
    many = [n // BLOCK for n in held]
    torch._foreach_copy_(s["first"], split(qm))
    torch._foreach_copy_(s["second"], split(qv))
    torch._foreach_copy_(s["first_scale"], list(sm.split(many)))
    torch._foreach_copy_(s["second_scale"], list(sv.split(many)))
    return dict(params=s["params"], first=split(_first_values(qm, sm)), second=split(_second_values(qv, sv)))


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "adamw":
        return _step_exact(s)
    x = s["x"]
    if kind == "product8":
        return _integers_exact(x, s["weight"], s["scale"])
    if kind == "feed8":
        pre = _integers_exact(x, s["w_in"], s["in_scale"])
        h = _gate_exact(case["act"], *pre.chunk(2, dim=1))
        return _integers_exact(h, s["w_out"], s["out_scale"])
    a, b = s["w_in"].double(), s["w_out"].double()
    leaves = [x.double().requires_grad_(True), a.requires_grad_(True), b.requires_grad_(True)]
    wants = kind == "feed_grad"
    with torch.set_grad_enabled(wants):
        gate, up = (torch.mm(leaves[0], w.t()) for w in leaves[1].chunk(2))
        y = torch.mm(_gate_exact(case["act"], gate, up), leaves[2].t())
    if not wants:
        return dict(y=y)
    # by torch's own differentiation
    dx, dw_in, dw_out = torch.autograd.grad(y, leaves, s["dy"].double())
    return dict(y=y.detach(), dx=dx, dw_in=dw_in, dw_out=dw_out)


def _gate_exact(act, g, u):
    if act == "silu":
        return u * g * torch.special.expit(g)
    if act == "relu":
        return u * g.clamp_min(0.0)
    if act == "gelu":
        return u * g * torch.special.ndtr(g)
    return u * g * torch.special.expit(2.0 * math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3))


def _integers_exact(x, w, w_scale):
    """Sums of whole numbers, which 64 bits hold; the codes as the definition has them, in 32 bits."""
    f = x.float()
    peak = f.abs().max(dim=1, keepdim=True).values
    zero = peak < LEAST
    codes = torch.mul(f, torch.div(torch.full_like(peak, 127.0), peak).masked_fill(zero, 0.0)).round().clamp(-127, 127)
    step = peak.double().masked_fill(zero, 0.0) / 127.0
    return torch.mm(codes.double(), w.double().t()) * (step * w_scale.double()[None, :])


def _step_exact(s):
    """The parameters, and the states where they are not put in 8 bits: a code is the definition's, in 32 bits."""
    c, b1, b2 = s["case"], *BETAS
    out = dict(params=[], first=[], second=[])
    for i, (p, g) in enumerate(zip(s["params"], s["grads"])):
        p, g = p.double(), g.double()
        if c["bits"] == 32:
            m, v = s["first"][i].double(), s["second"][i].double()
        else:
            at = torch.arange(p.numel(), device=p.device) // BLOCK
            k, j = s["first"][i].double(), s["second"][i].double()
            m = torch.sign(k) * (k / 127.0) ** 2 * s["first_scale"][i].double()[at]
            v = ((j / 255.0) ** 2 * s["second_scale"][i].double()[at]) ** 2
        m, v = b1 * m + (1.0 - b1) * g, b2 * v + (1.0 - b2) * g ** 2
        m_hat, v_hat = m / (1.0 - b1 ** c["step"]), v / (1.0 - b2 ** c["step"])
        out["params"].append((1.0 - 1e-3 * c["decay"]) * p - 1e-3 * m_hat / (v_hat.sqrt() + EPS))
        out["first"].append(m if c["bits"] == 32 else None)
        out["second"].append(v if c["bits"] == 32 else None)
    return out


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    kind, b = case["kind"], BYTES[case["type"]]
    if kind == "adamw":
        n = sum(_sizes(case))
        # parameters and states read and written, gradients read; of 8-bit states the values they stand for come back
        states = 16 if case["bits"] == 32 else 4 + 16 / BLOCK + 8
        return dict(bytes=n * (2 * b + BYTES[case["grads"]] + states), flops=n * (16 if case["bits"] == 32 else 40))
    n, D = case["rows"], case["width"]
    if kind == "product8":
        N = case["cols"]
        return dict(bytes=n * (D + N) * b + N * D + 4 * N, flops=2 * n * D * N)
    F = case["inner"]
    if kind == "feed8":
        return dict(bytes=2 * n * D * b + 3 * D * F + 4 * (2 * F + D), flops=6 * n * D * F)
    grad = kind == "feed_grad"
    return dict(bytes=n * D * b * (4 if grad else 2) + 3 * D * F * b * (2 if grad else 1),
                flops=n * D * F * (18 if grad else 6))
