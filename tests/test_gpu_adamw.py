"""yabt_adamw_step against its definition in float32 steps (equal but for the
oracle's own second rounding) and against the formulas in float64."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from yabt_amd import optim

from dense_plain import BLOCK, adamw32, adamw64, put, shown

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
# one value, around the four values of a lane, a block of 256, a wave's 1024 and a thread block's 4096
SIZES = [1, 3, 4, 5, 255, 256, 257, 1023, 1024, 1025, 4095, 4096, 4097, 10_007]
HOW = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)


def name(dt):
    return str(dt).replace("torch.", "")


def tensors(sizes, pt, gt, seed, zeros=0.2):
    gen = torch.Generator().manual_seed(seed)
    p = [torch.randn(n, generator=gen).to(pt) for n in sizes]
    g = [(torch.randn(n, generator=gen) * torch.exp(-6 * torch.rand(n, generator=gen))).to(gt) for n in sizes]
    for t in g:
        t[torch.rand(t.numel(), generator=gen) < zeros] = 0.0
    return p, g


def plain(p, g, m, v, step, lr, betas, eps, weight_decay, f=adamw32, dt=np.float32):
    return f(*(t.astype(dt) for t in (p, g, m, v)), step, lr, *betas, eps, weight_decay)


def near(got, want, steps=1):
    """Equal up to the last place of float32, which the oracle's second rounding may move."""
    got, want = np.asarray(got), np.asarray(want)
    off = np.abs(got.astype(np.float64) - want)
    assert np.all(off <= steps * np.spacing(np.abs(want).astype(np.float32))), np.max(off)


@pytest.mark.parametrize("gt", TYPES, ids=name)
@pytest.mark.parametrize("pt", TYPES, ids=name)
def test_steps_with_32_bits(pt, gt):
    p, g = tensors(SIZES, pt, gt, 1)
    dev = [t.cuda() for t in p]
    state = optim.adamw_state(dev)
    m = [np.zeros(n, np.float32) for n in SIZES]
    v = [np.zeros(n, np.float32) for n in SIZES]
    for step in (1, 2, 3):
        _, g = tensors(SIZES, pt, gt, 10 + step)
        old = [t.float().cpu().numpy() for t in dev]
        before = [(t.cpu().numpy(), s.cpu().numpy()) for t, s in zip(state.first, state.second)]
        optim.adamw_step(dev, [t.cuda() for t in g], state, step, **HOW)
        for i in range(len(SIZES)):
            want, m[i], v[i] = plain(old[i], g[i].float().numpy(), *before[i], step, **HOW)
            near(state.first[i].cpu().numpy(), m[i])
            near(state.second[i].cpu().numpy(), v[i])
            got = dev[i].float().cpu().numpy()
            if pt == torch.float32:
                near(got, want)
            else:                                # one rounding to the type
                u = torch.finfo(pt).eps / 2
                tiny = 2.0 ** -133 if pt == torch.bfloat16 else 2.0 ** -25
                assert np.all(np.abs(got - want) <= u * np.abs(want) * (1 + 1e-6) + tiny)


@pytest.mark.parametrize("step", [1, 7, 100_000])
def test_against_the_formulas_in_64_bits(step):
    """Each of the moments' three operations and the move's nine are off by half a
    unit at most, so the move by 16 units of its size, the parameter by one more."""
    p, g = tensors([5000], torch.float32, torch.float32, 3)
    gen = torch.Generator().manual_seed(9)
    m, v = 0.1 * torch.randn(5000, generator=gen), torch.rand(5000, generator=gen) ** 4
    dev, state = [p[0].cuda()], optim.AdamWState([m.cuda()], [v.cuda()])
    optim.adamw_step(dev, [g[0].cuda()], state, step, **HOW)
    wp, wm, wv = plain(p[0].numpy(), g[0].numpy(), m.numpy(), v.numpy(), step, **HOW, f=adamw64, dt=np.float64)
    u = 2.0 ** -24
    size = 0.9 * np.abs(m.numpy()) + 0.1 * np.abs(g[0].numpy())       # m may cancel
    em = 4 * u * (size + np.abs(g[0].numpy()) + np.abs(m.numpy()))
    assert np.all(np.abs(state.first[0].cpu().numpy() - wm) <= em)
    ev = 4 * u * (v.numpy() + g[0].numpy().astype(np.float64) ** 2)
    assert np.all(np.abs(state.second[0].cpu().numpy() - wv) <= ev)
    left1, left2 = 1 - 0.9 ** step, 1 - 0.999 ** step
    with np.errstate(divide="ignore", invalid="ignore"):
        root = np.sqrt(wv / left2)
        move = HOW["lr"] * np.abs(wm / left1) / (root + HOW["eps"])
        off = HOW["lr"] * em / left1 / (root + HOW["eps"]) + move * (np.where(wv > 0, 0.6 * ev / np.where(wv > 0, wv, 1), 0) + 12 * u)
    assert np.all(np.abs(dev[0].cpu().numpy() - wp) <= off + 4 * u * (np.abs(wp) + move))


@pytest.mark.parametrize("decay", [0.0, 0.1])
def test_the_same_bits_as_torchs_operations(decay):
    p, g = tensors([70_001], torch.float32, torch.float32, 4)
    p, g = p[0].cuda(), g[0].cuda()
    q, m, v = p.clone(), torch.zeros_like(p), torch.zeros_like(p)
    state = optim.adamw_state([q])
    for step in range(1, 20):
        g = g.roll(1) * 1.1
        optim.adamw_step([q], [g], state, step, lr=3e-3, eps=1e-8 / (1 - 0.999 ** step) ** 0.5, weight_decay=decay)
        scale = 3e-3 * (1 - 0.999 ** step) ** 0.5 / (1 - 0.9 ** step)
        m.lerp_(g, 0.1)
        v.lerp_(g.square(), 0.001)
        p.mul_(1.0 - 3e-3 * decay).addcdiv_(m, v.sqrt() + 1e-8, value=-scale)
        assert torch.equal(state.first[0], m) and torch.equal(state.second[0], v) and torch.equal(q, p), step


@pytest.mark.parametrize("pt,gt", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                   (torch.float32, torch.float16)], ids=str)
def test_steps_with_8_bits(pt, gt):
    p, _ = tensors(SIZES, pt, gt, 5)
    dev = [t.cuda() for t in p]
    state = optim.adamw_state(dev, bits=8)
    for step in (1, 2, 3, 4):
        _, g = tensors(SIZES, pt, gt, 20 + step, zeros=0.2 if step < 4 else 1.0)
        old = [t.float().cpu().numpy() for t in dev]
        held = [[t.cpu().numpy() for t in part] for part in (state.first, state.second, state.first_scale, state.second_scale)]
        optim.adamw_step(dev, [t.cuda() for t in g], state, step, **HOW)
        for i, n in enumerate(SIZES):
            m, v = shown(held[0][i], held[2][i], True), shown(held[1][i], held[3][i], False)
            want, m, v = plain(old[i], g[i].float().numpy(), m, v, step, **HOW)
            got = dev[i].float().cpu().numpy()
            u = 0 if pt == torch.float32 else torch.finfo(pt).eps / 2
            assert np.all(np.abs(got - want) <= u * np.abs(want) + 2 * np.spacing(np.abs(want)))
            for code, scale, value, steps, signed in (
                    (state.first[i], state.first_scale[i], m, 127, True),
                    (state.second[i], state.second_scale[i], np.sqrt(v), 255, False)):
                wc, ws = put(value, steps, signed)
                code = code.cpu().numpy().astype(np.int64)
                near(scale.cpu().numpy(), ws)
                # a value within the oracle's last place of a border may have the next code
                root = steps * np.sqrt(np.abs(value).astype(np.float64) / np.maximum(np.repeat(ws, BLOCK)[:n].astype(np.float64), 1e-300))
                border = np.abs(np.abs(root - np.floor(root)) - 0.5) < 1e-4
                assert np.all((code == wc) | border & (np.abs(code - wc) == 1))
                assert signed or np.all(code[value > 0] >= 1)
    mv = state.values()
    for i in range(len(SIZES)):
        assert np.array_equal(mv[0][i].cpu().numpy(), shown(state.first[i].cpu().numpy(), state.first_scale[i].cpu().numpy(), True))
        assert np.array_equal(mv[1][i].cpu().numpy(), shown(state.second[i].cpu().numpy(), state.second_scale[i].cpu().numpy(), False))


def test_8_bits_stay_near_32():
    """A moment's code is off by half a step: by 1/127 of the root of its part of
    the block's largest, so by at most (2 sqrt(part) + 1/254) / 254 of the largest."""
    p, g = tensors([4000], torch.float32, torch.float32, 6)
    a, b = [p[0].cuda()], [p[0].cuda()]
    s32, s8 = optim.adamw_state(a), optim.adamw_state(b, bits=8)
    optim.adamw_step(a, [g[0].cuda()], s32, 1, **HOW)
    optim.adamw_step(b, [g[0].cuda()], s8, 1, **HOW)
    assert torch.equal(a[0], b[0])               # zeros are held exactly
    m = s32.first[0].cpu().numpy()
    most = np.repeat(np.abs(np.concatenate([m, np.zeros(-4000 % 256, np.float32)])).reshape(-1, 256).max(axis=1), 256)[:4000]
    off = np.abs(s8.values()[0][0].cpu().numpy() - m)
    part = np.sqrt(np.abs(m) / most)
    assert np.all(off <= most * (2 * part + 1 / 254) / 254 * 1.0001)


def test_unaligned_views_and_what_lies_beside_them():
    for bits in (32, 8):
        flat = torch.full((9001,), 7.0, device="cuda")
        grads = torch.linspace(-1, 1, 9001, device="cuda").to(torch.bfloat16)
        p, g = flat[1:8000], grads[3:8002]
        q = p.clone()
        s, t = optim.adamw_state([p], bits), optim.adamw_state([q], bits)
        for step in (1, 2):
            optim.adamw_step([p], [g], s, step, **HOW)
            optim.adamw_step([q], [g.clone()], t, step, **HOW)
        assert torch.equal(p, q) and torch.equal(s.values()[0][0], t.values()[0][0])
        assert flat[0] == 7.0 and bool((flat[8000:] == 7.0).all())


def test_more_tensors_than_a_launch_takes_and_none():
    sizes = [(i * 37) % 301 for i in range(131)]            # some of them empty
    p, g = tensors(sizes, torch.float32, torch.float32, 8)
    a, b = [t.cuda() for t in p], [t.cuda() for t in p]
    sa, sb = optim.adamw_state(a), optim.adamw_state(b)
    grads = [None if i % 5 == 0 else t.cuda() for i, t in enumerate(g)]
    optim.adamw_step(a, grads, sa, 1, **HOW)
    for i in range(len(sizes)):
        optim.adamw_step(b[i:i + 1], grads[i:i + 1], optim.AdamWState(sb.first[i:i + 1], sb.second[i:i + 1]), 1, **HOW)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert all(torch.equal(a[i], p[i].cuda()) for i in range(0, len(sizes), 5))
    optim.adamw_step([], [], optim.adamw_state([]), 1)


def test_matrices_and_gradients_of_other_strides():
    gen = torch.Generator().manual_seed(2)
    p, g = torch.randn(64, 33, generator=gen).cuda(), torch.randn(33, 64, generator=gen).cuda()
    q, h = p.clone(), [torch.randn(64, 33, generator=gen).cuda() for _ in range(2)]
    s, t = optim.adamw_state([p, h[0]]), optim.adamw_state([q, h[1]])
    h[1].copy_(h[0])
    optim.adamw_step([p, h[0]], [g.t(), 2 * g.t()], s, 1)
    optim.adamw_step([q, h[1]], [g.t().contiguous(), (2 * g.t()).contiguous()], t, 1)
    assert torch.equal(p, q) and torch.equal(h[0], h[1])


def test_gradients_that_are_not_finite():
    for bits in (32, 8):
        p = torch.ones(600, device="cuda")
        g = torch.ones(600, device="cuda")
        g[300], g[599] = float("nan"), float("inf")
        s = optim.adamw_state([p], bits)
        optim.adamw_step([p], [g], s, 1)
        bad = ~torch.isfinite(p)
        assert bad[300] and bool(torch.isfinite(p[:256]).all()) and int(bad.sum()) <= 2
        m = s.values()[0][0]
        assert bool(torch.isfinite(m[:256]).all()) and not bool(torch.isfinite(m[300]))
        if bits == 8:
            assert bool(torch.isnan(m[256:]).all())


def test_tiny_and_huge_gradients():
    for scale in (1e-38, 1e-30, 1e18):
        for bits in (32, 8):
            gen = torch.Generator().manual_seed(1)
            g = (torch.randn(512, generator=gen) * scale)
            p = torch.zeros(512, device="cuda")
            s = optim.adamw_state([p], bits)
            optim.adamw_step([p], [g.cuda()], s, 1, **HOW)
            want, m, _ = plain(np.zeros(512), g.numpy(), np.zeros(512), np.zeros(512), 1, **HOW)
            near(p.cpu().numpy(), want, 2)
            assert bool(torch.isfinite(s.values()[0][0]).all()) and bool(torch.isfinite(s.values()[1][0]).all())


def test_betas_of_zero():
    p, g = tensors([1000], torch.float32, torch.float32, 11)
    d = p[0].cuda()
    s = optim.adamw_state([d])
    optim.adamw_step([d], [g[0].cuda()], s, 1, betas=(0.0, 0.0))
    assert torch.equal(s.first[0], g[0].cuda()) and torch.equal(s.second[0], (g[0] * g[0]).cuda())


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_count_on(bits):
    p, g = tensors([5000, 77], torch.float32, torch.bfloat16, 12)
    a, b = [t.cuda() for t in p], [t.cuda() for t in p]
    grads = [t.cuda() for t in g]
    sa, sb = optim.adamw_state(a, bits), optim.adamw_state(b, bits)
    step = torch.zeros(1, dtype=torch.int32, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step.add_(1)
        optim.adamw_step(a, grads, sa, step, **HOW)
        with pytest.raises(RuntimeError, match="device tensor"):
            optim.adamw_step(a, grads, sa, 1, **HOW)
    for t in range(1, 6):
        for q in grads:
            q.mul_(1.25)
        graph.replay()
        optim.adamw_step(b, grads, sb, t, **HOW)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(a + sa.first + sa.second, b + sb.first + sb.second)), t


def test_on_another_stream_and_twice_the_same():
    p, g = tensors([30_000], torch.float32, torch.float32, 13)
    out = []
    for k in range(2):
        d, h = p[0].cuda(), g[0].cuda()
        s = optim.adamw_state([d], 8)
        torch.cuda.synchronize()
        with torch.cuda.stream(torch.cuda.Stream()):
            for step in (1, 2, 3):
                optim.adamw_step([d], [h], s, step)
        torch.cuda.synchronize()
        out.append((d, s.first[0], s.second[0]))
    assert all(torch.equal(x, y) for x, y in zip(*out))


def test_refused_on_the_device():
    p, g = [torch.zeros(300, device="cuda") for _ in range(2)], [torch.zeros(300, device="cuda") for _ in range(2)]
    s = optim.adamw_state(p)
    for call, text in [(lambda: optim.adamw_step(p, g, s, 0), "counted"),
                       (lambda: optim.adamw_step(p, g, s, torch.ones(1, device="cuda")), "int32"),
                       (lambda: optim.adamw_step([p[0], p[0]], g, s, 1), "twice"),
                       (lambda: optim.adamw_step(p, [g[0], g[1].view(30, 10)], s, 1), "shapes"),
                       (lambda: optim.adamw_step(p, [g[0], g[1].double()], s, 1), "float32"),
                       (lambda: optim.adamw_step(p, [g[0], g[1].cpu()], s, 1), "must be on"),
                       (lambda: optim.adamw_step([p[0], torch.zeros(300, 2, device="cuda")[:, 0]], g, s, 1), "contiguous"),
                       (lambda: optim.adamw_step([p[0][:299], p[1]], [g[0][:299], g[1]], s, 1), "first moment 0")]:
        with pytest.raises(ValueError, match=text):
            call()


def test_a_parameter_that_requires_a_gradient():
    p = torch.ones(10, device="cuda", requires_grad=True)
    s = optim.adamw_state([p])
    with pytest.raises(RuntimeError, match="autograd"):
        optim.adamw_step([p], [torch.ones(10, device="cuda")], s, 1)
    before = p._version
    with torch.no_grad():
        optim.adamw_step([p], [torch.ones(10, device="cuda")], s, 1)
    assert p._version > before and bool((p < 1.0).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_a_moment_twice_is_refused(bits):
    p = [torch.ones(300, device="cuda"), torch.ones(300, device="cuda"), torch.ones(0, device="cuda"),
         torch.ones(0, device="cuda")]
    g = [torch.ones_like(t) for t in p]
    s = optim.adamw_state(p, bits)
    optim.adamw_step(p, g, s, 1)                      # two empty tensors are not one twice
    moved = [t.clone() for t in p]
    names = ["first", "second"] + ["first_scale", "second_scale"] * (bits == 8)
    for name in names:
        part = getattr(s, name)
        kept, part[1] = part[1], part[0]
        with pytest.raises(ValueError, match="twice"):
            optim.adamw_step(p, g, s, 2)
        part[1] = kept
    assert all(torch.equal(a, b) for a, b in zip(p, moved))
