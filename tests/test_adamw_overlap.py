"""An AdamW step's tensors that overlap are refused: two thread blocks would read
and write the values they share in no order."""

import ctypes

import pytest
import torch

from yabt_amd import _lib, optim

MB = 1 << 20


def table(*tensors):
    """yabt_adamw_tensor's eight words each, a megabyte apart where nothing else is said."""
    words = []
    for i, t in enumerate(tensors):
        at = dict(p=1, g=2, m=3, v=4, sm=5, sv=6)
        d = {k: (8 * i + j) * MB for k, j in at.items()} | dict(n=300, pt=0, gt=0) | t
        words += [d[k] for k in ("p", "g", "m", "v", "sm", "sv", "n")] + [d["pt"] | d["gt"] << 32]
    return (ctypes.c_int64 * len(words))(*words)


# param 0 at 1 MB, its moments at 3 and 4, its scales at 5 and 6; 300 values: 1200 bytes, or 300 of a code and 8 of scales
OVERLAPS = [
    ("the same parameter", [{}, dict(p=MB)], (32, 8)),
    ("a parameter's views", [{}, dict(p=MB + 400)], (32, 8)),
    ("a parameter's last value", [{}, dict(p=MB + 1196)], (32, 8)),
    ("a parameter's first value", [{}, dict(p=MB - 1196)], (32, 8)),
    ("inside a larger one", [dict(n=3000), dict(p=MB + 4000)], (32, 8)),
    ("a moment on a parameter", [dict(m=MB + 100)], (32, 8)),
    ("a moment on another's", [{}, dict(v=3 * MB + 296)], (32, 8)),
    ("both moments", [dict(v=3 * MB)], (32, 8)),
    ("scales on codes", [dict(sv=4 * MB + 296)], (8,)),
    ("both scales", [dict(sm=6 * MB + 4)], (8,)),
    ("a gradient on its parameter, elsewhere", [dict(g=MB + 4)], (32, 8)),
    ("a gradient on its parameter, in 16 bits", [dict(g=MB, gt=1)], (32, 8)),
    ("a gradient on another parameter", [{}, dict(g=MB)], (32, 8)),
    ("a gradient over two parameters", [dict(p=2 * MB - 1200), dict(p=2 * MB, g=2 * MB - 600)], (32, 8)),
    ("a gradient on its scales", [dict(g=5 * MB + 4)], (8,)),
    ("the first of 60 on the last", [dict(p=8 * 59 * MB + MB)] + [{}] * 59, (32, 8)),
]


@pytest.mark.parametrize("what,tensors,bits", OVERLAPS, ids=[o[0] for o in OVERLAPS])
def test_refused_by_the_c_entry(what, tensors, bits):
    lib = _lib.load()
    for b in bits:
        rc = lib.yabt_adamw_step(len(tensors), table(*tensors), b, 1, None, 1e-3, 0.9, 0.999, 1e-8, 0.0, None)
        assert rc == -3 and "overlap" in _lib.last_error(), (rc, _lib.last_error())


@pytest.mark.parametrize("tensors", [[dict(p=2 * MB + 8)], [dict(p=3 * MB)], [dict(g=6 * MB)], [{}, dict(g=MB)]], ids=str)
def test_refused_values(tensors):
    rc = _lib.load().yabt_adamw_values(len(tensors), table(*tensors), None)
    assert rc == -3 and "overlap" in _lib.last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_views_of_one_buffer(bits):
    """Those that lie side by side, and gradients in their place, are taken; overlapping ones leave all as it is."""
    gen = torch.Generator().manual_seed(0)
    flat, grad = torch.randn(2000, generator=gen).cuda(), torch.randn(2000, generator=gen).cuda()
    cuts = [flat[:300], flat[300:1700], flat[1700:]]
    q = [t.clone() for t in cuts]
    s, t = optim.adamw_state(cuts, bits), optim.adamw_state(q, bits)
    optim.adamw_step(cuts, [grad[:300], grad[300:1700], grad[1700:]], s, 1)
    optim.adamw_step(q, [grad[:300].clone(), grad[300:1700].clone(), grad[1700:].clone()], t, 1)
    assert all(torch.equal(a, b) for a, b in zip(cuts + s.first + s.second, q + t.first + t.second))
    optim.adamw_step(cuts, cuts, s, 2)
    optim.adamw_step(q, [b.clone() for b in q], t, 2)
    assert all(torch.equal(a, b) for a, b in zip(cuts + s.first + s.second, q + t.first + t.second))
    before = flat.clone()
    two, halves = [flat[:300], flat[100:400]], [grad[:300], grad[300:600]]
    for params, grads in ((two, halves), ([flat[:300], flat[400:700]], [grad[:300], flat[200:500]])):
        with pytest.raises(ValueError, match="overlap"):
            optim.adamw_step(params, grads, optim.adamw_state(params, bits), 1)
    state = optim.adamw_state([flat[:512]], bits)
    state.first[0] = state.second[0].view(torch.int8) if bits == 8 else flat[500:1012]
    with pytest.raises(ValueError, match="overlap"):
        optim.adamw_step([flat[:512]], [grad[:512]], state, 1)
    assert torch.equal(flat, before)
