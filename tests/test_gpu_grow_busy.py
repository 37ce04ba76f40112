"""The grower in rounds on a busy device: eight host threads, each on its own
default-priority stream, grow the same few trees again and again, and every
tree equals the one grown alone.

A scan launch has blocks for the largest round and those past the round's
count return at once.  On a device that other streams keep busy such a block
may start after the launch's controller has planned the next, larger round;
it has to return then too (k_scan's `round`).
"""

import threading

import numpy as np
import pytest
import torch

from yabt_amd import grow_hip as G

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0) if torch.cuda.is_available() else None


def _inputs(n, F, nb, seed):
    rng = np.random.default_rng(seed)
    X = rng.integers(0, nb, size=(n, F))
    lay = G.make_layouts(torch.from_numpy(X.astype(np.uint8)), DEV)
    # gradients with structure, so that the rounds' counts rise and fall
    g = (X[:, 0] > nb // 2) * 1.5 + (X[:, 1] > nb // 3) * (X[:, 2] < nb // 4) + rng.normal(size=n) * 0.3
    h = rng.uniform(0.1, 1.0, size=n)
    return lay, torch.from_numpy(g.astype(np.float32)).to(DEV), torch.from_numpy(h.astype(np.float32)).to(DEV)


def _grow(inputs, nb, max_leaves):
    lay, g, h = inputs
    n, F = lay.n, lay.F
    res = G.grow_device(lay, g, h, np.full(F, nb, np.int32), max_leaves=max_leaves)
    torch.cuda.current_stream().synchronize()
    out = {k: getattr(res, k).cpu().numpy() for k in ("feature", "thr_bin", "left", "right", "depth")}
    out["value"] = res.value.cpu().numpy().view(np.uint32)
    out["leaf"] = G.leaf_ids(res, n, F, max_leaves).cpu().numpy()
    return out


@pytest.mark.parametrize("n,F,max_leaves", [(300_000, 50, 63), (20_000, 130, 31)])
def test_trees_of_busy_streams_are_the_lone_ones(n, F, max_leaves):
    threads, repeats, nb = 8, 12, 256
    inputs = [_inputs(n, F, nb, 100 + s) for s in range(3)]
    alone = [_grow(x, nb, max_leaves) for x in inputs]
    torch.cuda.synchronize()
    print(f"busy streams: {threads} threads x {repeats} trees of {n} x {F}", flush=True)
    wrong, errors = [], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream(DEV)):
                for k in range(repeats):
                    j = (i + k) % len(inputs)
                    got = _grow(inputs[j], nb, max_leaves)
                    wrong.extend((i, k, name) for name in got if not np.array_equal(got[name], alone[j][name]))
        except Exception as e:   # noqa: BLE001 -- reported by the main thread
            errors.append((i, repr(e)))

    ts = [threading.Thread(target=work, args=(i,)) for i in range(threads)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not errors, errors
    assert not wrong, wrong[:8]
