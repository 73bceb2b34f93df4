"""A top-p next to 1 whose prefix ends among logits that weigh some 1e-11 of the highest.

The weights of a prefix's last candidates are summed as whole numbers of 2^-50 of the highest of them
(so that their order does not matter): n of them lose at most n 2^-50.  Everything else is in 64-bit
floats, 2^-53 of sums just above 1 a few dozen times.  The rows are made so that no border lies within
n 2^-50 + 2^-47 of what it is compared with; the reference sums in 80 bits."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
P = np.float32(1.0 - 2.0**-24)
U = np.float32(1.0 - 2.0**-24)
LIGHT = 8000


def row(V, seed):
    """One logit of 0, 8000 around -24.9 in falling order of index (the last ranks last), nothing else."""
    rng = np.random.default_rng(seed)
    l = np.full(V, -np.inf, np.float32)
    l[0] = 0.0
    at = np.sort(rng.choice(np.arange(1, V), LIGHT, replace=False))
    l[at] = np.sort(rng.uniform(-25.5, -24.3, LIGHT).astype(np.float32))[::-1]
    return l


def reference(l):
    """(id, probability, distance to the nearest border, number of light logits kept)."""
    idx = np.nonzero(l > -np.inf)[0]
    rank = idx[np.lexsort((idx, -l[idx]))]
    w = np.exp(l[rank].astype(np.longdouble))
    c = np.cumsum(w)
    t = np.longdouble(P) * c[-1]
    keep = int(np.searchsorted(c, t, side="left")) + 1
    near = np.abs(c - t).min()
    kept = np.sort(rank[:keep])
    wk = np.exp(l[kept].astype(np.longdouble))
    ck = np.cumsum(wk)
    target = np.longdouble(U) * ck[-1]
    i = int(np.searchsorted(ck, target, side="right"))
    return int(kept[i]), float(wk[i] / ck[-1]), float(min(near, np.abs(ck[:-1] - target).min())), keep - 1


@pytest.mark.parametrize("V", [16384, 65536, 262144])
def test_the_prefix_ends_among_light_logits(ops, V):
    bound = lambda n: n * 2.0**-50 + 2.0**-47  # noqa: E731
    rows, want, seed = [], [], 0
    while len(rows) < 12:
        l = row(V, seed)
        i, p, near, n = reference(l)
        if near > bound(n):
            rows.append(l), want.append((i, p))
        seed += 1
        assert seed < 60
    x = torch.from_numpy(np.stack(rows)).cuda()
    R = len(rows)
    ids, probs = ops.sample(x, torch.full((R,), float(U), device="cuda"), top_p=torch.full((R,), float(P), device="cuda"))
    assert ids.tolist() == [i for i, _ in want]
    assert np.allclose(probs.cpu().numpy(), [p for _, p in want], rtol=2.0**-23, atol=0)
