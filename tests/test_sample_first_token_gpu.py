"""A random number of 0 picks the lowest index that is kept, however little it weighs beside those
that follow it in the same warp: sums before an index are never what a larger sum leaves of them.

Exact: the kept weight before that index is 0, and with it already above 0."""
import numpy as np
import pytest
import torch

from test_sample_gpu import check

pytestmark = pytest.mark.gpu


def rows(V, first):
    """A light logit at index `first`, heavy ones soon after it but in no thread's share with it."""
    rng = np.random.default_rng(V + first)
    l = np.full((6, V), -np.inf, np.float32)
    for r in range(6):
        keep = first + 20 + rng.choice(V - first - 20, 1200, replace=False)
        l[r, keep] = rng.uniform(-3, 0, 1200)
        l[r, first] = -60.0 - r
        l[r, first + 20:first + 90] = rng.uniform(-1, 0, 70)
    return l


@pytest.mark.parametrize("V", [2500, 10751, 70001, 262144])
@pytest.mark.parametrize("first", [0, 26, 700])
@pytest.mark.parametrize("kw", [{}, {"k": 1100}, {"k": 2000}, {"p": 0.5}, {"p": 1 - 2.0**-24}, {"p": 1 - 2.0**-24, "T": 40.0}, {"mp": 1e-30}])
def test_zero_picks_the_first_kept(ops, V, first, kw):
    l = rows(V, first)
    ids, _ = check(ops, l, np.zeros(6, np.float32), **kw)
    if not kw or kw.get("k") == 2000 or "T" in kw or "mp" in kw:
        assert ids.tolist() == [first] * 6


@pytest.mark.parametrize("V", [16384, 100003])
def test_zero_beside_a_long_nucleus(ops, V):
    """Whole rows of even logits with lighter ones before them: the prefix of a top-p is long, and of the
    lighter ones it holds, the first is picked."""
    rng = np.random.default_rng(V)
    l = rng.uniform(-0.5, 0.0, (8, V)).astype(np.float32)
    l[:, :40] = -30.0
    l[:, 3] = np.linspace(-12, -2, 8)
    l[:, 4] = 17.0
    check(ops, l, np.zeros(8, np.float32), p=np.linspace(0.9, 0.9999999, 8).astype(np.float32), T=np.linspace(0.8, 3, 8))
