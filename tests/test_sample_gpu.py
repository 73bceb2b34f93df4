"""Sampling from f32 logits (g4_sample) against the definition in 64 bits.

Which token a row gives is a comparison of 64-bit sums of up to 786432 weights <= 1: both
sides' sums are within 786432 * 2^-53 < 1e-10 of the real ones (relative to the kept weight), so
ids have to be equal wherever no border lies within 1e-9 of the random number.  Probabilities
are one rounding to f32 (2^-24) away from the quotient.
"""
import ctypes as C

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def reference(l, u, T=1.0, k=0, p=1.0, mp=0.0):
    """(id, prob, distance of u to the next border, ids on both sides of it) of one f32 row."""
    l = np.asarray(l, np.float32).astype(np.float64)
    V = l.size
    ok = ~np.isnan(l) & (l > -np.inf)
    if not ok.any():
        return -1, 0.0, 1.0, {-1}
    idx = np.nonzero(ok)[0]
    rank = idx[np.lexsort((idx, -l[idx]))]
    m = l[rank[0]]
    if not T > 0:
        return int(rank[0]), 1.0, 1.0, {int(rank[0])}
    with np.errstate(invalid="ignore", over="ignore", under="ignore"):
        w = np.where(l[rank] == m, 1.0, np.exp((l[rank] - m) / np.float64(np.float32(T))))
    K = rank.size
    if 1 <= k < V:
        K = min(K, k)
    near = 1.0
    if p <= 0:
        K = 1
    elif p < 1:
        c = np.cumsum(w[:K])
        t = np.float64(np.float32(p)) * c[-1]
        near = min(near, np.abs(np.delete(c, -1) - t).min() / c[-1]) if K > 1 else near
        K = int(np.searchsorted(c, t, side="left")) + 1
    K = min(K, rank.size)
    if mp > 0:
        K = min(K, int((w >= min(np.float64(np.float32(mp)), 1.0)).sum()))
    kept = np.zeros(V)
    kept[rank[:K]] = w[:K]
    cdf = np.cumsum(kept)
    u = np.float32(u)
    u = min(max(float(u), 0.0), 1 - 2.0**-24) if u == u else 0.0
    t = u * cdf[-1]
    i = int(np.searchsorted(cdf, t, side="right"))
    i = min(i, int(np.nonzero(kept)[0][-1]))
    d = np.abs(cdf - t) / cdf[-1]
    if u > 0:
        near = min(near, d[kept > 0].min())
    return i, kept[i] / cdf[-1], near, {i}


def check(ops, logits, u, T=None, k=None, p=None, mp=None, cap=0.0, view=None):
    """Runs the rows of `logits` (numpy f32) and compares each with the reference."""
    R = logits.shape[0]
    dev = (lambda a, t: None if a is None else torch.tensor(np.broadcast_to(np.asarray(a), (R,)).copy(), dtype=t, device="cuda"))
    x = torch.from_numpy(np.ascontiguousarray(logits)).cuda() if view is None else view
    ids, probs = ops.sample(x, dev(u, torch.float32), dev(T, torch.float32), dev(k, torch.int32), dev(p, torch.float32),
                            dev(mp, torch.float32), cap=cap)
    ids, probs = ids.cpu().numpy(), probs.cpu().numpy()
    get = lambda a, r, d: d if a is None else np.broadcast_to(np.asarray(a), (R,))[r]  # noqa: E731
    for r in range(R):
        want, prob, near, _ = reference(logits[r], get(u, r, 0.0), get(T, r, 1.0), int(get(k, r, 0)), float(get(p, r, 1.0)),
                                        float(get(mp, r, 0.0)))
        if near < 1e-9:
            continue
        assert ids[r] == want, (r, ids[r], want, near)
        assert abs(probs[r] - prob) <= 2.0**-23 * prob, (r, probs[r], prob)
    return ids, probs


def rows(R, V, seed, scale=2.5):
    rng = np.random.default_rng(seed)
    return (scale * rng.standard_normal((R, V))).astype(np.float32), rng.random(R).astype(np.float32)


@pytest.mark.parametrize("V", [1, 2, 5, 31, 33, 127, 1000, 4099, 16385, 32003, 131073])
def test_vocab_sizes(ops, V):
    l, u = rows(9, V, V)
    check(ops, l, u)
    check(ops, l, u, T=0.7, k=np.arange(9) * 7)
    check(ops, l, u, T=1.3, p=np.linspace(0.05, 0.99, 9), mp=0.01)


@pytest.mark.parametrize("V", [262144, 300001, 786432])
def test_large_vocabularies(ops, V):
    l, u = rows(5, V, V, scale=3.0)
    check(ops, l, u)
    check(ops, l, u, T=0.8, k=[1, 64, 1000, 5000, V - 1], p=0.95)
    check(ops, l, u, p=[0.1, 0.5, 0.9, 0.99, 0.9999])
    check(ops, l, u, mp=[0.5, 0.1, 0.01, 0.001, 1e-6])


@pytest.mark.parametrize("rows_", [1, 3, 148, 257])
def test_row_counts(ops, rows_):
    l, u = rows(rows_, 3001, rows_)
    check(ops, l, u, T=np.linspace(0.3, 2.0, rows_), k=np.arange(rows_) % 90, p=0.9)


def test_every_setting_at_its_edges(ops):
    l, _ = rows(40, 2000, 4)
    u = np.linspace(0, 1, 40).astype(np.float32)
    check(ops, l, u, T=np.resize([0.0, -1.0, np.nan, 1e-30, 1e-3, 1e30, np.inf, 1.0], 40))
    # temperatures at which (logit - highest) / T passes 2^31, 2^32 and 2^33
    check(ops, l, u, T=np.resize([1e-7, 2e-9, 1e-9, 5e-10, 3e-10, 1e-10], 40))
    check(ops, l, u, T=np.resize([1e-7, 2e-9, 1e-9, 5e-10, 3e-10, 1e-10], 40), mp=1e-6)
    check(ops, l, u, T=np.resize([1e-7, 2e-9, 1e-9, 5e-10, 3e-10, 1e-10], 40), p=0.99)
    check(ops, l, u, k=np.resize([-5, 0, 1, 2, 1023, 1024, 1025, 1999, 2000, 2**31 - 1], 40))
    check(ops, l, u, p=np.resize([-1.0, 0.0, 1e-7, 0.5, 0.999999, 1.0, 2.0, np.nan], 40).astype(np.float32))
    check(ops, l, u, mp=np.resize([-1.0, 0.0, 1e-7, 0.3, 1.0, 5.0, np.nan], 40).astype(np.float32))
    ids, _ = check(ops, l, np.resize([0.0, 1 - 2.0**-24, 1.0, 3.0, -1.0, np.nan], 40).astype(np.float32))
    assert (ids >= 0).all()


def test_masked_and_non_finite_logits(ops):
    l, u = rows(8, 5000, 5)
    l[0, :] = -np.inf
    l[1, :] = np.nan
    l[2, :] = -np.inf
    l[2, 4321] = -3.4e38
    l[3, ::2] = np.nan
    l[4, 7] = l[4, 4000] = np.inf
    l[5, :2500] = -np.inf
    l[6, :] = np.finfo(np.float32).min
    l[7, ::3] = np.finfo(np.float32).min
    for kw in ({}, {"k": 50}, {"p": 0.8}, {"k": 2000, "p": 0.7, "mp": 0.05}):
        ids, probs = check(ops, l, u, **kw)
        assert ids[0] == -1 and ids[1] == -1 and probs[0] == 0 and ids[2] == 4321 and ids[4] in (7, 4000)


@pytest.mark.parametrize("kw", [{}, {"k": 700}, {"k": 3}, {"p": 0.5}, {"p": 0.25, "k": 1000}, {"mp": 1.0}])
def test_equal_logits(ops, kw):
    """Ties go to the lowest index; the weights are whole numbers here, so every border is exact."""
    R, V = 16, 8192
    l = np.zeros((R, V), np.float32)
    l[1::2, ::2] = -0.0  # -0 and +0 are equal
    l[2, 100:] = -5.0
    u = ((np.arange(R) + 0.37) / R).astype(np.float32)
    check(ops, l, u, **kw)
    few = np.random.default_rng(3).integers(0, 3, (R, V)).astype(np.float32)
    check(ops, few, u, **kw)


@pytest.mark.parametrize("order", ["falling", "rising", "blocks", "narrow", "wide"])
def test_rows_in_hard_orders(ops, order):
    """Rows whose large logits lie together, or whose values are nearly equal or far apart."""
    V = 70001
    l, u = rows(6, V, 11)
    l = np.sort(l, axis=1)
    if order == "falling":
        l = l[:, ::-1].copy()
    elif order == "blocks":
        l = np.roll(l, V // 3, axis=1)
    elif order == "narrow":
        l = np.random.default_rng(1).permuted(l, axis=1) * np.float32(1e-4) + np.float32(20.0)
    elif order == "wide":
        l = np.random.default_rng(2).permuted(l, axis=1) * np.float32(1e4)
    for kw in ({}, {"k": 64}, {"k": 1000}, {"k": 30000}, {"p": 0.3}, {"p": 0.95}, {"k": 40000, "p": 0.9}, {"mp": 0.2}):
        check(ops, l, u, **kw)


@pytest.mark.parametrize("V", [16384, 50001])
def test_borders_on_either_side_of_zero(ops, V):
    """Logits of few values, zero among them: a search whose bounds meet between -0 and +0 counts the
    zeros on one side only."""
    l = np.round(np.random.default_rng(V).standard_normal((12, V)) * 12).astype(np.float32) / 8
    u = np.linspace(0.03, 0.97, 12).astype(np.float32)
    check(ops, l, u, p=np.linspace(0.4, 0.99, 12))
    check(ops, l, u, k=(np.linspace(0.2, 0.95, 12) * V).astype(int))
    check(ops, l, u, k=(np.linspace(0.95, 0.2, 12) * V).astype(int), p=0.97)


def test_strided_and_unaligned_rows(ops):
    l, u = rows(7, 1003, 6)
    big = torch.zeros((7, 2048), device="cuda")
    for off in (0, 1, 2, 3, 4):
        view = big[:, off:off + 1003]
        view.copy_(torch.from_numpy(l))
        check(ops, l, u, k=40, p=0.9, view=view)
        check(ops, l, u, view=view)


def test_cap_is_softcap_first(rt, ctx, ops):
    """The same bits as g4_softcap in place and then no cap."""
    l, u = rows(12, 9001, 8, scale=20.0)
    x = torch.from_numpy(l).cuda()
    U = torch.from_numpy(u).cuda()
    k = torch.full((12,), 500, dtype=torch.int32, device="cuda")
    got = ops.sample(x, U, top_k=k, cap=30.0)
    full = ops.sample(x, U, cap=30.0)
    rt.call("g4_softcap", ctx.handle, C.c_void_p(x.data_ptr()), x.numel(), C.c_float(30.0))
    for a, b in ((got, ops.sample(x, U, top_k=k)), (full, ops.sample(x, U))):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("V", [3, 130, 4099, 9001])
def test_cap_keeps_masks_and_the_end_of_the_row(ops, V):
    """A -inf logit stays unpickable under a cap (g4_softcap would make it -cap), and nothing behind
    the row becomes a candidate, whatever the settings ask for."""
    l = np.full((6, V), -np.inf, np.float32)
    l[:, 0] = [5.0, -50.0, -1000.0, 0.0, -np.inf, 300.0]
    x = torch.from_numpy(l).cuda()
    u = torch.full((6,), 0.999999, device="cuda")
    k, p, mp = torch.full((6,), V - 1, dtype=torch.int32, device="cuda"), torch.full((6,), 0.9, device="cuda"), torch.full((6,), 1e-3, device="cuda")
    for kw in ({}, {"top_k": k}, {"top_p": p}, {"min_p": mp}, {"top_k": k, "top_p": p, "min_p": mp}):
        ids, probs = ops.sample(x, u, cap=30.0, **kw)
        assert ids.tolist() == [0, 0, 0, 0, -1, 0] and probs.tolist() == [1, 1, 1, 1, 0, 1]


def test_distribution_of_many_draws(ops):
    """100,000 uniform numbers of an even grid on one row: each token's share is its probability to
    within the grid's step (inverse of a cumulative sum)."""
    l = np.array([[1.0, -2.0, 0.5, 3.0, 2.5, -1.0, 0.0]], np.float32)
    n = 100000
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    x = torch.from_numpy(l).cuda().expand(n, 7)
    ids, _ = ops.sample(x.contiguous(), torch.from_numpy(u).cuda())
    share = np.bincount(ids.cpu().numpy(), minlength=7) / n
    w = np.exp(l[0].astype(np.float64))
    assert np.abs(share - w / w.sum()).max() <= 2.0 / n


def test_captured_call_replays_with_other_settings(rt):
    """One captured call on a stream of its own reads the logits and settings of each replay."""
    ctx = rt.Context(0)
    ops = rt.GPUOps(ctx)
    V, R = 20011, 5
    side = torch.cuda.Stream()
    x = torch.empty((R, V), device="cuda")
    u, T, p = (torch.ones(R, device="cuda") for _ in range(3))
    k = torch.zeros(R, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    ctx.set_stream(side)
    with torch.cuda.stream(side):
        x.zero_()
        ops.sample(x, u, T, k, p)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            ids, probs = ops.sample(x, u, T, k, p)
        for seed in range(4):
            l, un = rows(R, V, 100 + seed)
            kk, pp = [0, 1, 50, 3000][seed], [1.0, 0.9, 0.5, 0.8][seed]
            x.copy_(torch.from_numpy(l))
            u.copy_(torch.from_numpy(un))
            T.fill_(0.9), k.fill_(kk), p.fill_(pp)
            g.replay()
            side.synchronize()
            for r in range(R):
                want, prob, near, _ = reference(l[r], un[r], 0.9, kk, pp)
                if near > 1e-9:
                    assert int(ids[r]) == want


def test_the_same_call_twice_gives_the_same_bits(ops):
    l, u = rows(64, 100003, 9, scale=0.5)
    x, U = torch.from_numpy(l).cuda(), torch.from_numpy(u).cuda()
    p = torch.full((64,), 0.9, device="cuda")
    a = ops.sample(x, U, top_p=p)
    for _ in range(3):
        b = ops.sample(x, U, top_p=p)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_refusals(rt, ops):
    x = torch.zeros((2, 10), device="cuda")
    u = torch.zeros(2, device="cuda")
    for bad in (lambda: ops.sample(x.double(), u), lambda: ops.sample(x.cpu(), u), lambda: ops.sample(x, u[:1]),
                lambda: ops.sample(x, u.double()), lambda: ops.sample(x.t(), torch.zeros(10, device="cuda")),
                lambda: ops.sample(x, u, top_k=u), lambda: ops.sample(x, u, temperature=u.cpu()),
                lambda: ops.sample(torch.zeros((2, 786433), device="cuda"), u)):
        with pytest.raises(rt.G4Error):
            bad()
    ids, _ = ops.sample(x[:0], u[:0])
    assert ids.numel() == 0


@pytest.mark.parametrize("V", [8195, 16384, 70001, 128256, 262144, 786432])
@pytest.mark.parametrize("p", [0.6, 0.9, 0.97, 0.999])
def test_long_nuclei(ops, V, p):
    """Prefixes of some hundred to most of the row's logits, at flat and steep temperatures."""
    l, _ = rows(6, V, V + 1, scale=1.5)
    l[1] *= 0.05  # nearly flat
    l[2] = np.round(l[2] * 8) / 8  # few values, many ties
    l[3, V // 3:] = np.finfo(np.float32).min
    l[4, ::2] = np.nan
    u = np.array([0.0, 0.2, 0.5, 0.999, 1 - 2.0**-24, 0.77], np.float32)
    check(ops, l, u, p=p)
    check(ops, l, u[::-1].copy(), T=np.array([0.5, 3.0, 1.0, 0.02, 1.7, 40.0]), p=p)


def test_long_nuclei_of_rounded_logits(ops):
    """Logits on the bf16 grid lie on the borders of what the search compares them with."""
    l, u = rows(12, 100000, 3, scale=3.0)
    l = torch.from_numpy(l).bfloat16().float().numpy()
    check(ops, l, u, p=np.linspace(0.3, 0.98, 12))
    check(ops, l, u, T=1.9, p=np.linspace(0.98, 0.3, 12))


@pytest.mark.parametrize("rows_", [1, 40, 150, 330])
def test_long_nuclei_of_many_rows(ops, rows_):
    l, u = rows(rows_, 20480, rows_, scale=1.0)
    check(ops, l, u, T=np.linspace(0.2, 2.0, rows_), p=np.linspace(0.2, 0.99, rows_))


def test_long_nuclei_of_capped_strided_rows(rt, ctx, ops):
    """With a cap, from rows that are not 16-byte aligned, the same bits as from capped aligned ones."""
    l, u = rows(5, 30003, 12, scale=10.0)
    big = torch.zeros((5, 40001), device="cuda")
    view = big[:, 3:3 + 30003]
    view.copy_(torch.from_numpy(l))
    U, p = torch.from_numpy(u).cuda(), torch.tensor([0.5, 0.7, 0.9, 0.95, 0.99], device="cuda")
    got = ops.sample(view, U, top_p=p, cap=20.0)
    flat = torch.zeros((5, 30004), device="cuda")[:, :30003]
    capped = torch.from_numpy(l).cuda()
    rt.call("g4_softcap", ctx.handle, C.c_void_p(capped.data_ptr()), capped.numel(), C.c_float(20.0))
    flat.copy_(capped)
    for x in (flat, capped):
        want = ops.sample(x, U, top_p=p)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    check(ops, capped.cpu().numpy(), u, p=[0.5, 0.7, 0.9, 0.95, 0.99], view=capped)


@pytest.mark.parametrize("V", [257, 300, 512, 513, 2047, 2048, 2049])
def test_rankings_of_some_hundred_candidates(ops, V):
    """Rows that are ranked whole: even, crowded at one end, of few values, equal, masked, infinite."""
    rng = np.random.default_rng(V)
    l = rng.standard_normal((9, V)).astype(np.float32)
    l[1] = -np.exp(4 * rng.random(V))
    l[2] = np.round(l[2] * 4) / 4
    l[3] = 1.5
    l[4, : V - 3] = np.finfo(np.float32).min
    l[5, ::2] = -np.inf
    l[6, 5] = l[6, V - 1] = np.inf
    l[7] = np.sort(l[7])[::-1] * 1e-30
    l[8, rng.integers(0, V, 20)] = np.nan
    u = np.array([0.1, 0.5, 0.9, 0.3, 0.7, 0.999, 0.6, 0.0, 0.45], np.float32)
    for kw in ({"p": 0.97}, {"p": 0.9999, "T": 50.0}, {"k": V - 1}, {"k": 290, "p": 0.99}, {"mp": 1e-4}, {"mp": 0.9, "T": 20.0},
               {"k": V // 2 + 1, "p": 0.8, "mp": 1e-3, "T": 3.0}):
        check(ops, l, u, **kw)


def test_two_contexts_at_once(rt, ops):
    """Calls of two contexts on streams of their own, in flight together: the bits of one after the other."""
    sides = [(rt.Context(0), torch.cuda.Stream()) for _ in range(2)]
    data = []
    for i, kw in enumerate(({"top_p": 0.9}, {"top_k": 3000, "min_p": 0.01})):
        l, u = rows(30, 90000 + i, 50 + i, scale=1.2)
        x, U = torch.from_numpy(l).cuda(), torch.from_numpy(u).cuda()
        kw = {k: torch.full((30,), v, dtype=torch.int32 if k == "top_k" else torch.float32, device="cuda") for k, v in kw.items()}
        data.append((x, U, kw, ops.sample(x, U, **kw)))
    torch.cuda.synchronize()
    got = [[], []]
    for (c, s), _ in zip(sides, data):
        c.set_stream(s)
    for _ in range(20):
        for i, (x, U, kw, _) in enumerate(data):
            got[i].append(rt.GPUOps(sides[i][0]).sample(x, U, **kw))
    torch.cuda.synchronize()
    for i, (_, _, _, want) in enumerate(data):
        for ids, probs in got[i]:
            assert torch.equal(ids, want[0]) and torch.equal(probs, want[1])


@pytest.mark.parametrize("V", [300, 5001, 51815, 128256])
def test_min_p_beside_a_long_prefix(ops, V):
    """A min-p that ends before, inside or behind the prefix of a top-p, or of a top-k above 1024."""
    l, u = rows(12, V, V + 7, scale=1.7)
    l[3] = np.round(l[3] * 4) / 4
    l[4, ::2] = np.nan
    l[5] = 0.25
    mp = np.array([0.5, 0.2, 0.1, 0.05, 0.02, 0.02, 0.01, 5e-3, 2e-3, 1e-3, 1e-4, 1e-6], np.float32)
    T = np.linspace(0.4, 2.0, 12)
    for kw in ({"p": 0.9}, {"p": np.linspace(0.1, 0.99, 12)}, {"k": 1500}, {"k": V - 1}, {"k": 3000, "p": 0.8},
               {"k": np.linspace(1025, 9000, 12).astype(int)}):
        check(ops, l, u, T=T, mp=mp, **kw)
        check(ops, l, u[::-1].copy(), mp=mp[::-1].copy(), **kw)
