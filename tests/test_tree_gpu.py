"""Drafted-tree operators on the GPU: attention, RoPE/append at tree positions, acceptance,
compaction and forking of cached rows, against plain 64-bit or row-by-row restatements."""
import ctypes as C
import importlib

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
L = importlib.import_module("gemma4-js_b200._lib")


def random_tree(rng, n, wide=False):
    """parents with parents[i] < i; wide: many of them -1."""
    p = [-1] + [int(rng.integers(-1 if wide else 0, i)) for i in range(1, n)]
    return np.array(p, np.int32)


def depths(parents):
    d = []
    for i, p in enumerate(parents):
        d.append(0 if p < 0 else d[p] + 1)
    return d


def tree_reference(q, k, v, base, parents, window):
    """q [n, H, hd], k and v [rows, hd] in f64: (out, tol) per element.

    tol: one rounding of the result to bf16 (2^-8); one rounding of every weight to bf16 against the
    sum of the rounded weights (2^-8 of sum w |v - out|); scores accumulated in f32 (2^-20 of
    sum |q k|, twice, as a factor of the weights) and f32 sums over the keys (2^-16)."""
    n, H, hd = q.shape
    d = depths(parents)
    out, tol = np.zeros((n, H, hd)), np.zeros((n, H, hd))
    for i in range(n):
        keys = list(range(max(0, base + d[i] - window + 1) if window else 0, base))
        a = i
        while a >= 0:
            if not window or d[i] - d[a] < window:
                keys.append(base + a)
            a = parents[a]
        kk, vv = k[keys], v[keys]
        s = q[i] @ kk.T
        ds = 2.0**-20 * (np.abs(q[i]) @ np.abs(kk).T).max()
        w = np.exp(s - s.max(1, keepdims=True))
        w /= w.sum(1, keepdims=True)
        out[i] = w @ vv
        spread = np.stack([w[h] @ np.abs(vv - out[i, h]) for h in range(H)])
        tol[i] = 2.0**-8 * np.abs(out[i]) + (2.0**-8 + 2 * ds + 2.0**-16) * spread + 1e-6
    return out, tol


def cache_of(rt, ctx, hd, S, stride, rng, ring=0):
    cache = rt.KVCache(ctx, hd, stride if ring else S * stride, ring=ring, nseq=S if ring else 1)
    k, v = cache.storage()
    return cache, k, v


def fill(cache, k, v, seq, stride, pos, kk, vv):
    """Puts positions [0, len) (or the last ring ones) of a sequence into the cache's storage."""
    if not cache.ring:
        k[seq * stride + pos:seq * stride + pos + len(kk)] = kk
        v[seq * stride + pos:seq * stride + pos + len(vv)] = vv
        return
    mirror = cache.seq_rows - cache.ring
    r0 = seq * cache.seq_rows
    for j in range(max(0, len(kk) - cache.ring), len(kk)):
        s = (pos + j) % cache.ring
        for row in ([s, cache.ring + s] if s < mirror else [s]):
            k[r0 + row], v[r0 + row] = kk[j], vv[j]


def run_tree(rt, ctx, ops, seed, S, n, H, hd, contexts, window=0, ring=0, counts=None, shared=False, wide=False, scale=0.3):
    rng = np.random.default_rng(seed)
    trees = np.stack([random_tree(rng, n, wide) for _ in range(S)])
    if shared:
        trees[:] = trees[0]
    stride = max(contexts) + n
    cache, k, v = cache_of(rt, ctx, hd, S, stride, rng, ring)
    g = torch.Generator().manual_seed(seed)
    q = (scale * torch.randn((S, n, H, hd), generator=g)).to(torch.bfloat16)
    data = []
    for s in range(S):
        kk = (scale * torch.randn((contexts[s] + n, hd), generator=g)).to(torch.bfloat16)
        vv = torch.randn((contexts[s] + n, hd), generator=g).to(torch.bfloat16)
        fill(cache, k, v, s, stride, 0, kk.cuda(), vv.cuda())
        data.append((kk.double().numpy(), vv.double().numpy()))
    pos = torch.tensor(contexts, dtype=torch.int32, device="cuda")
    tr = torch.from_numpy(trees[0] if shared else trees).cuda()
    cn = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    out = torch.full((S, n, H, hd), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.attentionTree(q.cuda(), cache, pos, tr, counts=cn, seq_stride=stride, sliding=window > 0, window=window, out=out)
    ctx.check_device()
    out = out.double().cpu().numpy()
    for s in range(S):
        c = n if counts is None else counts[s]
        ref, tol = tree_reference(q[s].double().numpy()[:c], *data[s], contexts[s], trees[s][:c], window)
        err = np.abs(out[s, :c] - ref)
        assert (err <= tol).all(), (s, float((err / tol).max()), np.argwhere(err > tol)[:3])
        assert (out[s, c:] == 7.0).all()
    return out


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("n,H", [(1, 1), (1, 8), (5, 3), (16, 8), (17, 8), (33, 7), (64, 8)])
def test_shapes(rt, ctx, ops, hd, n, H):
    run_tree(rt, ctx, ops, hd + n, 2, n, H, hd, [300, 151])


@pytest.mark.parametrize("context", [0, 1, 2, 15, 63, 64, 65, 120, 127, 128, 129, 191, 255, 256, 257, 1000])
def test_context_lengths(rt, ctx, ops, context):
    for hd in (64, 256, 512):
        run_tree(rt, ctx, ops, context, 1, 9, 8, hd, [context])


@pytest.mark.parametrize("window", [1, 2, 5, 64, 100, 128, 511])
def test_windows(rt, ctx, ops, window):
    """Windows shorter than the tree is deep, and longer than the context."""
    run_tree(rt, ctx, ops, window, 3, 24, 8, 256, [700, 3, 129], window=window)
    run_tree(rt, ctx, ops, window, 2, 24, 4, 128, [0, 513], window=window)


def test_chain_and_star_trees(rt, ctx, ops):
    run_tree(rt, ctx, ops, 1, 2, 64, 8, 256, [200, 77], wide=True)
    rng = np.random.default_rng(0)
    for parents in (np.arange(64) - 1, np.full(64, -1), np.r_[-1, np.zeros(63, int)]):
        S, n, H, hd, base = 1, 64, 8, 256, 130
        cache, k, v = cache_of(rt, ctx, hd, S, base + n, rng)
        g = torch.Generator().manual_seed(3)
        kk, vv, q = (torch.randn(s, generator=g).to(torch.bfloat16) for s in ((base + n, hd), (base + n, hd), (1, n, H, hd)))
        kk, q = kk * 0.25, q * 0.25
        fill(cache, k, v, 0, base + n, 0, kk.cuda(), vv.cuda())
        out = ops.attentionTree(q.cuda(), cache, torch.tensor([base], dtype=torch.int32, device="cuda"),
                                torch.from_numpy(parents.astype(np.int32)).cuda(), sliding=True, window=50)
        ref, tol = tree_reference(q[0].double().numpy(), kk.double().numpy(), vv.double().numpy(), base, parents, 50)
        assert (np.abs(out[0].double().cpu().numpy() - ref) <= tol).all()


def test_long_context_is_split(rt, ctx, ops):
    run_tree(rt, ctx, ops, 5, 1, 8, 8, 256, [20011])
    run_tree(rt, ctx, ops, 6, 2, 27, 7, 512, [9001, 5003])
    run_tree(rt, ctx, ops, 7, 1, 40, 8, 64, [12001])
    run_tree(rt, ctx, ops, 8, 1, 64, 8, 128, [6000], window=4096)


def test_ragged_batch(rt, ctx, ops):
    run_tree(rt, ctx, ops, 9, 6, 20, 8, 256, [0, 1000, 31, 64, 500, 7], counts=[20, 0, 1, 7, 19, 20])
    run_tree(rt, ctx, ops, 10, 40, 12, 8, 256, [int(x) for x in np.random.default_rng(1).integers(0, 900, 40)], shared=True)


@pytest.mark.parametrize("hd", [128, 256, 512])
def test_ring_caches(rt, ctx, ops, hd):
    """Sequences before, at and past the wrap of their ring."""
    run_tree(rt, ctx, ops, 12, 4, 16, 8, hd, [10, 190, 200, 901], window=120, ring=max(16384 // hd, 160))


def test_large_scores(rt, ctx, ops):
    """Scores of some hundred: the running maximum moves far between tiles."""
    run_tree(rt, ctx, ops, 13, 2, 16, 8, 256, [700, 1500], scale=2.0)


def test_masked_rows_may_hold_anything(rt, ctx, ops):
    """NaN and infinities in rows that no row, or only some rows, see: behind the tree, before the
    window, in another branch."""
    S, n, H, hd, base, W = 2, 20, 8, 256, 333, 100
    rng = np.random.default_rng(2)
    stride = base + n + 90
    parents = np.array([-1, 0, 1, 2, 0, 4, 5, -1, 7, 8] + [3] * 10, np.int32)
    clean, got = [], []
    for bad in (False, True):
        cache, k, v = cache_of(rt, ctx, hd, S, stride, rng)
        g = torch.Generator().manual_seed(9)
        k.copy_((0.3 * torch.randn(k.shape, generator=g)).to(torch.bfloat16))
        v.copy_(torch.randn(v.shape, generator=g).to(torch.bfloat16))
        q = (0.3 * torch.randn((S, n, H, hd), generator=g)).to(torch.bfloat16).cuda()
        if bad:
            for s in range(S):
                r0 = s * stride
                for t, val in ((k, float("nan")), (v, float("inf"))):
                    t[r0 + base + n:r0 + stride] = val            # behind the tree
                    t[r0:r0 + base - W + 1] = float("nan")        # before every row's window
                    t[r0 + base + 5] = val                         # node 5: seen by 5 and 6 only
                v[r0 + base + 8, 17] = float("-inf")               # node 8: seen by 8 and 9 only
        pos = torch.full((S,), base, dtype=torch.int32, device="cuda")
        out = ops.attentionTree(q, cache, pos, torch.from_numpy(parents).cuda(), seq_stride=stride, sliding=True, window=W)
        (got if bad else clean).append(out.float().cpu())
    sees_bad = torch.zeros(n, dtype=torch.bool)
    sees_bad[[5, 6, 8, 9]] = True
    assert torch.equal(clean[0][:, ~sees_bad], got[0][:, ~sees_bad])
    assert not torch.isfinite(got[0][:, sees_bad]).all(dim=-1).any()
    ctx.check_device()


def test_rows_and_bad_trees_on_the_device(rt, ctx, ops):
    """A parent at or above its node counts as -1, a sequence past its rows is left out; both raise."""
    hd, n, H, stride = 128, 4, 8, 64
    cache = rt.KVCache(ctx, hd, 2 * stride)
    k, v = cache.storage()
    g = torch.Generator(device="cuda").manual_seed(1)
    k.copy_(0.3 * torch.randn(k.shape, device="cuda", generator=g))
    v.copy_(torch.randn(v.shape, device="cuda", generator=g))
    q = (0.3 * torch.randn((2, n, H, hd), device="cuda", generator=g)).to(torch.bfloat16)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    good = ops.attentionTree(q, cache, t([20, 30]), t([-1, -1, 0, 1]), seq_stride=stride)
    assert ctx.check_device() == 0
    bad = ops.attentionTree(q, cache, t([20, 30]), t([-1, 1, 0, 1]), seq_stride=stride)
    with pytest.raises(rt.G4Error):
        ctx.check_device()
    assert torch.equal(good, bad)
    out = torch.full_like(q, 3.0)
    ops.attentionTree(q, cache, t([20, 61]), t([-1, -1, 0, 1]), seq_stride=stride, out=out)
    with pytest.raises(rt.G4Error):
        ctx.check_device()
    assert torch.equal(out[0], good[0]) and (out[1] == 3.0).all()
    assert ctx.check_device() == 0


def test_matches_attention_rows_on_a_chain(rt, ctx, ops):
    """A chain is causal attention: the rows of g4_attention_rows within the tree's tolerance."""
    S, n, H, hd, stride = 3, 12, 8, 256, 800
    cache = rt.KVCache(ctx, hd, S * stride)
    k, v = cache.storage()
    g = torch.Generator(device="cuda").manual_seed(4)
    k.copy_(0.3 * torch.randn(k.shape, device="cuda", generator=g))
    v.copy_(torch.randn(v.shape, device="cuda", generator=g))
    q = (0.3 * torch.randn((S, n, H, hd), device="cuda", generator=g)).to(torch.bfloat16)
    pos = torch.tensor([700, 13, 512], dtype=torch.int32, device="cuda")
    chain = torch.arange(-1, n - 1, dtype=torch.int32, device="cuda")
    for window in (0, 128):
        a = ops.attentionTree(q, cache, pos, chain, seq_stride=stride, sliding=window > 0, window=window)
        b = torch.empty_like(q)
        rmap = L.G4Rows(pos.data_ptr(), 0, n, 0, 0)
        rt.call("g4_attention_rows", ctx.handle, q.data_ptr(), cache.handle, S * n, H, hd, C.byref(rmap), stride,
                int(window > 0), window, b.data_ptr())
        # each side: one bf16 rounding of the result, and weights rounded to bf16 once on one side (|v| < 6)
        assert (a.float() - b.float()).abs().max() <= 2 * 2.0**-8 * b.float().abs().max() + 2.0**-8


def test_attention_in_a_graph_and_on_another_stream(rt):
    ctx = rt.Context(0)
    ops = rt.GPUOps(ctx)
    hd, n, H, stride, S = 256, 16, 8, 3000, 2
    cache = rt.KVCache(ctx, hd, S * stride)
    k, v = cache.storage()
    k.copy_(0.3 * torch.randn(k.shape, device="cuda"))
    v.copy_(torch.randn(v.shape, device="cuda"))
    q = (0.3 * torch.randn((S, n, H, hd), device="cuda")).to(torch.bfloat16)
    pos = torch.tensor([2000, 2900], dtype=torch.int32, device="cuda")
    parents = torch.arange(-1, n - 1, dtype=torch.int32, device="cuda")
    eager = [ops.attentionTree(q, cache, p, parents, seq_stride=stride).clone()
             for p in (pos, torch.tensor([5, 77], dtype=torch.int32, device="cuda"))]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    ctx.set_stream(side)
    with torch.cuda.stream(side):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = ops.attentionTree(q, cache, pos, parents, seq_stride=stride)
        g.replay()
        side.synchronize()
        assert torch.equal(out, eager[0])
        pos.copy_(torch.tensor([5, 77], dtype=torch.int32))
        g.replay()
        side.synchronize()
        assert torch.equal(out, eager[1])


# ------------------------------------------------------------- RoPE / append --
@pytest.mark.parametrize("hd,ring", [(64, 0), (128, 0), (256, 0), (256, 200), (512, 0), (512, 64)])
def test_qkv_post_at_tree_positions(rt, ctx, hd, ring):
    """Each node equals g4_qkv_post_planes of one row at its depth (q, k rotated there; the same bits),
    stored at its own row; rows behind the count stay."""
    S, n, H, stride, angles = 3, 11, 4, 300, hd // 4
    rng = np.random.default_rng(hd)
    trees = np.stack([random_tree(rng, n) for _ in range(S)])
    counts = [11, 4, 0]
    pos = torch.tensor([190, 0, 77], dtype=torch.int32, device="cuda")
    y = torch.randn((S * n, (H + 2) * hd), device="cuda")
    qn, kn = torch.rand(hd, device="cuda") + 0.5, torch.rand(hd, device="cuda") + 0.5
    cache, k, v = cache_of(rt, ctx, hd, S, stride, rng, ring)
    k.fill_(5.0), v.fill_(5.0)
    q = torch.full((S * n, H, hd), 5.0, dtype=torch.bfloat16, device="cuda")
    tr, cn = torch.from_numpy(trees).cuda(), torch.tensor(counts, dtype=torch.int32, device="cuda")
    planes = L.G4Planes(y.data_ptr(), 1, 0, y.shape[1])
    rmap, tree = L.G4Rows(pos.data_ptr(), 0, n, 0, 0), L.G4Tree(tr.data_ptr(), n, n, cn.data_ptr())
    rt.call("g4_qkv_post_tree", ctx.handle, C.byref(planes), H, hd, qn.data_ptr(), kn.data_ptr(), C.c_float(1e-6), angles,
            C.c_float(1e4), C.byref(rmap), C.byref(tree), S * n, q.data_ptr(), cache.handle, stride)
    ctx.check_device()
    seq_rows = cache.seq_rows if ring else stride
    want_k, want_v = torch.full_like(k, 5.0), torch.full_like(v, 5.0)
    want_q = torch.full_like(q, 5.0)
    for s in range(S):
        d = depths(trees[s])
        for i in range(counts[s]):
            one_q = torch.empty((H, hd), dtype=torch.bfloat16, device="cuda")
            tk, tv = (torch.zeros((512, hd), dtype=torch.bfloat16, device="cuda") for _ in range(2))
            p1 = L.G4Planes(y[s * n + i].data_ptr(), 1, 0, y.shape[1])
            r1 = L.G4Rows(None, 0, 1, int(pos[s]) + d[i], 0)
            rt.call("g4_qkv_post_planes", ctx.handle, C.byref(p1), H, hd, 1, qn.data_ptr(), kn.data_ptr(), C.c_float(1e-6),
                    angles, C.c_float(1e4), C.byref(r1), 1, one_q.data_ptr(), tk.data_ptr(), tv.data_ptr(), 512)
            want_q[s * n + i] = one_q
            at = int(pos[s]) + i
            slots = [at] if not ring else [at % ring] + ([ring + at % ring] if at % ring < seq_rows - ring else [])
            for slot in slots:
                want_k[s * seq_rows + slot], want_v[s * seq_rows + slot] = tk[int(pos[s]) + d[i]], tv[int(pos[s]) + d[i]]
    assert torch.equal(q, want_q) and torch.equal(k, want_k) and torch.equal(v, want_v)


# ------------------------------------------------- acceptance and row moves --
def accept_reference(parents, tokens, picks, count):
    path, cur = [], 0
    if count == 0:
        return [], None
    while True:
        path.append(cur)
        nxt = [c for c in range(cur + 1, count) if parents[c] == cur and tokens[c] == picks[cur]]
        if not nxt:
            return path, picks[cur]
        cur = nxt[0]


@pytest.mark.parametrize("n", [1, 2, 16, 31, 32, 33, 64])
def test_accept(ops, n):
    rng = np.random.default_rng(n)
    S = 37
    trees = np.stack([random_tree(rng, n, wide=s % 2 == 1) for s in range(S)])
    if n > 3:
        trees[0] = np.arange(n) - 1
    tokens, picks = (rng.integers(0, 3, (S, n)).astype(np.int32) for _ in range(2))
    tokens[0], picks[0] = 5, 5  # the whole chain is accepted
    counts = rng.integers(0, n + 1, S).astype(np.int32)
    counts[0] = n
    d = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    for cn in (None, counts):
        path, acc, nxt = ops.treeAccept(d(trees), d(tokens), d(picks), None if cn is None else d(cn))
        path, acc, nxt = path.cpu().numpy(), acc.cpu().numpy(), nxt.cpu().numpy()
        for s in range(S):
            want, w_next = accept_reference(trees[s], tokens[s], picks[s], n if cn is None else int(cn[s]))
            assert acc[s] == len(want) and list(path[s][:len(want)]) == want and (path[s][len(want):] == -1).all()
            assert nxt[s] == (-1 if w_next is None else w_next)
        assert acc[0] == (n if n > 3 else acc[0])


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("ring", [0, 300])
def test_compact(rt, ctx, hd, ring):
    S, n, stride = 5, 40, 400
    rng = np.random.default_rng(hd + ring)
    caches = [rt.KVCache(ctx, hd, 10000 if ring else S * stride, ring=ring, nseq=S if ring else 1) for _ in range(3)]
    caches.append(rt.KVCache(ctx, 64, S * stride))  # caches of several kinds in one call
    pos = np.array([0, 290, 299, 17, 360], np.int32)
    path = np.full((S, n), -1, np.int32)
    acc = np.array([40, 7, 12, 0, 33], np.int32)
    for s in range(S):
        path[s, :acc[s]] = np.sort(rng.choice(n, acc[s], replace=False))
    want = []
    for c in caches:
        for t in c.storage():
            t.copy_(torch.randn(t.shape, device="cuda"))
            if c.ring:  # the mirrored rows of a ring repeat its first slots
                r = t.view(S, c.seq_rows, hd)
                r[:, c.ring:] = r[:, :c.seq_rows - c.ring]
        for t in c.storage():
            w = t.clone()
            rows = w.view(S, c.seq_rows if c.ring else stride, -1)
            for s in range(S):
                for j in range(acc[s]):
                    a, b = int(pos[s]) + j, int(pos[s] + path[s, j])
                    if c.ring:
                        a, b = a % c.ring, b % c.ring
                    rows[s, a] = rows[s, b]
                    if c.ring and a < c.seq_rows - c.ring:
                        rows[s, c.ring + a] = rows[s, b]
            want.append(w)
    d = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    rt.kv_compact(ctx, caches, d(pos), d(path), d(acc), seq_stride=stride)
    ctx.check_device()
    got = [t for c in caches for t in c.storage()]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_compact_leaves_bad_paths_alone(rt, ctx):
    """A path that does not rise, leaves the tree or the cache: that sequence stays as it is, and the
    device error word is raised; the others are moved."""
    S, n, stride, hd = 6, 8, 64, 128
    cache = rt.KVCache(ctx, hd, S * stride)
    k, v = cache.storage()
    k.copy_(torch.randn(k.shape, device="cuda"))
    old = k.clone().view(S, stride, hd)
    d = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    path = d([[0, 2, 5, -1, -1, -1, -1, -1], [0, 2, 2, -1, -1, -1, -1, -1], [0, 9, 10, -1, -1, -1, -1, -1],
              [1, 0, 3, -1, -1, -1, -1, -1], [0, 2, 5, -1, -1, -1, -1, -1], [0, 1, 2, 3, 4, 5, 6, 7]])
    rt.kv_compact(ctx, [cache], d([10, 10, 10, 10, 60, 10]), path, d([3, 3, 3, 3, 3, 9]), seq_stride=stride)
    with pytest.raises(rt.G4Error):
        ctx.check_device()
    new = k.view(S, stride, hd)
    assert torch.equal(new[0, 11], old[0, 12]) and torch.equal(new[0, 12], old[0, 15])
    assert torch.equal(new[1:], old[1:])


@pytest.mark.parametrize("hd", [64, 256, 512])
@pytest.mark.parametrize("ring", [0, 300])
def test_fork(rt, ctx, hd, ring):
    S, stride = 9, 500
    caches = [rt.KVCache(ctx, hd, 10000 if ring else S * stride, ring=ring, nseq=S if ring else 1), rt.KVCache(ctx, 128, S * stride)]
    pos = torch.tensor([437, 12, 0, 1, 2, 3, 4, 5, 0], dtype=torch.int32, device="cuda")
    src, dst = [0, 1, 0, 8, 0], [3, 4, 6, 2, 7]
    old, lens = [], pos.tolist()
    for c in caches:
        for t in c.storage():
            t.copy_(torch.randn(t.shape, device="cuda"))
            old.append(t.clone())
    rt.kv_fork(ctx, caches, pos, src, dst, seq_stride=stride)
    ctx.check_device()
    new = [t for c in caches for t in c.storage()]
    for c, a, b in zip([caches[0]] * 2 + [caches[1]] * 2, old, new):
        rows = c.seq_rows if c.ring else stride
        want = a.view(S, rows, -1).clone()
        for i, j in zip(src, dst):
            held = min(lens[i], c.ring) if c.ring else lens[i]
            want[j, :held] = want[i, :held]
            if c.ring:
                again = min(held, c.seq_rows - c.ring)
                want[j, c.ring:c.ring + again] = want[i, c.ring:c.ring + again]
        assert torch.equal(b.view(S, rows, -1), want)
    for i, j in zip(src, dst):
        lens[j] = lens[i]
    assert pos.tolist() == lens


def test_fork_of_many_sequences_and_bad_positions(rt, ctx):
    S, stride, hd = 301, 20, 64
    cache = rt.KVCache(ctx, hd, S * stride)
    k, _ = cache.storage()
    k.copy_(torch.randn(k.shape, device="cuda"))
    old = k.clone().view(S, stride, hd)
    pos = torch.zeros(S, dtype=torch.int32, device="cuda")
    pos[0], pos[1] = 20, 21
    rt.kv_fork(ctx, [cache], pos, [0] * 299, list(range(2, 301)), seq_stride=stride)
    ctx.check_device()
    assert torch.equal(k.view(S, stride, hd)[2:], old[:1].expand(299, stride, hd)) and (pos[2:] == 20).all()
    rt.kv_fork(ctx, [cache], pos, [1], [5], seq_stride=stride)
    with pytest.raises(rt.G4Error):
        ctx.check_device()
    assert int(pos[5]) == 20


@pytest.mark.parametrize("what", ["compact", "fork"])
@pytest.mark.parametrize("first", ["linear", "ring"])
def test_rows_move_in_all_caches_or_in_none(rt, ctx, what, first):
    """Caches of different extents: a position that only some of them hold changes none of them."""
    S, stride, hd = 3, 40, 64
    caches = [rt.KVCache(ctx, hd, S * stride), rt.KVCache(ctx, hd, 1000, ring=256, nseq=S)]
    if first == "ring":
        caches.reverse()
    old = []
    for c in caches:
        for t in c.storage():
            t.copy_(torch.randn(t.shape, device="cuda"))
            old.append(t.clone())
    pos = torch.tensor([39, 45, 7], dtype=torch.int32, device="cuda")
    if what == "compact":
        path = torch.tensor([[0, 2, -1]] * S, dtype=torch.int32, device="cuda")
        rt.kv_compact(ctx, caches, pos, path, torch.tensor([2, 2, 0], dtype=torch.int32, device="cuda"), seq_stride=stride)
    else:
        rt.kv_fork(ctx, caches, pos, [1], [2], seq_stride=stride)
    with pytest.raises(rt.G4Error):
        ctx.check_device()
    assert all(torch.equal(a, b) for a, b in zip(old, [t for c in caches for t in c.storage()]))
    assert pos.tolist() == [39, 45, 7]


def test_advance_each(rt, ctx):
    pos = torch.tensor([5, 6, 7, 8], dtype=torch.int32, device="cuda")
    by = torch.tensor([2, 0], dtype=torch.int32, device="cuda")
    rt.call("g4_advance_positions_each", ctx.handle, pos.data_ptr(), 1, 2, by.data_ptr())
    ctx.sync()
    assert pos.tolist() == [5, 8, 7, 8]


def test_refusals(rt, ctx, ops):
    d = lambda a, t=torch.int32: torch.tensor(a, dtype=t, device="cuda")  # noqa: E731
    cache, small = rt.KVCache(ctx, 256, 100), rt.KVCache(ctx, 128, 100)
    ringed = rt.KVCache(ctx, 256, 1000, ring=80, nseq=2)
    q = torch.zeros((1, 4, 8, 256), dtype=torch.bfloat16, device="cuda")
    par, pos = d([-1, 0, 1, 2]), d([10])
    bad = [
        lambda: ops.attentionTree(q, small, pos, par),                                   # head dim
        lambda: ops.attentionTree(q.float(), cache, pos, par),                            # type
        lambda: ops.attentionTree(q, cache, pos, par[:3]),                                # tree of other size
        lambda: ops.attentionTree(q, cache, pos, par.long()),
        lambda: ops.attentionTree(q, cache, pos.cpu(), par),
        lambda: ops.attentionTree(q, cache, pos, par, sliding=True, window=0),
        lambda: ops.attentionTree(q.expand(2, 4, 8, 256).contiguous(), cache, d([1, 2]), par, seq_stride=60),
        lambda: ops.attentionTree(q, cache, pos, par, seq_base=1),                        # no such position
        lambda: ops.attentionTree(torch.zeros((1, 65, 8, 256), dtype=torch.bfloat16, device="cuda"), cache, pos,
                                  d([-1] * 65)),
        lambda: ops.attentionTree(torch.zeros((1, 4, 9, 256), dtype=torch.bfloat16, device="cuda"), cache, pos, par),
        lambda: ops.attentionTree(q, ringed, pos, par),                                   # a ring is sliding only
        lambda: ops.attentionTree(q, ringed, pos, par, sliding=True, window=78),          # 4 + 78 - 1 > 80
        lambda: rt.kv_compact(ctx, [cache, cache], pos, par[None], d([1])),               # twice
        lambda: rt.kv_compact(ctx, [cache], pos, par[None], d([1, 2])),
        lambda: rt.kv_compact(ctx, [cache], pos, d([[0] * 65]), d([1])),
        lambda: rt.kv_compact(ctx, [cache], d([1, 2]), d([[0], [0]]), d([1, 1]), seq_stride=60),
        lambda: rt.kv_fork(ctx, [cache], d([1, 2, 3]), [0], [0], seq_stride=30),
        lambda: rt.kv_fork(ctx, [cache], d([1, 2, 3]), [0, 1], [1, 2], seq_stride=30),
        lambda: rt.kv_fork(ctx, [cache], d([1, 2, 3]), [0, 0], [2, 2], seq_stride=30),
        lambda: rt.kv_fork(ctx, [cache], d([1, 2, 3]), [0], [3], seq_stride=30),
        lambda: rt.kv_fork(ctx, [cache], d([1, 2, 3, 4]), [0], [3], seq_stride=30),       # past the cache
        lambda: ops.treeAccept(par, d([[1, 2, 3, 4]]), d([[1, 2, 3]])),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(rt.G4Error):
            f()
            pytest.fail(f"case {i} was not refused")
    assert ctx.check_device() == 0


def test_two_contexts_at_once(rt, ctx, ops):
    """Split and joined attention of two contexts on streams of their own, in flight together."""
    d = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    sides, calls = [], []
    for i, (hd, n, H, base) in enumerate(((256, 8, 8, 5000), (512, 27, 7, 9000))):
        c = rt.Context(0)
        cache = rt.KVCache(c, hd, base + n)
        for t in cache.storage():
            t.copy_(torch.randn(t.shape, device="cuda"))
        q = (torch.randn((1, n, H, hd), device="cuda") / hd**0.5).bfloat16()
        args = (q, cache, d([base]), d(random_tree(np.random.default_rng(i), n)))
        torch.cuda.synchronize()
        c_ops = rt.GPUOps(c)
        want = c_ops.attentionTree(*args)
        torch.cuda.synchronize()
        c.set_stream(torch.cuda.Stream())
        sides.append(c)
        calls.append((c_ops, args, want))
    got = [[o.attentionTree(*a) for o, a, _ in calls] for _ in range(20)]
    torch.cuda.synchronize()
    for c in sides:
        c.check_device()
    for pair in got:
        for out, (_, _, want) in zip(pair, calls):
            assert torch.equal(out, want)
