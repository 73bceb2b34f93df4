"""Measured cases of the sampling, drafted-tree and cache-row operators.

Four operators of a decode server:

  sample   one token per row of f32 logits: temperature, top-k, top-p and min-p, from one
           given uniform number per row
  tree     attention of a tree of drafted tokens (one bf16 KV head, up to 8 query heads)
           over each sequence's cached keys and the node's own ancestors
  commit   the accepted path of the tree (drafted tokens against the model's picks), and
           its K/V rows moved together behind the cached ones in every layer's cache
  fork     a sequence's cached rows copied to other sequences in every layer's cache

With `own` false, run() computes them from elementary torch operations; with `own` true it
calls this package's operators on the same data.
"""
import importlib
import math

import torch

own = False

_CTX = None  # the package's context and operators, made once as a serving program does


def _runtime():
    global _CTX
    if _CTX is None:
        rt = importlib.import_module("gemma4-js_b200.runtime")
        ctx = rt.Context(torch.cuda.current_device())
        _CTX = (rt, ctx, rt.GPUOps(ctx))
    return _CTX


# ------------------------------------------------------------------ cases ---
def listed():
    return [
        # One sequence, the benchmark model's vocabulary, the usual chat settings: the latency of a decode step.
        {"name": "sample_one_row", "op": "sample", "rows": 1, "vocab": 262144, "top_k": 64, "top_p": 0.95, "min_p": 0.0},
        # The benchmark's serving batch, each row with settings of its own around the usual ones.
        {"name": "sample_batch_topk", "op": "sample", "rows": 256, "vocab": 262144, "top_k": 64, "top_p": 0.95, "min_p": 0.0},
        # Nucleus sampling without a top-k: the mass of the whole row decides.
        {"name": "sample_batch_nucleus", "op": "sample", "rows": 64, "vocab": 262144, "top_k": 0, "top_p": 0.9, "min_p": 0.0},
        # Plain temperature sampling with a min-p floor, odd row count, odd vocabulary (rows not 16-byte aligned).
        {"name": "sample_minp_odd", "op": "sample", "rows": 37, "vocab": 32003, "top_k": 0, "top_p": 1.0, "min_p": 0.02},
        # One sequence, a short draft over a full cache of a global layer: the latency of a verify step.
        {"name": "tree_one_seq", "op": "tree", "nseq": 1, "nodes": 8, "heads": 8, "hd": 256, "context": 4096, "window": 0},
        # A serving batch with mid-size trees in a sliding layer.
        {"name": "tree_batch_window", "op": "tree", "nseq": 64, "nodes": 16, "heads": 8, "hd": 256, "context": 4096, "window": 512},
        # A serving batch with the largest trees in a global layer: the arithmetic counts.
        {"name": "tree_batch_large", "op": "tree", "nseq": 32, "nodes": 64, "heads": 8, "hd": 256, "context": 4096, "window": 0},
        # One long document at the wide head dimension of the checkpoint's global layers, odd length, 7 heads.
        {"name": "tree_long_hd512", "op": "tree", "nseq": 2, "nodes": 27, "heads": 7, "hd": 512, "context": 65501, "window": 0},
        # The end of a verify step of one sequence over the sliding layers' caches.
        {"name": "commit_one_seq", "op": "commit", "nseq": 1, "nodes": 16, "hd": 256, "caches": 28, "stride": 1024},
        # The same of a serving batch over the global layers' caches.
        {"name": "commit_batch", "op": "commit", "nseq": 256, "nodes": 32, "hd": 256, "caches": 7, "stride": 704},
        # One prompt, a second completion of it: a short prompt in a few caches.
        {"name": "fork_one", "op": "fork", "nseq": 2, "sources": 1, "hd": 256, "caches": 7, "context": 600, "stride": 1024},
        # Four prompts of up to 4096 tokens, eight sequences each.
        {"name": "fork_batch", "op": "fork", "nseq": 32, "sources": 4, "hd": 256, "caches": 7, "context": 4096, "stride": 4352},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        b = most.setdefault(c["op"], [0.0, 0.0])
        b[0], b[1] = max(b[0], w["bytes"]), max(b[1], w["flops"])
    while True:
        op = rng.choice(["sample", "sample", "tree", "tree", "tree", "commit", "fork"])
        if op == "sample":
            c = {"op": op, "rows": _log_int(rng, 1, 256), "vocab": _log_int(rng, 64, 262144),
                 "top_k": rng.choice([0, 0, 1, 20, 64, 200, 1000, 3000]), "top_p": rng.choice([1.0, 0.95, 0.9, 0.5]),
                 "min_p": rng.choice([0.0, 0.0, 0.02, 0.1])}
        elif op == "tree":
            c = {"op": op, "nseq": _log_int(rng, 1, 64), "nodes": _log_int(rng, 1, 64), "heads": rng.choice([8, 8, 4, rng.randint(1, 8)]),
                 "hd": rng.choice([64, 128, 256, 256, 512]), "context": _log_int(rng, 1, 32768),
                 "window": rng.choice([0, 0, 512, _log_int(rng, 1, 2048)])}
        elif op == "commit":
            c = {"op": op, "nseq": _log_int(rng, 1, 256), "nodes": _log_int(rng, 1, 64), "hd": rng.choice([64, 128, 256, 512]),
                 "caches": rng.randint(1, 28), "stride": _log_int(rng, 128, 704)}
        else:
            s = rng.randint(1, 4)
            stride = _log_int(rng, 64, 4352)
            c = {"op": op, "nseq": s + _log_int(rng, 1, 28), "sources": s, "hd": rng.choice([64, 128, 256, 512]),
                 "caches": rng.randint(1, 7), "context": _log_int(rng, 1, stride), "stride": stride}
        w = work(c)
        if w["bytes"] <= most[op][0] and w["flops"] <= max(most[op][1], 1.0):
            return c


def work(case):
    """Bytes and operations of one pass: inputs read once, outputs written once."""
    op = case["op"]
    if op == "sample":
        n = case["rows"] * case["vocab"]
        # 4 B per logit, one token and one probability per row; a weight (about 20 operations) per logit where
        # the mass of the whole row is asked for
        return {"bytes": 4.0 * n + 28.0 * case["rows"], "flops": float(n) * (2 if case["top_k"] else 22)}
    if op == "tree":
        ctx = 0.75 * case["context"]  # lengths are spread over [context / 2, context]
        seen = min(ctx, case["window"]) if case["window"] else ctx
        rows = case["nseq"] * case["nodes"]
        kv = case["nseq"] * (seen + case["nodes"]) * case["hd"] * 4.0
        depth = 1 + math.log2(case["nodes"] + 1) / 2
        return {"bytes": kv + rows * case["heads"] * case["hd"] * 4.0,
                "flops": 4.0 * rows * case["heads"] * case["hd"] * (seen + depth)}
    if op == "commit":
        moved = case["nseq"] * 0.5 * _depth_of(case["nodes"])  # about half of the accepted rows change their place
        return {"bytes": moved * case["caches"] * case["hd"] * 8.0 + 20.0 * case["nseq"] * case["nodes"], "flops": 0.0}
    rows = 0.75 * case["context"] * case["hd"] * 4.0 * case["caches"]
    return {"bytes": rows * case["nseq"], "flops": 0.0}


def _depth_of(nodes):
    return max(1, min(nodes, int(2 + math.log2(nodes))))


# ------------------------------------------------------------------ inputs --
def _trees(nseq, nodes, g):
    """parents [nseq, nodes]: node 0 is the root; a later node hangs under one of the nodes before it, the
    recent ones more often (drafts go deep before they go wide)."""
    i = torch.arange(nodes, device="cuda")
    back = (torch.rand((nseq, nodes), device="cuda", generator=g) ** 2 * i).floor().long() + 1
    parents = (i - back).clamp(min=0)
    parents[:, 0] = -1
    return parents.to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]

    def rand(*shape):
        return torch.rand(shape, device="cuda", generator=g)

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=g)

    if op == "sample":
        R, V = case["rows"], case["vocab"]
        # A language model's rows: weights fall off as a power of the rank, steeper in sure rows than in unsure
        # ones; capped to (-30, 30) as the head's logits are.
        steep = 1.2 + rand(R, 1)
        logits = 12.0 - steep * torch.log1p(V * rand(R, V)) + 0.25 * normal(R, V)
        state = {"op": op, "logits": 30.0 * torch.tanh(logits / 30.0), "uniform": rand(R),
                 "temperature": 0.6 + 0.8 * rand(R), "top_k": None, "top_p": None, "min_p": None}
        if case["top_k"]:
            k = torch.randint(1, 2 * case["top_k"], (R,), device="cuda", generator=g)
            state["top_k"] = k.to(torch.int32)
        if case["top_p"] < 1.0:
            state["top_p"] = (case["top_p"] + (0.5 - rand(R)) * (1.0 - case["top_p"])).clamp(0.05, 1.0)
        if case["min_p"] > 0.0:
            state["min_p"] = case["min_p"] * (0.5 + rand(R))
        if own:
            state["rt"] = _runtime()
        return state

    hd, S = case["hd"], case["nseq"]
    if op == "tree":
        n, ctx = case["nodes"], case["context"]
        stride = ctx + n
        pos = (ctx // 2 + (rand(S) * (ctx - ctx // 2 + 1)).long()).clamp(max=ctx).to(torch.int32)
        # normed keys and queries, unit values; what lies behind a sequence's rows is left at zero, as in a new cache
        k = (0.3 * normal(S, stride, hd)).to(torch.bfloat16)
        v = normal(S, stride, hd).to(torch.bfloat16)
        used = (torch.arange(stride, device="cuda") < pos[:, None] + n)[..., None]
        k, v = k * used, v * used
        state = {"op": op, "k": k, "v": v, "pos": pos, "parents": _trees(S, n, g), "window": case["window"],
                 "q": (0.3 * normal(S, n, case["heads"], hd)).to(torch.bfloat16)}
        if own:
            rt, ctx_, ops = state["rt"] = _runtime()
            cache = rt.KVCache(ctx_, hd, S * stride)
            cache.append(k.view(S * stride, hd), v.view(S * stride, hd), S * stride, 0)
            state["cache"], state["stride"] = cache, stride
        return state

    C, stride = case["caches"], case["stride"]
    k = normal(C, S, stride, hd).to(torch.bfloat16)
    v = normal(C, S, stride, hd).to(torch.bfloat16)
    if op == "commit":
        n = case["nodes"]
        parents = _trees(S, n, g)
        # Picks over a small alphabet next to the drafted tokens: a walk that accepts some of the nodes.
        tokens = torch.randint(0, 262144, (S, n), device="cuda", generator=g)
        child = torch.zeros((S, n), dtype=torch.int64, device="cuda")
        child.scatter_reduce_(1, parents.long().clamp(min=0), torch.arange(n, device="cuda").expand(S, n).contiguous(), "amax")
        follow = rand(S, n) < 0.85
        picks = torch.where(follow, tokens.gather(1, child), torch.randint(0, 262144, (S, n), device="cuda", generator=g))
        pos = (rand(S) * (stride - n + 1)).long().clamp(max=stride - n)
        state = {"op": op, "parents": parents, "tokens": tokens.to(torch.int32), "picks": picks.to(torch.int32),
                 "pos": pos.to(torch.int32)}
    else:
        m = case["sources"]
        ctx = case["context"]
        pos = (ctx // 2 + (rand(S) * (ctx - ctx // 2 + 1)).long()).clamp(max=ctx).to(torch.int32)
        dst = list(range(m, S))
        state = {"op": op, "pos": pos, "src": [d % m for d in dst], "dst": dst}
    state["stride"] = stride
    if own:
        rt, ctx_, ops = state["rt"] = _runtime()
        state["caches"] = []
        for c in range(C):
            cache = rt.KVCache(ctx_, hd, S * stride)
            cache.append(k[c].view(S * stride, hd), v[c].view(S * stride, hd), S * stride, 0)
            state["caches"].append(cache)
        views = [c.storage() for c in state["caches"]]
        state["out_k"] = [a.view(S, stride, hd) for a, _ in views]
        state["out_v"] = [b.view(S, stride, hd) for _, b in views]
    else:
        state["k"], state["v"] = k, v
    return state


# --------------------------------------------------------------- one pass ---
def run(state):
    op = state["op"]
    if op == "sample":
        return _sample_own(state) if own else _sample_plain(state)
    if op == "tree":
        return _tree_own(state) if own else _tree_plain(state)
    if op == "commit":
        return _commit_own(state) if own else _commit_plain(state)
    return _fork_own(state) if own else _fork_plain(state)


def _sample_own(s):
    _, _, ops = s["rt"]
    ids, probs = ops.sample(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                            min_p=s["min_p"])
    return {"ids": ids, "probs": probs}


def _tree_own(s):
    _, _, ops = s["rt"]
    return ops.attentionTree(s["q"], s["cache"], s["pos"], s["parents"], seq_stride=s["stride"],
                             sliding=s["window"] > 0, window=s["window"])


def _commit_own(s):
    rt, ctx, ops = s["rt"]
    path, accepted, nxt = ops.treeAccept(s["parents"], s["tokens"], s["picks"])
    rt.kv_compact(ctx, s["caches"], s["pos"], path, accepted, seq_stride=s["stride"])
    return {"accepted": accepted, "next": nxt, "k": s["out_k"], "v": s["out_v"]}


def _fork_own(s):
    rt, ctx, ops = s["rt"]
    rt.kv_fork(ctx, s["caches"], s["pos"], s["src"], s["dst"], seq_stride=s["stride"])
    return {"pos": s["pos"], "k": s["out_k"], "v": s["out_v"]}


def _sample_plain(s):
    """In 64 bits: a sum of 262144 weights next to the border of a token decides which token it is."""
    l = s["logits"].double()
    V = l.shape[1]
    order = torch.sort(l, dim=1, descending=True, stable=True).indices  # ties: the lowest index first
    ranked = l.gather(1, order)
    w = torch.exp((ranked - ranked[:, :1]) / s["temperature"].double()[:, None])
    rank = torch.arange(V, device=l.device)
    keep = torch.ones_like(w, dtype=torch.bool)
    if s["top_k"] is not None:
        k = s["top_k"].long()[:, None]
        keep = (rank < k) | (k >= V)
    if s["top_p"] is not None:
        p = s["top_p"].double()[:, None]
        mass = torch.cumsum(w * keep, dim=1)
        keep = keep & ((mass - w * keep < p * mass[:, -1:]) | (p >= 1.0) | (rank == 0))
    if s["min_p"] is not None:
        keep = keep & (w >= s["min_p"].double()[:, None])
    kept = torch.zeros_like(w).scatter_(1, order, w * keep)  # back in vocabulary order
    cdf = torch.cumsum(kept, dim=1)
    total = cdf[:, -1:]
    ids = torch.searchsorted(cdf, s["uniform"].double()[:, None] * total, right=True).clamp(max=V - 1)
    return {"ids": ids[:, 0].to(torch.int32), "probs": (kept.gather(1, ids) / total)[:, 0].float()}


def _ancestors(parents):
    """[S, n, n] truth values: node j is node i or one of its ancestors."""
    S, n = parents.shape
    p = parents.long()
    edge = torch.eye(n, device=p.device).expand(S, n, n).clone()
    edge.scatter_add_(2, p.clamp(min=0)[..., None], (p >= 0).float()[..., None])
    seen = edge
    for _ in range(6):  # 2^6 steps: every ancestor of up to 64 nodes
        seen = (torch.bmm(seen, seen) > 0).float()
    return seen > 0


def _tree_plain(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    S, n, H, hd = q.shape
    rows = k.shape[1]
    pos = s["pos"].long()
    anc = _ancestors(s["parents"])
    depth = anc.sum(2) - 1
    j = torch.arange(rows, device=q.device)[None, None]
    at = pos[:, None] + depth                                      # the position of each node
    node = (j - pos[:, None, None]).clamp(0, n - 1).expand(S, n, rows)
    key_at = torch.where(j < pos[:, None, None], j, pos[:, None, None] + depth[:, None].expand(S, n, n).gather(2, node))
    see = (j < pos[:, None, None]) | ((j < pos[:, None, None] + n) & anc.gather(2, node))
    if s["window"]:
        see = see & (key_at + s["window"] > at[..., None])
    logits = torch.bmm(q.reshape(S, n * H, hd), k.transpose(1, 2)).view(S, n, H, rows)
    logits = torch.where(see[:, :, None], logits, torch.full((), -math.inf, device=q.device))
    w = torch.exp(logits - logits.amax(3, keepdim=True))
    out = torch.bmm(w.view(S, n * H, rows), v).view(S, n, H, hd)
    return (out / w.sum(3, keepdim=True)).to(torch.bfloat16)


def _accept_plain(s):
    parents, tokens, picks = s["parents"].long(), s["tokens"], s["picks"]
    S, n = parents.shape
    i = torch.arange(n, device=parents.device)
    agrees = (parents >= 0) & (tokens == picks.gather(1, parents.clamp(min=0)))
    # of several children with the picked token the first one is taken
    twin = (parents[:, :, None] == parents[:, None]) & (i[None, :, None] > i[None, None]) & agrees[:, None]
    taken = (agrees & ~twin.any(2)) | (i == 0)
    anc = _ancestors(parents)
    on_path = (taken[:, None] | ~anc).all(2) & anc[:, :, 0]
    accepted = on_path.sum(1)
    path = torch.sort(torch.where(on_path, i, n), dim=1).values
    last = path.gather(1, accepted[:, None] - 1)
    return path, accepted, picks.gather(1, last)[:, 0]


def _commit_plain(s):
    path, accepted, nxt = _accept_plain(s)
    S, n = path.shape
    seq = torch.arange(S, device=path.device)[:, None]
    j = torch.arange(n, device=path.device)
    dst = s["pos"].long()[:, None] + j
    src = torch.where(j < accepted[:, None], s["pos"].long()[:, None] + path, dst)
    s["k"][:, seq, dst] = s["k"][:, seq, src]
    s["v"][:, seq, dst] = s["v"][:, seq, src]
    return {"accepted": accepted.to(torch.int32), "next": nxt.to(torch.int32), "k": list(s["k"].unbind(0)),
            "v": list(s["v"].unbind(0))}


def _fork_plain(s):
    k, v = s["k"], s["v"]
    src = torch.tensor(s["src"], device=k.device)
    dst = torch.tensor(s["dst"], device=k.device)
    rows = (torch.arange(k.shape[2], device=k.device) < s["pos"][src].long()[:, None])[..., None]
    k[:, dst] = torch.where(rows, k[:, src], k[:, dst])
    v[:, dst] = torch.where(rows, v[:, src], v[:, dst])
    s["pos"][dst] = s["pos"][src]
    return {"pos": s["pos"], "k": list(k.unbind(0)), "v": list(v.unbind(0))}


# ------------------------------------------------ the definition in 64 bits --
def exact(case, seed):
    s = prepare(case, seed)

    def prob(r):
        """The probability of the picked token of row r, from thresholds on the row (no ranking of all of it)."""
        l = s["logits"][r].double()
        V = l.numel()
        w = ((l - l.max()) / s["temperature"][r].double()).exp()
        inside = torch.ones(V, dtype=torch.bool, device=l.device)

        def first(count):  # the `count` highest logits, the lowest indices among equal ones
            level = l.topk(count).values[-1]
            above = l > level
            return above | ((l == level) & ((l == level).cumsum(0) <= count - int(above.sum())))

        if s["top_k"] is not None and int(s["top_k"][r]) < V:
            inside = first(int(s["top_k"][r]))
        if s["top_p"] is not None and float(s["top_p"][r]) < 1.0:
            need = float(s["top_p"][r].double()) * float(w[inside].sum())
            lo, hi = 1, int(inside.sum())
            while lo < hi:  # the smallest prefix that holds the mass
                mid = (lo + hi) // 2
                lo, hi = (lo, mid) if float(w[first(mid)].sum()) >= need else (mid + 1, hi)
            inside = first(lo)
        if s["min_p"] is not None:
            inside = inside & (w >= s["min_p"][r].double())
        total = w[inside].sum()
        reach = (w * inside).cumsum(0) > s["uniform"][r].double() * total
        return w[int(reach.to(torch.int8).argmax())] / total

    def rows(b):
        """One sequence's rows: each node's visible rows collected by walking up its parents."""
        n = s["q"].shape[1]
        pos, W = int(s["pos"][b]), s["window"]
        parents = s["parents"][b].tolist()
        depth, see = [], torch.zeros((n, s["k"].shape[1]), dtype=torch.bool)
        for i in range(n):
            depth.append(0 if parents[i] < 0 else depth[parents[i]] + 1)
            see[i, max(0, pos + depth[i] - W + 1) if W else 0:pos] = True
            a = i
            while a >= 0:
                see[i, pos + a] = not W or depth[i] - depth[a] < W
                a = parents[a]
        q, k, v = s["q"][b].double(), s["k"][b].double(), s["v"][b].double()
        p = torch.softmax((q @ k.T).masked_fill(~see.cuda()[:, None], -math.inf), dim=2)
        return p @ v

    if case["op"] == "sample":
        return {"ids": None, "probs": torch.stack([prob(r) for r in range(case["rows"])])}
    if case["op"] == "tree":
        return torch.stack([rows(b) for b in range(case["nseq"])])
    return None  # rows are moved, not computed
