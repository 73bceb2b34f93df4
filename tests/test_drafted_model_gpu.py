"""Drafted, sampled and forked decoding of the whole model: the operators used together."""
import importlib

import numpy as np
import pytest
import torch

from test_sample_gpu import reference

pytestmark = pytest.mark.gpu
model = importlib.import_module("gemma4-js_b200.model")
W_KW = dict(embed_sigma=0.03, embed_tail=0.5)


def small_cfg(**kw):
    base = dict(hidden=512, layers=5, vocab=4096, intermediate=1024, intermediate_late=1024, window=16)
    base.update(kw)
    return model.ModelConfig().small(**base)


def greedy_run(m, prompts, steps):
    B = len(prompts)
    cur = torch.tensor([m.prefill(s, p) for s, p in enumerate(prompts)], dtype=torch.int32, device="cuda")
    out = [cur.tolist()]
    for _ in range(steps):
        cur = m.decode_step(ids_dev=cur, batch=B).clone()
        out.append(cur.tolist())
    return np.array(out, np.int32).T  # [B, steps + 1]


def build(rt, ctx, cfg, w, B, **kw):
    return model.Gemma4Model(ctx, cfg, w, max_batch=B, max_seq=kw.pop("max_seq", 96), max_rows=kw.pop("max_rows", 40), **kw)


@pytest.mark.parametrize("shape", ["ring", "linear", "shared_hd512"])
def test_drafted_greedy_decoding_gives_the_greedy_tokens(rt, shape):
    """Trees of 8 nodes whose branches hold some of the greedy continuation: every step accepts
    exactly the nodes that agree, and the tokens are those of plain decoding.  (16 rows a step: the
    linears of plain decode steps, row for row the same bits.)"""
    kw = dict(head_dim_global=512, kv_share=True, layers=10, first_shared=5) if shape == "shared_hd512" else {}
    cfg = small_cfg(**kw)
    w = model.random_weights(cfg, seed=31, **W_KW)
    prompts = [[1, 2, 3, 500, 4000, 7, 9, 11], [5, 6, 7]]
    ctx = rt.Context(0)
    plain = build(rt, ctx, cfg, w, 2, ring_kv=shape != "linear")
    want = greedy_run(plain, prompts, 40)
    m = build(rt, ctx, cfg, w, 2, ring_kv=shape != "linear")
    for s, p in enumerate(prompts):
        assert m.prefill(s, p) == want[s][0]
    parents = torch.tensor([-1, 0, 1, 2, 0, 4, 1, 3], dtype=torch.int32, device="cuda")
    rng = np.random.default_rng(5)
    done = [0, 0]  # index of the current token in want[s]
    got = [[int(want[0][0])], [int(want[1][0])]]
    while max(done) < 30:
        tok = rng.integers(0, cfg.vocab, (2, 8)).astype(np.int32)
        right = [int(rng.integers(0, 5)) for _ in range(2)]  # drafted tokens that agree
        for s in range(2):
            c = want[s][done[s]:]
            tok[s, 0] = c[0]
            for depth, node in ((1, 1), (2, 2), (3, 3), (4, 7)):
                if depth <= right[s]:
                    tok[s, node] = c[depth]
            if right[s] == 0 and rng.random() < 0.5:
                tok[s, 4] = c[1]  # the other branch agrees
                right[s] = 1
        out = m.verify_step(torch.from_numpy(tok).cuda(), parents)
        acc, nxt = out["accepted"].tolist(), out["next"].tolist()
        for s in range(2):
            c = want[s][done[s]:]
            assert acc[s] == right[s] + 1, (s, done, right, acc)
            assert nxt[s] == c[acc[s]]
            got[s] += [int(x) for x in c[1:acc[s]]] + [nxt[s]]
            done[s] += acc[s]
    ctx.check_device()
    pos = m.seq_pos.tolist()
    for s in range(2):
        assert pos[s] == len(prompts[s]) + done[s]
        assert got[s] == list(want[s][:done[s] + 1])
    # and plain decoding goes on from the compacted caches
    m.buf["next"][:2] = torch.tensor([want[s][done[s]] for s in range(2)], dtype=torch.int32, device="cuda")
    nxt = m.decode_step(batch=2).tolist()
    assert nxt == [int(want[s][done[s] + 1]) for s in range(2)]


def test_ragged_trees_and_a_captured_verify_step(rt):
    """counts: a sequence with few nodes, one that sits a step out; the step captured as a graph
    and replayed with other tokens gives the tokens of the eager one."""
    cfg = small_cfg()
    w = model.random_weights(cfg, seed=33, **W_KW)
    prompts = [[1, 2, 3], [400, 401, 402, 403, 404], [7, 7, 7, 7]]
    ctx = rt.Context(0)
    want = greedy_run(build(rt, ctx, cfg, w, 3), prompts, 24)
    m = build(rt, ctx, cfg, w, 3)
    for s, p in enumerate(prompts):
        m.prefill(s, p)
    m.buf["next"][:3] = torch.from_numpy(want[:, 0].copy()).cuda()
    parents = torch.tensor([-1, 0, 1, 2, 3], dtype=torch.int32, device="cuda")
    counts = torch.tensor([5, 2, 0], dtype=torch.int32, device="cuda")
    tok = torch.from_numpy(np.ascontiguousarray(want[:, :5])).cuda()
    out = m.verify_step(tok, parents, counts)
    assert out["accepted"].tolist() == [5, 2, 0] and m.seq_pos.tolist() == [8, 7, 4]
    assert out["next"].tolist() == [want[0][5], want[1][2], want[2][0]]
    done = [5, 2, 0]
    side = torch.cuda.Stream()
    tokens = torch.zeros((3, 5), dtype=torch.int32, device="cuda")

    def feed():
        tokens.copy_(torch.from_numpy(np.stack([want[s][done[s]:done[s] + 5] for s in range(3)])))

    feed()
    warm = m.verify_step(tokens, parents)  # sizes the workspaces
    assert warm["accepted"].tolist() == [5, 5, 5]
    done = [d + 5 for d in done]
    feed()
    torch.cuda.synchronize()
    ctx.set_stream(side)
    with torch.cuda.stream(side):
        g = torch.cuda.CUDAGraph()
        m._capturing = True
        with torch.cuda.graph(g, stream=side):
            out = m.verify_step(tokens, parents)
        m._capturing = False
        for wrong in (4, 2):
            feed()
            tokens[:, wrong] = (tokens[:, wrong] + 1) % cfg.vocab
            g.replay()
            side.synchronize()
            assert out["accepted"].tolist() == [wrong] * 3
            assert out["next"].tolist() == [want[s][done[s] + wrong] for s in range(3)]
            done = [d + wrong for d in done]
    ctx.check_device()


def test_sampled_decoding_picks_from_the_models_logits(rt, ctx):
    cfg = small_cfg()
    w = model.random_weights(cfg, seed=35, **W_KW)
    B = 3
    m = build(rt, ctx, cfg, w, B)
    for s in range(B):
        m.prefill(s, [1 + s, 2, 3])
    sm = model.Sampling(uniform=torch.zeros(B, device="cuda"), temperature=torch.tensor([1.0, 0.7, 2.0], device="cuda"),
                        top_k=torch.tensor([50, 0, 200], dtype=torch.int32, device="cuda"),
                        top_p=torch.tensor([0.9, 0.8, 1.0], device="cuda"))
    rng = np.random.default_rng(1)
    for step in range(6):
        u = rng.random(B).astype(np.float32)
        sm.uniform.copy_(torch.from_numpy(u))
        ids = m.decode_step(batch=B, sampling=sm).tolist()
        logits = m.buf["logits"][:B].clone()
        rt.call("g4_softcap", ctx.handle, logits.data_ptr(), logits.numel(), cfg.softcap)
        l = logits.cpu().numpy()
        for b in range(B):
            want, prob, near, _ = reference(l[b], u[b], [1.0, 0.7, 2.0][b], [50, 0, 200][b], [0.9, 0.8, 1.0][b])
            if near > 1e-9:
                assert ids[b] == want and abs(float(m.buf["val"][b]) - prob) < 1e-6


def test_sampled_steps_replay_and_drafts_of_the_samples_are_accepted(rt):
    """A captured sampled step with its random numbers written before each replay; then a chain that
    drafts exactly those samples is accepted whole under the same numbers."""
    cfg = small_cfg()
    w = model.random_weights(cfg, seed=36, **W_KW)
    ctx = rt.Context(0)
    m = build(rt, ctx, cfg, w, 1)
    first = m.prefill(0, [9, 8, 7, 6])
    m.buf["next"][0] = first
    sm = model.Sampling(uniform=torch.zeros(1, device="cuda"), temperature=torch.full((1,), 0.8, device="cuda"),
                        top_k=torch.full((1,), 40, dtype=torch.int32, device="cuda"))
    m.capture_decode(batch=1, sampling=sm)
    u = np.random.default_rng(8).random(6).astype(np.float32)
    toks = [first]
    for x in u:
        sm.uniform.fill_(float(x))
        torch.cuda.synchronize()
        toks.append(int(m.replay_decode()[0].item()))
        torch.cuda.synchronize()
    assert len(set(toks)) > 1
    n = 6
    d = build(rt, rt.Context(0), cfg, w, 1)
    assert d.prefill(0, [9, 8, 7, 6]) == first
    tree = model.Sampling(uniform=torch.from_numpy(u).cuda(), temperature=torch.full((n,), 0.8, device="cuda"),
                          top_k=torch.full((n,), 40, dtype=torch.int32, device="cuda"))
    out = d.verify_step(torch.tensor([toks[:n]], dtype=torch.int32, device="cuda"),
                        torch.arange(-1, n - 1, dtype=torch.int32, device="cuda"), sampling=tree)
    assert out["accepted"].tolist() == [n] and out["picks"][0].tolist() == toks[1:] and out["next"].tolist() == [toks[n]]


@pytest.mark.parametrize("ring_kv", [True, False])
def test_forked_sequences_go_on_like_their_source(rt, ctx, ring_kv):
    cfg = small_cfg()
    w = model.random_weights(cfg, seed=37, **W_KW)
    m = build(rt, ctx, cfg, w, 4, ring_kv=ring_kv)
    prompt = [int(x) for x in np.random.default_rng(3).integers(0, cfg.vocab, 40)]
    first = m.prefill(1, prompt)
    m.buf["next"][1] = first
    m.fork(1, [0, 3])
    assert m.seq_pos.tolist() == [40, 40, 0, 40] and m.buf["next"][[0, 1, 3]].tolist() == [first] * 3
    for _ in range(8):
        nxt = m.decode_step(batch=4).tolist()
        assert nxt[0] == nxt[1] == nxt[3]
    ctx.check_device()


def test_verify_refusals(rt, ctx):
    cfg = small_cfg()
    w = model.random_weights(cfg, seed=38, **W_KW)
    m = build(rt, ctx, cfg, w, 2, max_rows=10)
    t = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    for f in (lambda: m.verify_step(t(3, 2), t(2)), lambda: m.verify_step(t(2, 6), t(6)),
              lambda: m.verify_step(t(2, 4).long(), t(4)), lambda: m.verify_step(t(2, 4), t(3)),
              lambda: m.fork(0, [2]), lambda: m.fork(0, [0]), lambda: m.fork(0, [1, 1]),
              lambda: m.decode_step(batch=2, sampling=model.Sampling(uniform=torch.zeros(1, device="cuda")))):
        with pytest.raises(rt.G4Error):
            f()
