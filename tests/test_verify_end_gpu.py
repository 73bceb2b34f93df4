"""Verify steps of sequences near the end of their cache: the tree's nodes that fit are verified as
decode steps would, a full sequence sits the step out, and the other sequences do not notice."""
import importlib

import numpy as np
import pytest
import torch

from test_drafted_model_gpu import W_KW, small_cfg

pytestmark = pytest.mark.gpu
model = importlib.import_module("gemma4-js_b200.model")
MAX_SEQ = 200  # above ring + mirror: sliding layers have ring caches if they are asked for


def started(rt, cfg, w, prompts, ring_kv):
    ctx = rt.Context(0)
    m = model.Gemma4Model(ctx, cfg, w, max_batch=len(prompts), max_seq=MAX_SEQ, max_rows=40, ring_kv=ring_kv)
    assert any(Ly["kv"].ring for Ly in m.layers) == ring_kv
    for s, p in enumerate(prompts):
        for i in range(0, len(p), 40):
            m.buf["next"][s] = m.prefill(s, p[i:i + 40])
    return m


@pytest.mark.parametrize("ring_kv", [True, False])
@pytest.mark.parametrize("counted", [False, True])
def test_the_end_of_the_cache(rt, ring_kv, counted):
    n = 4  # (16 rows a step: the linears of plain decode steps, row for row the same bits)
    cfg = small_cfg()
    w = model.random_weights(cfg, seed=41, **W_KW)
    rng = np.random.default_rng(7)
    # one place short of the tree, the last place, none, and a sequence far from its end
    prompts = [[int(x) for x in rng.integers(0, cfg.vocab, MAX_SEQ - free)] for free in (n - 1, 1, 0, 100)]
    B = len(prompts)
    want = []
    for p in (prompts[0], prompts[1], prompts[3]):  # greedy steps while the cache has a place
        plain = started(rt, cfg, w, [p], ring_kv)
        toks = [int(plain.buf["next"][0])]
        for _ in range(min(n, MAX_SEQ - len(p))):
            toks.append(int(plain.decode_step(batch=1)[0]))
        assert plain.ctx.check_device() == 0
        want.append(toks)
    m = started(rt, cfg, w, prompts, ring_kv)
    last = int(m.buf["next"][2])
    tok = np.zeros((B, n), np.int32)
    for s, toks in zip((0, 1, 3), want):
        tok[s, :len(toks[:n])] = toks[:n]
    counts = torch.full((B,), n, dtype=torch.int32, device="cuda") if counted else None
    out = m.verify_step(torch.from_numpy(tok).cuda(), torch.arange(-1, n - 1, dtype=torch.int32, device="cuda"), counts)
    assert m.ctx.check_device() == 0
    assert out["accepted"].tolist() == [n - 1, 1, 0, n]
    assert m.seq_pos.tolist() == [MAX_SEQ] * 3 + [MAX_SEQ - 100 + n]
    assert out["next"].tolist() == [want[0][n - 1], want[1][1], last, want[2][n]]
    assert out["path"].tolist() == [[0, 1, 2, -1], [0, -1, -1, -1], [-1] * 4, [0, 1, 2, 3]]
    # all but the last sequence are full now: they sit the next step out, and it goes on
    nxt = out["next"].tolist()
    again = m.verify_step(m.buf["next"][:B].clone().view(B, 1), torch.full((1,), -1, dtype=torch.int32, device="cuda"))
    assert again["accepted"].tolist() == [0, 0, 0, 1] and again["next"].tolist()[:3] == nxt[:3]
    assert m.ctx.check_device() == 0


def test_counts_outside_the_tree_still_raise(rt):
    cfg = small_cfg()
    w = model.random_weights(cfg, seed=42, **W_KW)
    m = started(rt, cfg, w, [[1, 2, 3], [4, 5]], False)
    tok = torch.ones((2, 3), dtype=torch.int32, device="cuda")
    for bad in ([4, 1], [1, -1]):
        m.verify_step(tok, torch.arange(-1, 2, dtype=torch.int32, device="cuda"),
                      torch.tensor(bad, dtype=torch.int32, device="cuda"))
        with pytest.raises(rt.G4Error):
            m.ctx.check_device()
