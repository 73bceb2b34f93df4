"""Captured steps replayed after other calls of the same model, and after the caller dropped what it
captured them with."""
import gc
import importlib
import weakref

import numpy as np
import pytest
import torch

from test_drafted_model_gpu import W_KW, build, greedy_run, small_cfg

pytestmark = pytest.mark.gpu
model = importlib.import_module("gemma4-js_b200.model")


def test_a_captured_sampled_step_keeps_its_settings(rt):
    cfg = small_cfg()
    w = model.random_weights(cfg, seed=43, **W_KW)
    B, steps = 2, 5
    u = torch.rand((steps, B), generator=torch.Generator().manual_seed(1))

    def run(drop):
        m = build(rt, rt.Context(0), cfg, w, B)
        for s in range(B):
            m.buf["next"][s] = m.prefill(s, [3 + s, 2, 1])
        uniform = torch.zeros(B, device="cuda")
        sm = model.Sampling(uniform=uniform, temperature=torch.full((B,), 0.7, device="cuda"),
                            top_k=torch.full((B,), 60, dtype=torch.int32, device="cuda"))
        m.capture_decode(batch=B, sampling=sm)
        kept = [weakref.ref(sm.temperature), weakref.ref(sm.top_k)]
        g = m.graph
        if drop:  # the caller keeps graph and random numbers, lets go of the rest, and memory is used again
            sm.temperature = sm.top_k = None
            del sm
            m.capture_decode(batch=1)  # another graph of the model takes the first one's place in it
            gc.collect()
            assert all(r() is not None for r in kept)
            junk = [torch.full((64,), 1e9, device="cuda") for _ in range(200)]  # noqa: F841
        out = []
        for i in range(steps):
            uniform.copy_(u[i])
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            out.append(m.buf["next"][:B].tolist())
        m.ctx.check_device()
        return out

    assert run(True) == run(False)


def test_a_captured_verify_step_survives_a_larger_one(rt):
    """Captured with two nodes a sequence; then a step of eight, whose buffers replace the captured ones,
    and memory handed out again; the replay still verifies, and leaves that memory alone."""
    cfg = small_cfg()
    w = model.random_weights(cfg, seed=44, **W_KW)
    prompts = [[1, 2, 3], [9, 8]]
    want = greedy_run(build(rt, rt.Context(0), cfg, w, 2), prompts, 20)
    ctx = rt.Context(0)
    m = build(rt, ctx, cfg, w, 2)
    for s, p in enumerate(prompts):
        m.prefill(s, p)
    chain = lambda n: torch.arange(-1, n - 1, dtype=torch.int32, device="cuda")  # noqa: E731
    done, two = 0, chain(2)
    tokens = torch.from_numpy(np.ascontiguousarray(want[:, :2])).cuda()
    m.verify_step(tokens, two)
    done += 2
    torch.cuda.synchronize()
    home, side = ctx.stream, torch.cuda.Stream()
    ctx.set_stream(side)
    with torch.cuda.stream(side):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = m.verify_step(tokens, two)
    ctx.set_stream(home)
    torch.cuda.synchronize()
    big = m.verify_step(torch.from_numpy(np.ascontiguousarray(want[:, done:done + 8])).cuda(), chain(8))
    assert big["accepted"].tolist() == [8, 8]
    done += 8
    junk = [torch.full((n,), 7.0, device="cuda") for n in [2 * 2 * cfg.vocab, 4, 64] * 50]
    for _ in range(2):
        tokens.copy_(torch.from_numpy(np.ascontiguousarray(want[:, done:done + 2])))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert out["accepted"].tolist() == [2, 2] and out["next"].tolist() == want[:, done + 2].tolist()
        done += 2
    assert all(bool((t == 7.0).all()) for t in junk)
    ctx.check_device()
