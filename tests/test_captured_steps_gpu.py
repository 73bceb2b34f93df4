"""Captured steps replayed after other calls of the same model."""
import importlib

import numpy as np
import pytest
import torch

from test_drafted_model_gpu import W_KW, build, greedy_run, small_cfg

pytestmark = pytest.mark.gpu
model = importlib.import_module("gemma4-js_b200.model")


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
