"""Library objects that outlive the context they were made with (garbage collection destroys them in
any order): their destruction reads nothing of it and leaves no error for the next call."""
import importlib

import numpy as np
import pytest
import torch

from test_drafted_model_gpu import W_KW, small_cfg

pytestmark = pytest.mark.gpu
model = importlib.import_module("gemma4-js_b200.model")


def test_a_context_destroyed_before_its_objects(rt):
    cfg = small_cfg()
    w = model.random_weights(cfg, seed=45, **W_KW)
    want = None
    for _ in range(4):
        ctx = rt.Context(0)
        m = model.Gemma4Model(ctx, cfg, w, max_batch=1, max_seq=64, max_rows=16, persistent=True)
        first = m.prefill(0, [1, 2, 3])
        assert m.decoder() is not None and want in (None, first)
        want = first
        ctx.sync()
        ctx.close()
        blocks = [np.full(64, 0x5A5A5A5A, np.int32) for _ in range(64)]  # the context's memory is used again
        m._dec.close()
        for Ly in m.layers:
            Ly["kv"].close()
            for name in ("qkv", "o", "gu", "down", "pg", "pp"):
                Ly[name].close()
        m.top.close(), m.head.close(), m.ple.close()
        del m, blocks
        assert torch.cuda.current_device() == 0
        torch.zeros(4, device="cuda").sum().item()
