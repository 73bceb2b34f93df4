"""Rows with one rank to keep (g4_sample: temperature not above 0, top-k 1, top-p 0) whose highest
logit is shared by many: the lowest index with probability 1, whatever other settings the call has.

Whole numbers and exact quotients: no tolerance.  The outputs hold sentinels before the call."""
import ctypes as C
import importlib

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
L = importlib.import_module("gemma4-js_b200._lib")


def tied_rows(V):
    l = np.zeros((7, V), np.float32)         # 0: an idle slot of zeros
    l[1] = 1.0e4 + np.arange(V) % 97         # under a cap all the same
    l[2, : V // 2] = -1.0                    # the later half
    l[3, ::3] = -2.5                         # two of three
    l[4] = -0.0
    l[4, 5::7] = 0.0                         # -0 and +0 are equal
    l[5, : V - 1] = -np.inf                  # one logit, the last
    l[6, :17] = np.nan
    l[6, V // 2:] = np.inf
    return l


def run(ctx, x, how, cap):
    R, V = x.shape
    ids = torch.full((R,), -77, dtype=torch.int32, device="cuda")
    probs = torch.full((R,), -77.0, device="cuda")
    L.call("g4_sample", ctx.handle, x.data_ptr(), x.stride(0), R, V, cap, C.byref(how), ids.data_ptr(), probs.data_ptr())
    return ids.tolist(), probs.tolist()


@pytest.mark.parametrize("V", [1, 2049, 8193, 9001, 50257, 262144])
@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("how", ["t0", "t_negative", "t_nan", "k1", "p0", "k1_p_mp", "t0_p"])
def test_the_lowest_index_of_the_highest_logit(ctx, V, cap, how):
    l = tied_rows(V)
    R = len(l)
    full = lambda v, t=torch.float32: torch.full((R,), v, dtype=t, device="cuda")  # noqa: E731
    u = full(0.9)
    kept = {"t0": {"temperature": full(0.0)}, "t_negative": {"temperature": full(-1.0)},
            "t_nan": {"temperature": full(float("nan"))}, "k1": {"top_k": full(1, torch.int32)}, "p0": {"top_p": full(0.0)},
            "k1_p_mp": {"top_k": full(1, torch.int32), "top_p": full(0.9), "min_p": full(0.1)},
            "t0_p": {"temperature": full(0.0), "top_p": full(0.5)}}[how]
    s = L.G4Sampling(*[kept[n].data_ptr() if n in kept else None for n in ("temperature", "top_k", "top_p", "min_p")],
                     u.data_ptr())
    x = torch.from_numpy(l).cuda()
    capped = x.clone()
    if cap:
        L.call("g4_softcap", ctx.handle, capped.data_ptr(), capped.numel(), C.c_float(cap))
        capped[torch.isneginf(x)] = -np.inf  # a mask stays one
    c = capped.cpu().numpy()
    c = np.where(np.isnan(c), -np.inf, c)
    want = [int(np.argmax(row)) if (row > -np.inf).any() else -1 for row in c]  # the first of equal ones
    for view in (x, torch.nn.functional.pad(x, (1, 2))[:, 1:1 + V]):  # rows on 16 bytes and off them
        ids, probs = run(ctx, view, s, cap)
        assert ids == want
        assert probs == [0.0 if w < 0 else 1.0 for w in want]
    ctx.check_device()


def test_greedy_rows_beside_sampled_ones(ctx, ops):
    """Idle slots of zeros at temperature 0 among rows at other temperatures: the others are as without."""
    V, R = 32768, 40
    g = torch.Generator(device="cuda").manual_seed(3)
    x = 2.0 * torch.randn((R, V), device="cuda", generator=g)
    u, t = torch.rand(R, device="cuda", generator=g), 0.5 + torch.rand(R, device="cuda", generator=g)
    alone = ops.sample(x, u, temperature=t)
    x[::4], t[::4] = 0.0, 0.0
    ids, probs = ops.sample(x, u, temperature=t)
    idle = torch.arange(R, device="cuda") % 4 == 0
    assert (ids[idle] == 0).all() and (probs[idle] == 1).all()
    assert torch.equal(ids[~idle], alone[0][~idle]) and torch.equal(probs[~idle], alone[1][~idle])
