"""Precision of drafted-tree attention: softmax weights to the accuracy of g4_attention_rows, in
every head dimension and every split of the work.

A weight goes to the tensor cores as a bf16 head and a bf16 tail: the head is off by at most 2^-8 of
the weight, what is left is exact in 32 bits, and its own rounding takes 2^-8 of that, 2^-16 of the
weight.  The f32 sums over up to some thousand keys (truncated once per 16 keys and part) take
another 2^-16, a score summed in f32 2^-20 of sum |q k|, as a factor of the weights and of their sum.
The result is rounded to bf16 once (2^-8)."""
import ctypes as C
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
L = importlib.import_module("gemma4-js_b200._lib")


def reference(q, k, v, base, parents, window=0):
    """q [n, H, hd], k, v [rows, hd] in f64: the result and what it may be off by, per element."""
    n = q.shape[0]
    depth, see = [], torch.zeros((n, k.shape[0]), dtype=torch.bool, device=q.device)
    for i, p in enumerate(parents):
        depth.append(0 if p < 0 else depth[p] + 1)
        see[i, max(0, base + depth[i] - window + 1) if window else 0:base] = True
        a = i
        while a >= 0:
            see[i, base + a] = not window or depth[i] - depth[a] < window
            a = parents[a]
    s = torch.einsum("nhd,kd->nhk", q, k).masked_fill(~see[:, None], -float("inf"))
    ds = 2.0**-20 * torch.einsum("nhd,kd->nhk", q.abs(), k.abs()).amax(2, keepdim=True)
    w = torch.softmax(s, 2)
    out, size = w @ v, w @ v.abs()
    return out, 2.0**-8 * out.abs() + (2.0**-15 + 2 * ds) * size + 1e-30


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("n,H", [(1, 8), (5, 3), (16, 8), (40, 8), (64, 7)])
@pytest.mark.parametrize("context,window", [(3, 0), (300, 0), (300, 64), (4100, 0)])
def test_weights_to_sixteen_bits(rt, ctx, ops, hd, n, H, context, window):
    S, stride = 2, context + n
    g = torch.Generator(device="cuda").manual_seed(hd + n + context)
    cache = rt.KVCache(ctx, hd, S * stride)
    k, v = cache.storage()
    k.copy_(0.3 * torch.randn(k.shape, device="cuda", generator=g))
    v.copy_(torch.randn(v.shape, device="cuda", generator=g))
    q = (0.3 * torch.randn((S, n, H, hd), device="cuda", generator=g)).to(torch.bfloat16)
    parents = [-1] + [i // 2 for i in range(n - 1)]
    pos = torch.tensor([context, context // 2], dtype=torch.int32, device="cuda")
    out = ops.attentionTree(q, cache, pos, torch.tensor(parents, dtype=torch.int32, device="cuda"), seq_stride=stride,
                            sliding=window > 0, window=window)
    for s, base in enumerate(pos.tolist()):
        rows = slice(s * stride, s * stride + base + n)
        ref, tol = reference(q[s].double(), k[rows].double(), v[rows].double(), base, parents, window)
        err = (out[s].double() - ref).abs()
        assert (err <= tol).all(), (s, float((err / tol).max()))
    ctx.check_device()


@pytest.mark.parametrize("n", [4, 24])
def test_a_chain_is_attention_rows_to_two_roundings(rt, ctx, ops, n):
    """Both operators round the same value to bf16 once."""
    S, H, hd, stride = 3, 8, 256, 800
    g = torch.Generator(device="cuda").manual_seed(n)
    cache = rt.KVCache(ctx, hd, S * stride)
    k, v = cache.storage()
    k.copy_(0.3 * torch.randn(k.shape, device="cuda", generator=g))
    v.copy_(torch.randn(v.shape, device="cuda", generator=g))
    q = (0.3 * torch.randn((S, n, H, hd), device="cuda", generator=g)).to(torch.bfloat16)
    pos = torch.tensor([700, 13, 512], dtype=torch.int32, device="cuda")
    chain = torch.arange(-1, n - 1, dtype=torch.int32, device="cuda")
    a, b = ops.attentionTree(q, cache, pos, chain, seq_stride=stride), torch.empty_like(q)
    rmap = L.G4Rows(pos.data_ptr(), 0, n, 0, 0)
    rt.call("g4_attention_rows", ctx.handle, q.data_ptr(), cache.handle, S * n, H, hd, C.byref(rmap), stride, 0, 0,
            b.data_ptr())
    for s, base in enumerate(pos.tolist()):
        rows = slice(s * stride, s * stride + base + n)
        _, tol = reference(q[s].double(), k[rows].double(), v[rows].double(), base, chain.tolist())
        assert ((a[s].double() - b[s].double()).abs() <= 2 * tol).all()
