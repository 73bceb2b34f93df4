"""Values (V) that are not finite in drafted-tree attention: a row that sees one is not finite in its
column, and no other element of the result knows of it, wherever the key lies in its tile.

The rest is compared bit for bit: columns of P V do not meet one another."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("n,H", [(3, 8), (24, 8)])
@pytest.mark.parametrize("base,window,ring", [(266, 0, 0), (400, 0, 0), (4096, 0, 0), (330, 100, 0), (330, 100, 272), (255, 256, 0)])
def test_one_column_of_the_rows_that_see_it(rt, ctx, ops, hd, n, H, base, window, ring):
    """Keys 260 (in a tile of its own sequence's end at base 266, between whole ones at base 400), one
    at the border of the windows, and the drafted node 1 of a branch; at base 255 with a window of 256
    they lie in three tiles, none of which every row sees whole."""
    S = 2
    stride = base + n
    if ring:
        cache = rt.KVCache(ctx, hd, stride, ring=ring, nseq=S)
        stride = cache.seq_rows
    else:
        cache = rt.KVCache(ctx, hd, S * stride)
    k, v = cache.storage()
    g = torch.Generator(device="cuda").manual_seed(hd + base)
    k.copy_(0.3 * torch.randn(k.shape, device="cuda", generator=g))
    v.copy_(torch.randn(v.shape, device="cuda", generator=g))
    q = (0.3 * torch.randn((S, n, H, hd), device="cuda", generator=g)).to(torch.bfloat16)
    parents = [-1] + [0] * (n - 1)
    parents[n - 1] = 1
    depth = torch.tensor([0] + [1] * (n - 2) + [2])
    pos = torch.full((S,), base, dtype=torch.int32, device="cuda")

    def run():
        return ops.attentionTree(q, cache, pos, torch.tensor(parents, dtype=torch.int32, device="cuda"),
                                 seq_stride=None if ring else stride, sliding=window > 0, window=window)

    if ring:  # rows of the mirror repeat the first slots
        for t in (k, v):
            t = t.view(S, stride, hd)
            t[:, ring:] = t[:, :stride - ring]
    clean = run()
    assert torch.isfinite(clean).all()
    bad = [(260 if base > 260 else 130, 0, float("inf")), (base - window + 1 if window else 70, hd - 1, float("nan")),
           (base + 1, hd // 2, float("-inf")), (base - 1, 5, float("nan"))]
    for key, col, val in bad:
        for s in range(S):
            slots = [key % ring, ring + key % ring] if ring else [key]
            for slot in slots:
                if not ring or slot < stride:
                    v[s * stride + slot, col] = val
    got = run()
    hit = torch.zeros((n, hd), dtype=torch.bool)
    for key, col, _ in bad:
        for i in range(n):
            if key < base:
                hit[i, col] |= not window or key > base + int(depth[i]) - window
            else:
                hit[i, col] |= i in (1, n - 1)
    hit = hit[None, :, None].expand(S, n, H, hd).cuda()
    assert not torch.isfinite(got[hit]).any()
    assert torch.equal(got[~hit], clean[~hit])
    ctx.check_device()


def test_a_column_of_values_that_are_all_infinite(rt, ctx, ops):
    hd, n, H, base = 256, 20, 8, 200
    cache = rt.KVCache(ctx, hd, base + n)
    k, v = cache.storage()
    k.copy_(0.1 * torch.randn(k.shape, device="cuda"))
    v.copy_(torch.randn(v.shape, device="cuda"))
    q = torch.randn((1, n, H, hd), device="cuda").to(torch.bfloat16)
    pos = torch.tensor([base], dtype=torch.int32, device="cuda")
    chain = torch.arange(-1, n - 1, dtype=torch.int32, device="cuda")
    clean = ops.attentionTree(q, cache, pos, chain)
    v[:, 33] = float("inf")
    got = ops.attentionTree(q, cache, pos, chain)
    assert not torch.isfinite(got[..., 33]).any()
    keep = torch.arange(hd, device="cuda") != 33
    assert torch.equal(got[..., keep], clean[..., keep])
    ctx.check_device()
