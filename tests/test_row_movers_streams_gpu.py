"""Operators on a context stream that is not torch's current one keep their inputs from reuse until
that stream is done with them, also where the caller gives the output or there is none."""
import pytest
import torch

pytestmark = pytest.mark.gpu

SLEEP = 400_000_000  # clocks: some 0.2 s, during which a block freed too early would be handed out again


@pytest.fixture
def side(rt):
    ctx = rt.Context(0)
    ctx.set_stream(torch.cuda.Stream())
    return ctx


def reused(ctx, make, call):
    """Whether the memory of an input that the caller drops right after the call is handed out while
    the call still waits on the context's stream."""
    call(make())  # the first call of a kernel loads it, which may wait for the device
    torch.cuda.synchronize()
    t = make()
    torch.cuda.synchronize()
    with torch.cuda.stream(ctx._stream):
        torch.cuda._sleep(SLEEP)
    call(t)
    ptr, like = t.data_ptr(), (t.shape, t.dtype)
    del t
    again = torch.empty(like[0], dtype=like[1], device="cuda")
    busy = not ctx._stream.query()
    torch.cuda.synchronize()
    assert busy, "the stream was done before the memory was asked for"
    return again.data_ptr() == ptr


def test_attention_tree_with_an_output(rt, side):
    ops = rt.GPUOps(side)
    hd, n, H, S = 128, 4, 8, 3
    cache = rt.KVCache(side, hd, S * 64)
    cache.storage()[0].zero_(), cache.storage()[1].zero_()
    q = torch.zeros((S, n, H, hd), dtype=torch.bfloat16, device="cuda")
    pos = torch.full((S,), 9, dtype=torch.int32, device="cuda")
    chain = torch.arange(-1, n - 1, dtype=torch.int32, device="cuda")
    cnt = torch.full((S,), n, dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)
    args = {"q": q, "seq_pos": pos, "parents": chain, "counts": cnt, "out": out}
    for name, t in args.items():
        def call(x, name=name):
            ops.attentionTree(cache=cache, seq_stride=64, **{**args, name: x})
        assert not reused(side, t.clone, call), name
    side.check_device()


@pytest.mark.parametrize("name", ["path", "accepted", "seq_pos"])
def test_kv_compact(rt, side, name):
    caches = [rt.KVCache(side, 64, 3 * 32)]
    args = {"path": torch.tensor([[0, 1, 2, -1]] * 3, dtype=torch.int32, device="cuda"),
            "accepted": torch.tensor([3, 2, 1], dtype=torch.int32, device="cuda"),
            "seq_pos": torch.tensor([5, 6, 7], dtype=torch.int32, device="cuda")}
    assert not reused(side, args[name].clone, lambda x: rt.kv_compact(side, caches, seq_stride=32, **{**args, name: x}))
    side.check_device()


def test_kv_fork(rt, side):
    caches = [rt.KVCache(side, 64, 3 * 32)]
    make = lambda: torch.tensor([5, 6, 7], dtype=torch.int32, device="cuda")  # noqa: E731
    assert not reused(side, make, lambda x: rt.kv_fork(side, caches, x, [0], [2], seq_stride=32))
    side.check_device()
