"""What a captured step points at outlives the capture: buffers that a later, larger step outgrows,
and the settings' tensors.  Host logic only."""
import gc
import importlib
import weakref

import torch

model = importlib.import_module("gemma4-js_b200.model")


def bare():
    m = object.__new__(model.Gemma4Model)
    m.buf, m.dev, m._outgrown = {}, torch.device("cpu"), []
    return m


def test_outgrown_tree_buffers_are_kept():
    m = bare()
    first = m._tree_buffer("logits", 8, torch.float32)
    kept = weakref.ref(first)
    del first
    assert m._tree_buffer("logits", 5, torch.float32) is kept()  # large enough: the same one
    second = m._tree_buffer("logits", 9, torch.float32)
    gc.collect()
    assert kept() is not None and second is not kept() and second.numel() >= 9


def test_outgrown_buffers_take_no_more_than_the_one_in_use():
    m = bare()
    for n in range(1, 300):
        assert m._tree_buffer("vals", n, torch.float32).numel() >= n
    assert sum(t.numel() for t in m._outgrown) <= m._tree_buffer("vals", 1, torch.float32).numel()
