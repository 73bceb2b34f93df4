"""Checks of the settings' tensors (model.Sampling) without a GPU."""
import importlib

import pytest
import torch

model = importlib.import_module("gemma4-js_b200.model")
rt = importlib.import_module("gemma4-js_b200.runtime")


class Tensor:
    """Enough of a device tensor for the checks."""

    def __init__(self, device, dtype=torch.float32, n=4):
        self.device, self.dtype, self.n, self.is_cuda = torch.device(device), dtype, n, True

    def is_contiguous(self):
        return True

    def numel(self):
        return self.n

    def data_ptr(self):
        return 4096


def test_settings_of_another_gpu_are_refused():
    here = torch.device("cuda", 0)
    s = model.Sampling(uniform=Tensor("cuda:0"), temperature=Tensor("cuda:0"), top_k=Tensor("cuda:0", torch.int32))
    assert s.struct(4, here).uniform == 4096 and s.struct(4).temperature == 4096
    for name in ("uniform", "temperature", "top_k", "top_p", "min_p"):
        bad = model.Sampling(uniform=Tensor("cuda:0"))
        setattr(bad, name, Tensor("cuda:1", torch.int32 if name == "top_k" else torch.float32))
        with pytest.raises(rt.G4Error, match=name):
            bad.struct(4, here)
        if name != "uniform":
            with pytest.raises(rt.G4Error, match=name):
                bad.struct(4)
    for bad in (Tensor("cuda:0", n=3), Tensor("cuda:0", torch.float64), torch.zeros(4)):
        with pytest.raises(rt.G4Error, match="uniform"):
            model.Sampling(uniform=bad).struct(4, here)
        with pytest.raises(rt.G4Error, match="uniform"):
            model.Sampling(uniform=bad).struct(4)
