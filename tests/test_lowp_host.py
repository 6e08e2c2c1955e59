"""The host side of the low-precision operators, without a GPU: what reaches an entry point."""

import pytest
import torch

import int_crush_converter_b200 as B
from int_crush_converter_b200 import rmsnorm


class Elsewhere(torch.Tensor):
    """Stands in for a tensor of another GPU: `to` gives the copy that a kernel may read."""

    is_cuda = True
    copy = None

    def to(self, device):
        Elsewhere.copy = torch.Tensor.to(self.as_subclass(torch.Tensor), device, copy=True)
        return Elsewhere.copy


@pytest.mark.parametrize("fmt", ["int8", "mxfp4", "nvfp4"])
def test_rmsnorm_reads_the_weight_on_its_own_device(monkeypatch, fmt):
    """Whatever device the weight is on, the kernel is given one on the device that it runs on."""
    calls = []
    monkeypatch.setattr(rmsnorm, "device_of", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(rmsnorm, "call", lambda name, dev, *args: calls.append(args))
    weight = torch.ones(64).as_subclass(Elsewhere)
    B.rmsnorm_quantize(torch.zeros(2, 64), weight, fmt=fmt)
    assert calls[0][7] == Elsewhere.copy.data_ptr() != weight.data_ptr()
