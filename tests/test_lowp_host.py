"""The host side of the low-precision operators, without a GPU: what reaches an entry point."""

import importlib
import os
import subprocess
import sys
import warnings

import pytest
import torch

import int_crush_converter_b200 as B
from int_crush_converter_b200 import _native as nat
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


def test_the_library_builds_without_torch():
    """Without torch (or its headers) the C library is all there is to build."""
    csrc = os.path.join(os.path.dirname(B.__file__), "csrc")
    r = subprocess.run(["make", "-n", "-B", "-C", csrc, "PYTHON=false"], capture_output=True, text=True)
    assert r.returncode == 0 and "lowp_gemm.cu" in r.stdout and "binding.cpp" not in r.stdout
    r = subprocess.run(["make", "-n", "-B", "-C", csrc, f"PYTHON={sys.executable}"], capture_output=True, text=True)
    assert r.returncode == 0 and "binding.cpp" in r.stdout


def test_without_the_binding_calls_go_the_long_way(monkeypatch):
    """Said once, and the same checks and calls follow."""
    calls = []
    monkeypatch.setattr(nat, "_fast", None)
    monkeypatch.delattr(B, "_binding", raising=False)
    monkeypatch.setitem(sys.modules, B.__name__ + "._binding", None)
    monkeypatch.setattr(rmsnorm, "device_of", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(rmsnorm, "call", lambda name, dev, *args: calls.append(name))
    with pytest.warns(RuntimeWarning, match="make -C"):
        B.rmsnorm_quantize(torch.zeros(2, 64), torch.ones(64))
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        B.rmsnorm_quantize(torch.zeros(2, 64), torch.ones(64))
    assert calls == ["ic_rmsnorm_quantize"] * 2
    with pytest.raises(ValueError, match="eps"):
        B.rmsnorm_quantize(torch.zeros(2, 64), torch.ones(64), eps=-1.0)


def test_a_binding_that_does_not_load_is_an_error(monkeypatch):
    """One of another torch, for instance."""
    def load(name, package=None):
        raise ImportError("undefined symbol")
    monkeypatch.setattr(nat, "_fast", None)
    monkeypatch.setattr(importlib, "import_module", load)
    with pytest.raises(ImportError, match="undefined symbol.*make -C"):
        nat.binding()


@pytest.mark.parametrize("fmt,blocks", [("mxfp4", 10), ("nvfp4", 20)])
def test_block_scales_of_flat_scale_bytes(fmt, blocks):
    """Scale bytes are taken in any shape; row by row they are the same."""
    want = torch.randint(0, 100, (130, blocks), dtype=torch.uint8)
    q = B.FP4Tensor.from_block_scales(torch.zeros(130, 160, dtype=torch.uint8), want, None if fmt == "mxfp4" else torch.ones(130), fmt)
    q.scales = q.scales.reshape(-1)
    q.check("test")
    assert torch.equal(q.block_scales(), want)
