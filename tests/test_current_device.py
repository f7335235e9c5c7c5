"""The operators around the projections launch on their tensors' device, whichever is current. No GPU needed: tensors
without storage, a device and streams that are not there, and the library's entries replaced by what notes its call."""
from __future__ import annotations

import contextlib
import types

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from vllm_espalier_b200 import _lib, adapters, norms, speculative


def block_norm(dev):
    x = torch.empty(3, 64, device=dev)
    return lambda: norms.BlockNorm(64, pre=True)(x, x)


def adapt(dev):
    ad = adapters.Adapters(torch.empty(2, 1, 8, 64, dtype=torch.bfloat16, device=dev),
                           torch.empty(2, 32, 8, dtype=torch.bfloat16, device=dev), [32])
    x, y = (torch.empty(3, n, dtype=torch.bfloat16, device=dev) for n in (64, 32))
    return lambda: ad(x, y, torch.empty(3, dtype=torch.int32, device=dev))


def verify(dev):
    i, f = (lambda n: torch.empty(n, dtype=torch.int32, device=dev)), (lambda *n: torch.empty(*n, device=dev))
    return lambda: speculative.verify(f(5, 20), i(3), i(3), f(3), f(2, 20), 3)


@pytest.mark.parametrize("make", [block_norm, adapt, verify])
@pytest.mark.parametrize("current", [0, 1])
@pytest.mark.parametrize("device", [0, 1])
def test_launch_is_on_the_tensors_device(monkeypatch, make, current, device):
    at, calls = [current], []

    @contextlib.contextmanager
    def on(index):
        at.append(index)
        yield
        at.pop()

    def note(*args):
        calls.append((at[-1], args[-1]))
        return _lib.ESP_OK
    entries = types.SimpleNamespace(esp_block_norm=note, esp_adapt=note, esp_verify=note)
    for module in (norms, adapters, speculative):
        monkeypatch.setattr(module, "lib", lambda: entries)
    monkeypatch.setattr(torch.cuda, "is_available", lambda: False)      # (a GPU's would be looked for)
    monkeypatch.setattr(torch.Tensor, "data_ptr", lambda t: 4096)
    monkeypatch.setattr(torch.cuda, "device", on)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: at[-1], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 1000 + index, raising=False)
    with FakeTensorMode():
        make(torch.device("cuda", device))()
    assert calls == [(device, 1000 + device)] and at == [current]


def test_host_tensors_do_not_reach_the_library(monkeypatch):
    """ext() calls that do not look at their tensors' device themselves: the stream of a device that has none is refused."""
    calls = []
    monkeypatch.setattr(_lib, "lib", lambda: types.SimpleNamespace(esp_combine=lambda *a: calls.append(a) or _lib.ESP_OK,
                                                                   esp_down_combine=lambda *a: calls.append(a) or _lib.ESP_OK))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)
    t = torch.zeros(4, 8)
    with pytest.raises(ValueError):
        _lib._Ext.combine(t, t, t, 1, 8, 4)
    with pytest.raises(ValueError):
        _lib._Ext.down_epilogue(t, t, t, t, 1, 4, 8, 1, 4, 4)
    assert not calls
