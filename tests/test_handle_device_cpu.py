"""The binding's handle takes its device from the library, whatever torch is imported (or is not): a stand-in for the
library answers here, so that no GPU is needed."""
from __future__ import annotations

import ctypes
import sys
import types

import pytest
import torch

import emugemm

INVALID_HANDLE, INVALID_POINTER = 1, 3


class StandIn:
    """Every call succeeds; handles are on device 3."""

    def emugemm_get_device(self, handle, device):
        device._obj.value = 3
        return 0

    def __getattr__(self, name):
        return lambda *args: 0


@pytest.fixture()
def library(monkeypatch):
    lib = StandIn()
    monkeypatch.setattr(emugemm, "_lib", lib)


def test_handle_beside_a_torch_without_cuda(library, monkeypatch):
    def no_cuda():
        raise AssertionError("Torch not compiled with CUDA enabled")

    monkeypatch.setitem(sys.modules, "torch", types.SimpleNamespace(cuda=types.SimpleNamespace(current_device=no_cuda)))
    with emugemm.Handle() as h:
        assert h.device == 3


def test_handle_made_before_torch_refuses_host_tensors(library, monkeypatch):
    monkeypatch.delitem(sys.modules, "torch")
    with emugemm.Handle() as h:
        with pytest.raises(ValueError):
            h._at(torch.zeros(4))
        with pytest.raises(ValueError):
            h.q4_unpack(1, 1, 1, 32, 4096, torch.zeros(4), 1)


def test_get_device_refusals():
    lib = emugemm.lib()
    d = ctypes.c_int(-1)
    assert lib.emugemm_get_device(None, ctypes.byref(d)) == INVALID_HANDLE
    assert lib.emugemm_get_device(ctypes.create_string_buffer(1 << 16), None) == INVALID_POINTER
    assert d.value == -1
