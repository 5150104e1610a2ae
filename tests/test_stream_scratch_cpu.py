"""Clearing the device error drops the streams' scratch, whose counters a launch that
gave up may have left set (host bookkeeping, no GPU needed)."""
import torch

from kernels import _lib


def test_clear_device_error_drops_the_devices_scratch(monkeypatch):
    held = {(0, 11): "a", (0, 12): "b", (1, 11): "c"}
    monkeypatch.setattr(_lib, "_STREAM_SCRATCH", held)
    monkeypatch.setattr(_lib, "_WORKSPACES", {})
    _lib.clear_device_error(torch.device("cuda", 0))
    assert held == {(1, 11): "c"}


def test_clear_device_error_makes_the_binding_forget(monkeypatch):
    class Native:
        calls = 0

        def forget(self):
            self.calls += 1

    native = Native()
    monkeypatch.setattr(_lib, "_STREAM_SCRATCH", {(0, 11): "a"})
    monkeypatch.setattr(_lib, "_WORKSPACES", {})
    monkeypatch.setattr(_lib, "_binding", native)
    _lib.clear_device_error(torch.device("cuda", 0))
    assert native.calls == 1
