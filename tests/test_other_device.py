"""Calls whose tensors lie on another device than the current one, on devices
made up for the test (no GPU): what depends on the device is asked of the
tensors'."""
import contextlib

import pytest
import torch

import moe_b200 as mb


@pytest.fixture
def two_devices(monkeypatch):
    """Tensors count as lying on device 1; device 0 is current.  state["current"] is the current device."""
    state = {"current": 0}

    @contextlib.contextmanager
    def device(dev):
        before, state["current"] = state["current"], dev.index
        try:
            yield
        finally:
            state["current"] = before

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: state["current"], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(mb, "_same_device", lambda what, *tensors: torch.device("cuda", 1))
    return state


def test_norm_gradients_ask_their_tensors_device_for_the_workspace(two_devices, monkeypatch):
    """Device 1 has more SMs than the current one and needs more workspace."""
    calls = []

    class Lib:
        @staticmethod
        def moe_b200_block_norm_backward_workspace_bytes(T, d):
            return (1024, 4096)[two_devices["current"]]

        @staticmethod
        def moe_b200_block_norm_backward(*args):
            nbytes = args[-2]
            calls.append((two_devices["current"], nbytes))
            return mb.OK if nbytes >= (1024, 4096)[two_devices["current"]] else mb.ERR_WORKSPACE

        @staticmethod
        def moe_b200_last_error():
            return b"workspace too small"

    monkeypatch.setattr(mb, "lib", lambda: Lib)
    x, w = torch.zeros((4, 16)).bfloat16(), torch.ones((16,)).bfloat16()
    mb.block_norm_backward(x, x, x, x, w_post=w, w_pre=w)
    assert calls == [(1, 4096)] and two_devices["current"] == 0
