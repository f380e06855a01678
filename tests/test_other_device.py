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
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 1000 + index, raising=False)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(mb, "_same_device", lambda what, *tensors: torch.device("cuda", 1))
    monkeypatch.setattr(mb, "_device_of", lambda t: torch.device("cuda", 1), raising=False)
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


def test_the_layers_calls_run_on_their_tensors_device(two_devices, monkeypatch):
    """Every call with its tensors' device current and on that device's current stream."""
    seen = []

    class Lib:
        def __getattr__(self, name):
            def call(*args):
                if name.endswith("_bytes"):
                    return 256
                seen.append((name[9:], two_devices["current"], args[-1] == 1001))
                return mb.OK
            return call

    monkeypatch.setattr(mb, "lib", Lib)
    x, a, w = torch.zeros((4, 16)).half(), torch.zeros((4, 1), dtype=torch.int32), torch.ones((4, 1))
    seg = torch.tensor([0, 4], dtype=torch.int32)
    up, gate_up = torch.zeros((1, 16, 16)).half(), torch.zeros((1, 32, 16)).half()
    bufs = mb.allocate_buffers(mb.MoEParams(4, 1, 2, 16), device="cpu")
    mb.B200Scatter().run(x, a, w, bufs, mb.MoEParams(4, 1, 2, 16))
    p = mb.pack(x, a, w, 2, workspace=mb.Workspace(4, 1, 2, device="cpu"))
    mb.unpermute(x, w, a, 4, 1)
    mb.grouped_swiglu(x, seg, gate_up, up)
    mb.grouped_swiglu(x, seg, gate_up, up, row_token=p.perm)
    mb.grouped_ffn(x, seg, up, up)
    mb.ffn_weights_from_reference(up, up)
    mb.route(x, mb.RouterWeights(torch.zeros((16, 2)), torch.float16), 1)
    mb.ep_layout(torch.zeros((1, 2), dtype=torch.int32), 0, [0, 2])
    assert [s[0] for s in seen] == ["workspace_init", "pack", "workspace_init", "pack", "unpermute", "grouped_swiglu",
                                    "grouped_swiglu_gather", "grouped_ffn", "ffn_weights_from_reference", "router_prepare", "route",
                                    "ep_layout"]
    assert all(current == 1 and on_its_stream for _, current, on_its_stream in seen), seen
    assert two_devices["current"] == 0


def test_tensors_that_are_on_no_gpu_are_refused():
    x, a, w = torch.zeros((4, 16)).half(), torch.zeros((4, 1), dtype=torch.int32), torch.ones((4, 1))
    for f in (lambda: mb.unpermute(x, w, a, 4, 1), lambda: mb.Workspace(4, 1, 2, device="cpu"),
              lambda: mb.grouped_ffn(x, a[:2, 0], torch.zeros((1, 16, 16)).half(), torch.zeros((1, 16, 16)).half())):
        with pytest.raises(mb.MoEB200Error) as e:
            f()
        assert e.value.status == mb.ERR_INVALID_ARG
