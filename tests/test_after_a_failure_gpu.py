"""A call that failed with a CUDA error does not fail the calls behind it."""
import ctypes

import pytest
import torch

import moe_b200 as mb

pytestmark = pytest.mark.gpu


def fail_once():
    """A receive buffer of 10^15 bytes: the allocation is refused."""
    first, ctx = (ctypes.c_int32 * 2)(0, 64), ctypes.c_void_p()
    status = mb.lib().moe_b200_ep_create(1, 0, 64, 32, 8192, 2 ** 31 - 1, first, 1000, ctypes.byref(ctx))
    assert status == mb.ERR_CUDA and not ctx.value
    assert b"out of memory" in mb.lib().moe_b200_last_error()


@pytest.mark.parametrize("op", ["norm", "norm_backward", "w4", "grouped_mm", "pack", "unpermute"])
def test_next_call(cuda, op):
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((16, 64), generator=g, device="cuda").bfloat16()
    w = torch.randn((2, 64, 64), generator=g, device="cuda").bfloat16()
    one, seg = torch.ones(64, device="cuda").bfloat16(), torch.tensor([0, 7, 16], dtype=torch.int32, device="cuda")
    a = torch.randint(0, 2, (16, 1), generator=g, device="cuda", dtype=torch.int32)
    wq = torch.randint(0, 256, (2, 64, 32), generator=g, device="cuda", dtype=torch.uint8)
    ws = torch.ones((2, 64, 2), device="cuda").bfloat16()
    wts, pos = torch.ones(16, 1, device="cuda"), torch.arange(16, dtype=torch.int32, device="cuda")
    space = mb.Workspace(16, 1, 2)
    call = {"norm": lambda: mb.block_norm(x, x, one, one).normed,
            "norm_backward": lambda: mb.block_norm_backward(x, x, x, x, one, one).d_y,
            "w4": lambda: mb.expert_linear_w4(x, a, wq, ws), "grouped_mm": lambda: mb.grouped_mm(x, seg, w),
            "pack": lambda: mb.pack(x, a, wts, 2, workspace=space).packed,
            "unpermute": lambda: mb.unpermute(x, wts, pos, 16, 1)}[op]
    want = call()
    fail_once()
    assert torch.equal(call(), want)
