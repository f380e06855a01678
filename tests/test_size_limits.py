"""Sizes near 2^31 that the host refuses, because tile and row indices behind
them are 32-bit (no GPU: nothing is launched)."""
import pytest

import moe_b200 as mb

P, BIG = 0x1000000000, 2 ** 31 - 8  # addresses far apart that are never followed


@pytest.mark.parametrize("which", ["rows", "N", "K"])
@pytest.mark.parametrize("fn", ["forward", "dgrad", "wgrad"])
def test_grouped_products(fn, which):
    s = dict(rows=4, N=16, K=16) | {which: BIG}
    x, seg, w, y = (P * (64 + 64 * i) for i in range(4))
    if fn == "wgrad":
        got = mb.lib().moe_b200_grouped_mm_wgrad(w, x, seg, 1, s["rows"], s["N"], s["K"], mb.BF16, y, None)
    else:
        f = mb.lib().moe_b200_grouped_mm if fn == "forward" else mb.lib().moe_b200_grouped_mm_dgrad
        got = f(x, seg, None, 1, s["rows"], s["N"], s["K"], 1, w, mb.BF16, y, None)
    assert got == mb.ERR_UNSUPPORTED


@pytest.mark.parametrize("d,N", [(2 ** 31 - 128, 16), (2 ** 31 - 256, 16), (2 ** 30, 16), (64, BIG)])
def test_4bit_products(d, N):
    x, a, q, s, y = (P * (64 + 64 * i) for i in range(5))
    assert mb.lib().moe_b200_expert_linear_w4(x, 0, a, 1, 1, 1, d, N, q, s, None, 32, mb.ACT_NONE, mb.BF16, y, None) == mb.ERR_UNSUPPORTED
