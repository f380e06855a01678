"""What the C entry points of the norms, the grouped and the 4-bit products
refuse of their pointers (no GPU: nothing is launched)."""
import pytest

import moe_b200 as mb

P = 0x100000  # addresses that are never followed: every call here is refused


def norm(res32=0, **ptrs):
    a = dict(y=P, r=P + 0x10000, wo=P + 0x20000, wn=P + 0x20100, ga=P + 0x30000, ro=P + 0x40000, no=P + 0x50000) | ptrs
    return mb.lib().moe_b200_block_norm(a["y"], 16, a["r"], 16, res32, a["wo"], a["wn"], a["ga"], mb.GATE_FULL, 1.0, 1e-6, 4, 16,
                                        mb.BF16, a["ro"], a["no"], None)


def norm_backward(res32=0, form=mb.GATE_FULL, **ptrs):
    names = ("dr", "dn", "r", "y", "wo", "wn", "ga", "d_r", "d_y", "d_wo", "d_wn", "d_g", "ws")
    a = {n: P + 0x10000 * i for i, n in enumerate(names)} | ptrs
    nbytes = mb.lib().moe_b200_block_norm_backward_workspace_bytes(4, 16)
    return mb.lib().moe_b200_block_norm_backward(a["dr"], a["dn"], a["r"], 16, res32, a["y"], 16, a["wo"], a["wn"], a["ga"], form, 1.0,
                                                 1e-6, 4, 16, mb.BF16, a["d_r"], a["d_y"], a["d_wo"], a["d_wn"], a["d_g"], a["ws"],
                                                 nbytes, None)


def grouped(fn, se=None, **ptrs):
    a = dict(x=P, seg=P + 0x10000, w=P + 0x20000, y=P + 0x30000) | ptrs
    if fn == "wgrad":
        return mb.lib().moe_b200_grouped_mm_wgrad(a["w"], a["x"], a["seg"], 2, 4, 16, 16, mb.BF16, a["y"], None)
    f = mb.lib().moe_b200_grouped_mm if fn == "forward" else mb.lib().moe_b200_grouped_mm_dgrad
    return f(a["x"], a["seg"], se, 2, 4, 16, 16, 2, a["w"], mb.BF16, a["y"], None)


def w4(**ptrs):
    a = dict(x=P, asgn=P + 0x10000, q=P + 0x20000, s=P + 0x30000, z=None, out=P + 0x40000) | ptrs
    return mb.lib().moe_b200_expert_linear_w4(a["x"], 0, a["asgn"], 2, 2, 4, 64, 32, a["q"], a["s"], a["z"], 32, mb.ACT_NONE, mb.BF16,
                                              a["out"], None)


@pytest.mark.parametrize("name", ["y", "r", "wo", "wn", "ga", "ro", "no"])
def test_norm_pointers_inside_an_element(name):
    assert norm(**{name: P + 0x60000 + 1}) == mb.ERR_INVALID_ARG
    if name in ("r", "ro"):  # fp32
        assert norm(res32=1, **{name: P + 0x60000 + 2}) == mb.ERR_INVALID_ARG


@pytest.mark.parametrize("name", ["dr", "dn", "r", "y", "wo", "wn", "ga", "d_r", "d_y", "d_wo", "d_wn", "d_g"])
def test_norm_backward_pointers_inside_an_element(name):
    at = P + 0x200000
    assert norm_backward(**{name: at + 1}) == mb.ERR_INVALID_ARG
    if name in ("dr", "r", "d_r"):
        assert norm_backward(res32=1, **{name: at + 2}) == mb.ERR_INVALID_ARG
    if name in ("d_wo", "d_wn"):
        assert norm_backward(**{name: at + 2}) == mb.ERR_INVALID_ARG
    if name == "d_g":
        for form in (mb.GATE_TOKEN, mb.GATE_CHANNEL):
            assert norm_backward(form=form, d_g=at + 2) == mb.ERR_INVALID_ARG


@pytest.mark.parametrize("fn", ["forward", "dgrad", "wgrad"])
def test_grouped_tables_inside_an_element(fn):
    assert grouped(fn, seg=P + 0x10002) == mb.ERR_INVALID_ARG
    if fn != "wgrad":
        assert grouped(fn, se=P + 0x11001) == mb.ERR_INVALID_ARG


def test_w4_assignments_inside_an_element():
    assert w4(asgn=P + 0x10002) == mb.ERR_INVALID_ARG


# Results that lie on what is read, or on one another.  (T, d = 4, 16: a 16-bit
# row set of 128 bytes, a 16-bit vector of 32, fp32 twice that.)

ROWS, VEC = 128, 32


@pytest.mark.parametrize("out", ["ro", "no"])
@pytest.mark.parametrize("read", ["y", "r", "ga"])
def test_norm_results_on_other_rows(out, read):
    at = P + 0x60000
    for off in (-ROWS + 2, -32, 32, ROWS - 2):
        assert norm(**{out: at + off, read: at}) == mb.ERR_INVALID_ARG


def test_norm_results_on_vectors_and_on_one_another():
    at = P + 0x60000
    for out in ("ro", "no"):
        for vec in ("wo", "wn"):
            for off in (-VEC + 2, 0, ROWS - 2):
                assert norm(**{out: at, vec: at + off}) == mb.ERR_INVALID_ARG
    assert norm(ro=at, no=at) == norm(ro=at, no=at + ROWS - 2) == norm(ro=at, no=at - ROWS + 2) == mb.ERR_INVALID_ARG
    # the same start, but rows of another width lie on other rows
    assert norm(res32=1, r=at, no=at) == norm(res32=1, y=at, ro=at) == mb.ERR_INVALID_ARG


@pytest.mark.parametrize("out,size", [("d_r", ROWS), ("d_y", ROWS), ("d_g", ROWS), ("d_wo", 64), ("d_wn", 64), ("ws", 256)])
def test_norm_backward_results_on_other_rows(out, size):
    at = P + 0x200000
    names = ["dr", "dn", "r", "y", "ga", "wo", "wn", "d_r", "d_y", "d_g", "d_wo", "d_wn", "ws"]
    for other in names:
        if other == out:
            continue
        step = 256 if "ws" in (out, other) else 4
        for off in (-step, 0, step):
            if off == 0 and other in ("dr", "dn", "r", "y", "ga") and out in ("d_r", "d_y", "d_g") and (out, other) not in (
                    ("d_r", "y"), ("d_r", "ga")):
                continue  # the same rows: right
            if off < 0 and off + {"ws": 256, "d_wo": 64, "d_wn": 64, "wo": VEC, "wn": VEC}.get(other, ROWS) <= 0:
                continue  # ends before
            if off > 0 and off >= size:
                continue  # begins behind
            assert norm_backward(**{out: at, other: at + off}) == mb.ERR_INVALID_ARG, (other, off)


@pytest.mark.parametrize("fn", ["forward", "dgrad", "wgrad"])
def test_grouped_results_on_what_is_read(fn):
    at = P + 0x60000
    size = {"wgrad": 2 * 16 * 16 * 2}.get(fn, ROWS)
    for read, nbytes in (("x", ROWS), ("w", ROWS if fn == "wgrad" else 1024), ("seg", 12)):
        for off in (-(nbytes // 16 * 16) + 16 if nbytes > 16 else 0, 0, size - 16):
            assert grouped(fn, **{"y": at, read: at + off}) == mb.ERR_INVALID_ARG
    if fn != "wgrad":
        assert grouped(fn, y=at, se=at + 4) == mb.ERR_INVALID_ARG


def test_w4_results_on_what_is_read():
    at = P + 0x60000
    size = 4 * 32 * 2
    for read, nbytes in (("x", 2 * 64 * 2), ("asgn", 16), ("q", 4 * 32 * 32), ("s", 4 * 32 * 2 * 2), ("z", 4 * 32 * 2)):
        for off in (-nbytes + 16, 0, size - 16):
            assert w4(**{"out": at, read: at + off}) == mb.ERR_INVALID_ARG


def test_no_bytes_overlap_nothing():
    """A product without rows has operands of no bytes, wherever they point."""
    L, at = mb.lib(), P + 0x60000
    for x in (at - 16, at, at + 512, at + 4096):
        # (the result overlaps its table, which refuses the call before anything is enqueued)
        assert L.moe_b200_grouped_mm_wgrad(x, x, at + 4, 2, 0, 16, 16, mb.BF16, at, None) == mb.ERR_INVALID_ARG
