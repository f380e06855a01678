"""The block norms over so many rows that the stages of the shared-memory ring
are refilled, for each of its forms, against 64 bits; and the gradients against
differentiation of the forward's definition.  Tolerances as in
test_block_norm_gpu."""
import pytest
import torch

import moe_b200 as mb
from test_block_norm_gpu import assert_close, backward64, check, dbl, forward64, make

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32

# (gate, norm behind the block, norm before the next, with a block at all)
FORMS = [(None, True, True, True), ("token", True, True, True), ("channel", True, True, True), ("full", True, True, True),
         ("token", False, True, True), (None, False, True, True),   # no norm behind the block
         (None, False, True, False),                                 # the norm alone
         ("channel", False, True, True), ("full", True, False, True)]  # rarer ones


@pytest.mark.parametrize("gate,post,pre,with_y", FORMS)
@pytest.mark.parametrize("T,d", [
    (20003, 64), (16001, 512),                 # a row a warp
    (12001, 1024), (12007, 2048), (5003, 4096),  # a row a CTA of 64, 128, 256 threads
    (1501, 8192), (901, 16384)])               # of 512 and 1024
@pytest.mark.parametrize("dtype,res", [(BF, BF), (HF, F32)])
def test_rows_enough_to_refill_the_ring(cuda, T, d, dtype, res, gate, post, pre, with_y):
    p = make(T, d, dtype, res, gate, post, pre, seed=T)
    if not with_y:
        p["y"] = None
    check(p)
    assert mb.device_status() == 0


@pytest.mark.parametrize("T,d", [(20003, 64), (12007, 2048), (1501, 8192)])
def test_strided_rows_through_the_ring(cuda, T, d):
    """y and the residual as columns of one wider tensor, in 16-byte steps."""
    p = make(T, d, BF, BF, "token", True, True, seed=d)
    wide = torch.randn((T, 2 * d + 8), device="cuda").to(BF)
    p["y"], p["residual"] = wide[:, :d], wide[:, d + 8:]
    check(p)


@pytest.mark.parametrize("T,d", [(20003, 64), (12007, 2048)])
def test_results_on_the_rows_of_the_ring(cuda, T, d):
    """The results take the places of the rows that the ring has read."""
    p = make(T, d, BF, BF, "token", True, True, seed=d)
    want = mb.block_norm(p["residual"], p["y"], p["w_post"], p["w_pre"], p["gate"], 0.3)
    mb.block_norm(p["residual"], p["y"], p["w_post"], p["w_pre"], p["gate"], 0.3, out=mb.BlockNormResult(p["residual"], p["y"]))
    assert torch.equal(p["residual"], want.residual_out) and torch.equal(p["y"], want.normed)


def gradients64(p, residual_out, scale, eps):
    """The gradients by differentiating forward64, which states the definition:
    the norm before the next block at the stored residual_out, then the branch."""
    leaf = {k: dbl(p[k]).requires_grad_(True) for k in ("y", "w_post", "w_pre", "gate") if p[k] is not None}
    r, ds, got = dbl(residual_out).requires_grad_(True), dbl(p["d_res"]), {}
    if p["w_pre"] is not None:
        n = forward64(dict(residual=r, y=None, w_post=None, w_pre=leaf["w_pre"], gate=None), scale, eps)[2]
        by_r, got["d_w_pre"] = torch.autograd.grad(n, [r, leaf["w_pre"]], dbl(p["d_normed"]))
        ds = ds + by_r
    got["d_residual"] = ds
    if p["y"] is not None:
        names = [k for k in ("y", "w_post", "gate") if k in leaf]
        s = forward64(dict(residual=torch.zeros_like(r), y=leaf["y"], w_post=leaf.get("w_post"), w_pre=None, gate=leaf.get("gate")),
                      scale, eps)[0]
        got |= {"d_" + k: g for k, g in zip(names, torch.autograd.grad(s, [leaf[k] for k in names], ds))}
    return got


@pytest.mark.parametrize("gate,post,pre,with_y", FORMS)
@pytest.mark.parametrize("T,d", [(4, 96), (37, 33), (300, 520), (2500, 264), (3, 8200)])
@pytest.mark.parametrize("dtype,res", [(BF, BF), (HF, F32)])
def test_gradients_are_those_of_the_forward(cuda, T, d, dtype, res, gate, post, pre, with_y):
    scale, eps = 0.7, 1e-5
    p = make(T, d, dtype, res, gate, post, pre, seed=T + d)
    if not with_y:
        p["y"] = None
    kw = dict(w_post=p["w_post"], w_pre=p["w_pre"], gate=p["gate"], scale=scale, eps=eps)
    f = mb.block_norm(p["residual"], p["y"], **kw)
    b = mb.block_norm_backward(p["d_res"], p["d_normed"], f.residual_out, p["y"], **kw)._asdict()
    want, mag = gradients64(p, f.residual_out, scale, eps), backward64(p, f.residual_out, scale, eps)[1]
    assert {k for k, t in b.items() if t is not None} == set(want)
    for k, ref in want.items():
        assert_close(b[k], ref, mag[k], k, ops=128 + (T if k in ("d_w_post", "d_w_pre", "d_gate") else 0))
