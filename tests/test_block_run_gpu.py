"""The operators together, as a model runs them around and inside the layer:
one training step (norm, router, pack, products, unpermute, norm, and the way
back) and one decode step with 4-bit experts, each against 64 bits.

Tolerance: the longest way from an input to a gradient passes 10 roundings to
16 bits, each of at most half a step relative to its value.  Every stage is
linear in what was rounded before it (norms nearly so) and the roundings are
independent of the data, so in the 2-norm the result is off by at most about
their sum, 10 half steps; fp32 errors are far below."""
import subprocess
import sys

import pytest
import torch

import moe_b200 as mb
from conftest import PKG

pytestmark = pytest.mark.gpu


def off(got, ref):
    assert torch.isfinite(got).all()
    return float((got.double() - ref).norm() / ref.norm())


def rms(v, w, eps):
    return v / (v.pow(2).mean(1, keepdim=True) + eps).sqrt() * w


def make(T, d, E, K, seed, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s, scale=1.0, at=0.0: (torch.randn(s, generator=g, device="cuda") * scale + at).to(dtype)  # noqa: E731
    p = dict(r=rand(T, d, scale=1.5), w1=rand(d, scale=0.2, at=1.0), w_post=rand(d, scale=0.2, at=1.0),
             w2=rand(d, scale=0.2, at=1.0), gate=rand(T, 1, scale=0.2, at=0.7))
    p["router"] = mb.RouterWeights(torch.randn((d, E), generator=g, device="cuda") * d ** -0.5, dtype)
    return p, rand


@pytest.mark.parametrize("dtype,T,d,E,K,F", [(torch.bfloat16, 300, 256, 12, 3, 176), (torch.float16, 37, 512, 40, 4, 320),
                                             (torch.bfloat16, 1, 128, 8, 2, 64)])
def test_training_step(cuda, dtype, T, d, E, K, F):
    eps, scale = 1e-5, 0.8
    p, rand = make(T, d, E, K, T, dtype)
    w_up, w_down = rand(E, F, d, scale=d ** -0.5), rand(E, d, F, scale=F ** -0.5)
    dr2, dn2 = rand(T, d, scale=0.3), rand(T, d, scale=0.3)

    n = mb.block_norm(p["r"], w_pre=p["w1"], eps=eps).normed
    asgn, wts = mb.route(n, p["router"], K)
    packed = mb.pack(n, asgn, wts, E)
    mid, y = mb.grouped_ffn(packed.packed, packed.expert_start, w_up, w_down)
    out = mb.unpermute(y, packed.packed_weights, packed.slot_pos, T, K)
    f = mb.block_norm(p["r"], out, p["w_post"], p["w2"], p["gate"], scale, eps)

    b2 = mb.block_norm_backward(dr2, dn2, f.residual_out, out, p["w_post"], p["w2"], p["gate"], scale, eps)
    d_y = (b2.d_y.float()[packed.perm.long()] * packed.packed_weights[:, None]).to(dtype)
    seg = packed.expert_start
    d_w_down = mb.grouped_mm_wgrad(d_y, mid, seg)
    d_mid = mb.grouped_mm_dgrad(d_y, seg, w_down)
    d_w_up = mb.grouped_mm_wgrad(d_mid, packed.packed, seg)
    d_packed = mb.grouped_mm_dgrad(d_mid, seg, w_up)
    d_n = mb.unpermute(d_packed, torch.ones_like(packed.packed_weights), packed.slot_pos, T, K)
    b1 = mb.block_norm_backward(b2.d_residual, d_n, p["r"], w_pre=p["w1"], eps=eps)
    assert mb.device_status() == 0

    leaf = {k: p[k].double().requires_grad_(True) for k in ("r", "w1", "w_post", "w2", "gate")}
    leaf |= {"w_up": w_up.double().requires_grad_(True), "w_down": w_down.double().requires_grad_(True)}
    x = rms(leaf["r"], leaf["w1"], eps)
    o = torch.zeros((T, d), dtype=torch.float64, device="cuda")
    for k in range(K):
        e = asgn[:, k].long()
        o = o + wts[:, k:k + 1].double() * torch.einsum("tf,tdf->td", torch.einsum("td,tfd->tf", x, leaf["w_up"][e]),
                                                        leaf["w_down"][e])
    r2 = leaf["r"] + scale * leaf["gate"] * rms(o, leaf["w_post"], eps)
    n2 = rms(r2, leaf["w2"], eps)
    got = dict(zip(leaf, torch.autograd.grad([r2, n2], list(leaf.values()), [dr2.double(), dn2.double()])))
    bound = 10 * torch.finfo(dtype).eps / 2
    assert off(f.residual_out, r2.detach()) < bound and off(f.normed, n2.detach()) < bound
    for name, mine in (("r", b1.d_residual), ("w1", b1.d_w_pre), ("w_post", b2.d_w_post), ("w2", b2.d_w_pre),
                       ("gate", b2.d_gate), ("w_up", d_w_up), ("w_down", d_w_down)):
        assert off(mine, got[name]) < bound, name


def decode_step(p, q, asgn, K, eps, scale):
    n = mb.block_norm(p["r"], w_pre=p["w1"], eps=eps).normed
    h = mb.expert_linear_w4(n, asgn, *q["gate_up"], act="swiglu")
    y = mb.expert_linear_w4(h.view(asgn.shape[0], K, -1), asgn, *q["down"])
    out = mb.unpermute(y, q["wts"], q["slots"], asgn.shape[0], K)
    return mb.block_norm(p["r"], out, p["w_post"], p["w2"], p["gate"], scale, eps)


def weights64(wq, ws, wz):
    w = torch.stack([wq & 15, wq >> 4], dim=-1).flatten(-2).double()
    group = w.shape[-1] // ws.shape[-1]
    z = 8.0 if wz is None else wz.double().repeat_interleave(group, -1)
    return (w - z) * ws.double().repeat_interleave(group, -1)


@pytest.mark.parametrize("T", [1, 13, 96])
def test_decode_step_captured_and_replayed(cuda, T):
    """A batch whose last tokens are padding (expert -1), captured once and
    replayed with other tokens and experts."""
    dtype, d, E, K, I, group, eps, scale = torch.bfloat16, 512, 24, 4, 192, 64, 1e-6, 0.5
    p, rand = make(T, d, E, K, T, dtype)
    g = torch.Generator(device="cuda").manual_seed(2)

    def quant(n, k, zeros):
        return (torch.randint(0, 256, (E, n, k // 2), generator=g, device="cuda", dtype=torch.uint8),
                ((0.5 + torch.rand((E, n, k // group), generator=g, device="cuda")) * 0.2 * k ** -0.5).to(dtype),
                torch.randint(0, 16, (E, n, k // group), generator=g, device="cuda", dtype=torch.uint8) if zeros else None)

    q = {"gate_up": quant(2 * I, d, True), "down": quant(d, I, False),
         "slots": torch.arange(T * K, dtype=torch.int32, device="cuda")}
    live = max(1, T - 3)

    def route(r):
        n = mb.block_norm(r, w_pre=p["w1"], eps=eps).normed
        asgn, wts = mb.route(n, p["router"], K)
        asgn[live:] = -1
        return asgn, wts

    asgn, wts = route(p["r"])
    q["wts"] = wts.flatten().contiguous()
    decode_step(p, q, asgn, K, eps, scale)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = decode_step(p, q, asgn, K, eps, scale)
    p["r"].copy_(rand(T, d, scale=1.5))
    a2, w2 = route(p["r"])
    asgn.copy_(a2)
    q["wts"].copy_(w2.flatten())
    graph.replay()
    torch.cuda.synchronize()
    assert mb.device_status() == 0

    r = p["r"].double()
    x, gu, dn = rms(r, p["w1"].double(), eps), weights64(*q["gate_up"]), weights64(*q["down"])
    o = torch.zeros_like(r)
    for k in range(K):
        e = a2[:live, k].long()
        v = torch.einsum("td,tnd->tn", x[:live], gu[e])
        h = torch.nn.functional.silu(v[:, :I]) * v[:, I:]
        o[:live] += w2[:live, k:k + 1].double() * torch.einsum("tn,tdn->td", h, dn[e])
    r2 = r + scale * p["gate"].double() * rms(o, p["w_post"].double(), eps)
    bound = 10 * torch.finfo(dtype).eps / 2
    assert off(got.residual_out, r2) < bound
    assert off(got.normed, rms(r2, p["w2"].double(), eps)) < bound
    assert torch.equal(got.residual_out[live:], p["r"][live:])  # padding: the block adds nothing


FIRST_CALLS = """
import sys; sys.path.insert(0, sys.argv[1])
import torch, moe_b200 as mb
mb.lib()
x = torch.randn((40, 256), device="cuda").bfloat16()
w = torch.randn((2, 128, 256), device="cuda").bfloat16()
one = torch.ones((256,), device="cuda").bfloat16()
dy = torch.randn((40, 128), device="cuda").bfloat16()
seg = torch.tensor([0, 15, 40], dtype=torch.int32, device="cuda")
big = torch.randn((3000, 256), device="cuda").bfloat16()
bseg = torch.tensor([0, 1500, 3000], dtype=torch.int32, device="cuda")
asgn = torch.zeros((40, 1), dtype=torch.int32, device="cuda")
wq = torch.randint(0, 256, (2, 64, 128), dtype=torch.uint8, device="cuda")
ws = torch.ones((2, 64, 2), device="cuda").bfloat16()
torch.cuda.synchronize()

def calls():
    f = mb.block_norm(big, big, one, one)
    b = mb.block_norm_backward(big, big, big, big, one, one)
    return [f.residual_out, f.normed, *b[:4], mb.grouped_mm(x, seg, w), mb.grouped_mm(big, bseg, w), mb.grouped_mm_dgrad(dy, seg, w),
            mb.grouped_mm_wgrad(dy, x, seg), mb.expert_linear_w4(x, asgn, wq, ws)]

graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = calls()
graph.replay()
want = calls()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, want)) and mb.device_status() == 0
print("captured first")
"""


def test_first_calls_may_be_captured(cuda):
    """A process whose first call of each operator is made during a capture."""
    out = subprocess.run([sys.executable, "-c", FIRST_CALLS, PKG], capture_output=True, text=True, timeout=300)
    assert "captured first" in out.stdout, out.stderr[-2000:]
