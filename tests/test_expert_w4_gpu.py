"""GPU numerics of the 4-bit expert products against 64 bits, element by
element.

Tolerances: x and q - z are exact 16-bit numbers and their products exact in
fp32.  The tensor core adds them up in fp32, where each of the d additions is
off by at most 2^-23 of the largest partial sum (it may cut instead of round);
scaling, the sum over groups and the joining of parts add a few more fp32
roundings: (d + 64) 2^-23 sum |x||w| covers them.  The 16-bit result adds half
a step.  SwiGLU: silu's slope is at most 1.1 and |silu(g)| <= |g|, so an error
of g and u moves silu(g) u by at most 1.1 |dg||u| + |g||du|, and the fp32
exponential and division add 16 x 2^-24."""
import pytest
import torch

import moe_b200 as mb


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def make(T, K, E, d, N, group, dtype, zeros=False, per_slot=False, asgn=None, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((T, K, d) if per_slot else (T, d), generator=g, device="cuda").to(dtype)
    wq = torch.randint(0, 256, (E, N, d // 2), generator=g, device="cuda", dtype=torch.uint8)
    ws = ((0.5 + torch.rand((E, N, d // group), generator=g, device="cuda")) * 0.01).to(dtype)
    wz = torch.randint(0, 16, (E, N, d // group), generator=g, device="cuda", dtype=torch.uint8) if zeros else None
    if asgn is None:
        asgn = torch.rand((T, E), generator=g, device="cuda").topk(K, dim=1).indices.to(torch.int32)
    return x, asgn.contiguous(), wq, ws, wz


def weights64(wq, ws, wz):
    E, N, half = wq.shape
    q = torch.stack([wq & 15, wq >> 4], dim=-1).reshape(E, N, 2 * half).double()
    group = 2 * half // ws.shape[2]
    z = 8.0 if wz is None else wz.double().repeat_interleave(group, 2)
    return (q - z) * ws.double().repeat_interleave(group, 2)


def check(x, asgn, wq, ws, wz, act=None, got=None):
    T, K = asgn.shape
    d = x.shape[-1]
    y = mb.expert_linear_w4(x, asgn, wq, ws, wz, act) if got is None else got
    w = weights64(wq, ws, wz)
    rows = (x if x.dim() == 3 else x.unsqueeze(1).expand(T, K, d)).reshape(T * K, d).double()
    N = w.shape[1]
    e = asgn.flatten().long()
    live = (e >= 0) & (e < w.shape[0])
    ref, mag = (torch.zeros((T * K, N), dtype=torch.float64, device="cuda") for _ in range(2))
    for i in e[live].unique().tolist():
        at = (e == i).nonzero().flatten()
        ref[at], mag[at] = rows[at] @ w[i].T, rows[at].abs() @ w[i].abs().T
    err = (d + 64) * 2.0 ** -23 * mag
    if act:
        g, u, eg, eu = ref[:, :N // 2], ref[:, N // 2:], err[:, :N // 2], err[:, N // 2:]
        ref = g * torch.sigmoid(g) * u
        err = 1.1 * eg * u.abs() + g.abs() * eu + eg * eu + 16 * 2.0 ** -24 * ref.abs()
    h = half_step(x.dtype)
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 1e-38
    bound = h * ref.abs() + (1 + h) * err + tiny
    off = (y.double() - ref).abs()
    assert (off <= bound).all(), f"worst {float((off / bound).max()):.3g} of the bound"
    assert not y[~live].any()
    return y


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("act", [None, "swiglu"])
@pytest.mark.parametrize("T,K,E,d,N,per_slot", [
    (1, 1, 1, 128, 16, False),        # the smallest call
    (1, 4, 60, 256, 80, False),       # a single token
    (3, 2, 5, 384, 48, True),         # slots >= experts, a row for each slot
    (40, 4, 8, 128, 112, False),      # about 20 rows an expert: several passes of rows
    (9, 8, 128, 640, 32, True),       # fewer slots than experts
])
def test_products(cuda, dtype, group, act, T, K, E, d, N, per_slot):
    check(*make(T, K, E, d, N, group, dtype, zeros=group != 64, per_slot=per_slot, seed=T + d), act=act)
    assert mb.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("d,group", [(32, 32), (96, 32), (64, 64), (1408, 32), (1408, 128), (2080, 32), (4096, 128), (8192, 64),
                                     (14336, 128)])
def test_lengths(cuda, d, group):
    """Reduced lengths of one group, in no multiple of a step, and long ones."""
    check(*make(2, 2, 4, d, 24, group, torch.bfloat16, zeros=True, seed=d))
    check(*make(30, 2, 2, d, 40, group, torch.float16, seed=d))


@pytest.mark.gpu
@pytest.mark.parametrize("N", [8, 24, 40, 264, 1000])
def test_widths(cuda, N):
    check(*make(5, 3, 6, 256, N, 64, torch.bfloat16, seed=N))


@pytest.mark.gpu
@pytest.mark.parametrize("T,K,E", [(100, 1, 3), (7, 4, 60), (150, 4, 60), (1024, 4, 9)])
def test_one_expert_takes_all(cuda, T, K, E):
    """Every slot on one expert: also the same expert twice for a token."""
    asgn = torch.full((T, K), E - 1, dtype=torch.int32, device="cuda")
    check(*make(T, K, E, 128, 32, 32, torch.bfloat16, asgn=asgn))


@pytest.mark.gpu
@pytest.mark.parametrize("E", [4, 60])
def test_empty_slots_and_bad_experts(cuda, E):
    """-1 gives a row of zeros silently, another expert out of range zeros and
    the status; both with slots below and above the number of experts."""
    a = torch.tensor([[0, -1], [3, 1], [-1, -1], [2, 0], [3, -1]], dtype=torch.int32, device="cuda")
    p = make(5, 2, E, 256, 64, 64, torch.bfloat16, asgn=a)
    check(*p)
    check(*p, act="swiglu")
    assert mb.device_status() == 0
    a[1, 0], a[0, 0] = E, -2
    check(p[0], a, *p[2:])
    assert mb.device_status() == mb.DEV_BAD_ASSIGNMENT
    a.fill_(-1)
    check(p[0], a, *p[2:])
    assert mb.device_status() == 0


@pytest.mark.gpu
def test_bad_rows_stay_alone(cuda):
    """NaN in one token's row (a padded token) reaches no other token that
    shares its experts, and an empty slot's row is zeros all the same."""
    x, a, wq, ws, wz = make(12, 2, 3, 256, 48, 128, torch.bfloat16)
    want = mb.expert_linear_w4(x, a, wq, ws, wz)
    x[5] = float("nan")
    a[7] = -1
    got = mb.expert_linear_w4(x, a, wq, ws, wz)
    keep = [s for s in range(24) if s // 2 not in (5, 7)]
    assert torch.equal(got[keep], want[keep])
    assert not got[14:16].any()


@pytest.mark.gpu
@pytest.mark.parametrize("T,K,E,d", [(1024, 4, 1024, 64), (32, 1, 1024, 2048), (33, 1, 1, 256), (8, 4, 3, 128), (2048, 2, 2, 96)])
def test_table_limits(cuda, T, K, E, d):
    """The most slots and experts, and the border of the one-warp slot lists."""
    check(*make(T, K, E, d, 16, 32, torch.bfloat16, zeros=True, seed=E, asgn=torch.randint(-1, E, (T, K), device="cuda", dtype=torch.int32)))
    assert mb.device_status() == 0


@pytest.mark.gpu
def test_no_tokens(cuda):
    p = make(0, 2, 3, 128, 16, 32, torch.float16)
    assert mb.expert_linear_w4(*p).shape == (0, 16)


@pytest.mark.gpu
def test_offsets_past_32_bits(cuda):
    E, N, d = 130, 8192, 8192  # 4.4e9 bytes of weights
    wq = torch.zeros((E, N, d // 2), dtype=torch.uint8, device="cuda")
    wq[-1] = torch.randint(0, 256, (N, d // 2), device="cuda", dtype=torch.uint8)
    ws = torch.full((E, N, d // 32), 0.004, dtype=torch.bfloat16, device="cuda")
    x = torch.randn((2, d), device="cuda").bfloat16()
    a = torch.full((2, 1), E - 1, dtype=torch.int32, device="cuda")
    y = mb.expert_linear_w4(x, a, wq, ws)
    check(x, torch.zeros_like(a), wq[-1:], ws[-1:], None, got=y)


@pytest.mark.gpu
def test_same_bits_streams_and_graphs(cuda):
    p = make(33, 4, 16, 512, 96, 128, torch.bfloat16, zeros=True)
    want = mb.expert_linear_w4(*p, act="swiglu")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = mb.expert_linear_w4(*p, act="swiglu", stream=s)
    s.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mb.expert_linear_w4(*p, act="swiglu")
    q = make(33, 4, 16, 512, 96, 128, torch.bfloat16, zeros=True, seed=4)
    for a, b in zip(p, q):
        a.copy_(b)
    graph.replay()
    check(*p, act="swiglu", got=out)


@pytest.mark.gpu
def test_result_on_the_rows_is_refused(cuda):
    x, a, wq, ws, wz = make(3, 2, 4, 64, 64, 32, torch.bfloat16, per_slot=True)
    with pytest.raises(mb.MoEB200Error, match="overlaps"):
        mb.expert_linear_w4(x, a, wq, ws, out=x.view(6, 64))


# ------------------------------------------------------------- refusals ----

def test_refusals():
    x, a = torch.zeros((3, 64)).half(), torch.zeros((3, 2), dtype=torch.int32)
    wq, ws = torch.zeros((4, 32, 32), dtype=torch.uint8), torch.zeros((4, 32, 2)).half()
    bad = [
        lambda: mb.expert_linear_w4(x, a, wq, ws, act="gelu"),
        lambda: mb.expert_linear_w4(x[:2], a, wq, ws),
        lambda: mb.expert_linear_w4(x[:, :32], a, wq, ws),
        lambda: mb.expert_linear_w4(x, a.long(), wq, ws),
        lambda: mb.expert_linear_w4(x, a[:, 0], wq, ws),
        lambda: mb.expert_linear_w4(x, a, wq.to(torch.int8), ws),
        lambda: mb.expert_linear_w4(x, a, wq, ws.bfloat16()),
        lambda: mb.expert_linear_w4(x, a, wq, torch.zeros((4, 32, 3)).half()),
        lambda: mb.expert_linear_w4(x, a, wq, ws, w_zero=torch.zeros((4, 32, 2))),
        lambda: mb.expert_linear_w4(x.float(), a, wq, ws.float()),
        lambda: mb.expert_linear_w4(x, a, wq, ws, out=torch.zeros((6, 16)).half()),
        lambda: mb.expert_linear_w4(x, a, wq, ws),                                # not on a GPU
    ]
    for f in bad:
        with pytest.raises(mb.MoEB200Error) as e:
            f()
        assert e.value.status == mb.ERR_INVALID_ARG


def test_c_refusals():
    p = 0x10000

    def call(x=p, a=p, T=2, K=2, E=4, d=64, N=32, wq=p, ws=p, wz=None, group=32, act=0, dt=0, out=p):
        return mb.lib().moe_b200_expert_linear_w4(x, 0, a, T, K, E, d, N, wq, ws, wz, group, act, dt, out, None)

    assert call(T=0) == mb.OK
    assert call(T=-1) == call(K=0) == call(E=0) == call(d=0) == call(N=0) == call(dt=2) == call(act=2) == mb.ERR_INVALID_ARG
    assert call(x=None) == call(a=None) == call(wq=None) == call(ws=None) == call(out=None) == mb.ERR_INVALID_ARG
    assert call(x=p + 2) == call(wz=p + 4) == mb.ERR_INVALID_ARG
    assert call(group=16) == call(group=128) == call(N=12) == call(N=24, act=1) == call(T=2049) == mb.ERR_UNSUPPORTED
    assert call(E=mb.MAX_EXPERTS + 1) == mb.ERR_UNSUPPORTED
