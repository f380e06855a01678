"""GPU numerics of the block norms (forward and backward) against their
formulas in 64 bits, element by element.

Tolerances: u = 2^-24 is the relative error of one fp32 operation.  A row sum
takes at most 16 sequential additions a thread, 5 shuffles and 32 warp parts,
and each output a few products and one rsqrt on top, so an fp32 result is off
by less than 128 u of the magnitudes that went into it (the sum of absolute
values, written out in mags()); a 16-bit result by half a step more, a column
sum over T tokens by T u more.  fp16 results below 2^-14 have an absolute step
of 2^-24."""
import pytest
import torch

import moe_b200 as mb

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def assert_close(got, ref, mag, name, ops=128):
    """|got - ref| <= half a step of |ref| + ops * u * mag (+ half the smallest fp16 step)."""
    assert torch.isfinite(ref).all()
    step = half_step(got.dtype) if got.dtype != torch.float32 else U
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 1e-38
    bound = step * ref.abs() + ops * U * (1 + step) * mag + tiny
    err = (got.double() - ref).abs()
    assert (err <= bound).all(), f"{name}: worst {float((err / bound).max()):.3g} of the bound"


def rand(g, shape, dtype, scale=1.0, at=0.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale + at).to(dtype)


def make(T, d, dtype, res, gate, post, pre, seed=0):
    g = torch.Generator(device="cuda").manual_seed(1 + seed)
    shape = {None: None, "token": (T, 1), "channel": (1, d), "full": (T, d)}[gate]
    return dict(residual=rand(g, (T, d), res, 1.5), y=rand(g, (T, d), dtype, 0.7),
                w_post=rand(g, (d,), dtype, 0.2, 1.0) if post else None, w_pre=rand(g, (d,), dtype, 0.2, 1.0) if pre else None,
                gate=rand(g, shape, dtype, 0.3, 0.6) if shape else None,
                d_res=rand(g, (T, d), res, 0.3), d_normed=rand(g, (T, d), dtype, 0.3) if pre else None)


def dbl(t):
    return None if t is None else t.double()


def forward64(p, scale, eps):
    r, y, wo, wn, ga = (dbl(p[k]) for k in ("residual", "y", "w_post", "w_pre", "gate"))
    z = torch.zeros_like(r)
    if y is not None:
        z = y if wo is None else y / (y.pow(2).mean(1, keepdim=True) + eps).sqrt() * wo
        z = scale * z * (1.0 if ga is None else ga)
    s, mag = r + z, r.abs() + z.abs()
    if wn is None:
        return s, mag, None, None
    c = 1 / (s.pow(2).mean(1, keepdim=True) + eps).sqrt()
    # an error of s moves c too: by at most the mean of its relative size
    return s, mag, s * c * wn, c * wn.abs() * (mag + s.abs() * (mag * s.abs()).mean(1, keepdim=True) * c * c)


def backward64(p, residual_out, scale, eps):
    y, wo, wn, ga, dn = (dbl(p[k]) for k in ("y", "w_post", "w_pre", "gate", "d_normed"))
    r, ds = dbl(residual_out), dbl(p["d_res"])
    out, mag = {}, {}
    m_ds = ds.abs()
    if wn is not None:
        c = 1 / (r.pow(2).mean(1, keepdim=True) + eps).sqrt()
        u = dn * wn
        ds = ds + c * (u - r * c * c * (u * r).mean(1, keepdim=True))
        m_ds = m_ds + c * (u.abs() + r.abs() * c * c * (u * r).abs().mean(1, keepdim=True))
        out["d_w_pre"], mag["d_w_pre"] = (dn * r * c).sum(0), (dn * r * c).abs().sum(0)
    out["d_residual"], mag["d_residual"] = ds, m_ds
    if y is None:
        return out, mag
    a = torch.ones_like(y[:, :1]) if wo is None else 1 / (y.pow(2).mean(1, keepdim=True) + eps).sqrt()
    yh, w = y * a, (1.0 if wo is None else wo)
    if ga is not None:
        e, m = scale * ds * yh * w, (scale * m_ds * yh * w).abs()
        axis = {(y.shape[0], 1): 1, (1, y.shape[1]): 0}.get(tuple(ga.shape))
        if tuple(ga.shape) == tuple(y.shape):
            axis = None
        out["d_gate"], mag["d_gate"] = (e, m) if axis is None else (e.sum(axis, keepdim=True), m.sum(axis, keepdim=True))
    q = scale * ds * (1.0 if ga is None else ga)
    m_q = (scale * m_ds * (1.0 if ga is None else ga)).abs()
    if wo is not None:
        out["d_w_post"], mag["d_w_post"] = (q * yh).sum(0), (m_q * yh.abs()).sum(0)
        v, m_v = q * wo, m_q * wo.abs()
        q = a * (v - yh * (v * yh).mean(1, keepdim=True))
        m_q = a * (m_v + yh.abs() * (m_v * yh.abs()).mean(1, keepdim=True))
    out["d_y"], mag["d_y"] = q, m_q
    return out, mag


def run_both(p, scale, eps, stream=None):
    kw = dict(w_post=p["w_post"], w_pre=p["w_pre"], gate=p["gate"], scale=scale, eps=eps, stream=stream)
    f = mb.block_norm(p["residual"], p["y"], **kw)
    b = mb.block_norm_backward(p["d_res"], p["d_normed"], f.residual_out, p["y"], **kw)
    return f, b


def check(p, scale=0.7, eps=1e-5, got=None):
    T = p["residual"].shape[0]
    f, b = got or run_both(p, scale, eps)
    s, m_s, n, m_n = forward64(p, scale, eps)
    if p["y"] is None:
        assert f.residual_out is p["residual"]
    else:
        assert f.residual_out.dtype == p["residual"].dtype
        assert_close(f.residual_out, s, m_s, "residual_out")
    assert (f.normed is None) == (n is None)
    if n is not None:
        assert_close(f.normed, n, m_n, "normed")
    out, mag = backward64(p, f.residual_out, scale, eps)
    for name, t in b._asdict().items():
        assert (t is None) == (name not in out), name
        if t is not None:
            assert_close(t, out[name], mag[name], name, ops=128 + (T if name in ("d_w_post", "d_w_pre", "d_gate") else 0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,res", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32),
                                       (torch.bfloat16, torch.float32), (torch.float16, torch.float16)])
@pytest.mark.parametrize("gate", [None, "token", "channel", "full"])
@pytest.mark.parametrize("T,d", [(1, 8), (5, 64), (37, 256), (129, 1000), (3, 2048), (33, 33)])
def test_all_forms(cuda, dtype, res, gate, T, d):
    check(make(T, d, dtype, res, gate, True, True, seed=T + d))


@pytest.mark.gpu
@pytest.mark.parametrize("post,pre,with_y", [(True, False, True), (False, True, True), (False, False, True), (False, True, False)])
@pytest.mark.parametrize("T,d", [(2, 1), (70, 513), (600, 96)])
def test_parts(cuda, post, pre, with_y, T, d):
    p = make(T, d, torch.bfloat16, torch.bfloat16, "full" if with_y else None, post, pre)
    if not with_y:
        p["y"] = None
    check(p)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [1, 7, 255, 257, 511, 520, 4096, 4104, 8192, 8200, 16384, 16383])
@pytest.mark.parametrize("res", [torch.bfloat16, torch.float32])
def test_widths(cuda, d, res):
    """Every width class: threads a row, chunks a thread, aligned and not."""
    check(make(3, d, torch.bfloat16, res, "channel", True, True, seed=d))


@pytest.mark.gpu
@pytest.mark.parametrize("gate", ["token", "channel", "full"])
@pytest.mark.parametrize("T,d", [(2500, 177), (1200, 255), (1200, 1001), (700, 2050), (400, 4097), (300, 8201)])
def test_rows_that_begin_inside_a_word(cuda, gate, T, d):
    """Columns in pairs: with odd d every other row begins inside a word, and a
    CTA has several rows; with even d the rows end inside a 16-byte step."""
    check(make(T, d, torch.float16, torch.float32, gate, True, True, seed=d))
    check(make(T, d, torch.bfloat16, torch.bfloat16, gate, True, True, seed=d + 1))


@pytest.mark.gpu
@pytest.mark.parametrize("d,stride", [(65, 66), (65, 67), (66, 67), (64, 66)])
def test_strides_and_starts_of_either_kind(cuda, d, stride):
    """Row strides that agree with d in pairs and that do not, and a tensor that begins inside a word."""
    g = torch.Generator(device="cuda").manual_seed(stride)
    for start in (0, 1, 2):
        p = make(90, d, torch.bfloat16, torch.bfloat16, "full", True, True, seed=d + start)
        p["y"] = torch.as_strided(rand(g, (start + 90 * stride,), torch.bfloat16), (90, d), (stride, 1), start)
        check(p)
        flat = rand(g, (start + 90 * d,), torch.bfloat16)
        p["d_normed"] = flat[start:].view(90, d)
        check(p)


@pytest.mark.gpu
def test_many_rows_share_the_columns(cuda):
    """More rows than a grid holds at once: column sums over many rows a CTA."""
    check(make(5000, 72, torch.bfloat16, torch.bfloat16, "channel", True, True))


@pytest.mark.gpu
def test_rows_of_zeros_and_large_values(cuda):
    p = make(6, 128, torch.bfloat16, torch.float32, None, True, True)
    p["y"][0] = 0
    p["residual"][0] = 0
    p["y"][1] *= 1e15
    p["residual"][2] *= 1e-15
    check(p, eps=1e-6)


@pytest.mark.gpu
def test_a_bad_row_stays_alone(cuda):
    """Infinities and NaN in one row (a padded token) reach no other row."""
    p = make(9, 320, torch.bfloat16, torch.bfloat16, "token", True, True)
    clean = run_both(p, 1.0, 1e-6)
    for k, v in (("y", float("nan")), ("residual", float("inf")), ("d_res", float("nan"))):
        p[k][4] = v
    f, b = run_both(p, 1.0, 1e-6)
    keep = torch.arange(9, device="cuda") != 4
    assert torch.equal(f.normed[keep], clean[0].normed[keep]) and torch.equal(f.residual_out[keep], clean[0].residual_out[keep])
    assert torch.equal(b.d_y[keep], clean[1].d_y[keep]) and torch.equal(b.d_residual[keep], clean[1].d_residual[keep])


@pytest.mark.gpu
@pytest.mark.parametrize("d,off", [(64, 8), (64, 3), (33, 1)])
def test_strided_rows(cuda, d, off):
    """y and the residual as columns of wider tensors, aligned and not."""
    p = make(11, d, torch.float16, torch.float16, "token", True, True)
    wide = torch.randn((11, 2 * d + 16), device="cuda").half()
    p["y"] = wide[:, off:off + d]
    p["residual"] = wide[:, d + 8:2 * d + 8]
    check(p)


@pytest.mark.gpu
def test_in_place(cuda):
    p = make(50, 264, torch.bfloat16, torch.bfloat16, "channel", True, True)
    want = mb.block_norm(p["residual"], p["y"], p["w_post"], p["w_pre"], p["gate"], 0.3)
    mb.block_norm(p["residual"], p["y"], p["w_post"], p["w_pre"], p["gate"], 0.3,
                  out=mb.BlockNormResult(p["residual"], p["y"]))
    assert torch.equal(p["residual"], want.residual_out) and torch.equal(p["y"], want.normed)


@pytest.mark.gpu
@pytest.mark.parametrize("T,d", [(7, 40), (9, 33), (2500, 64), (700, 1024)])
def test_results_on_rows_that_are_read(cuda, T, d):
    """Either result on any of the rows that are read: the same bits."""
    bf = torch.bfloat16
    p = make(T, d, bf, bf, "full", True, True, seed=d)
    want = mb.block_norm(p["residual"], p["y"], p["w_post"], p["w_pre"], p["gate"], 0.3)
    for first, second in (("residual", "y"), ("y", "residual"), ("gate", "y"), ("residual", "gate")):
        q = {k: v.clone() if v is not None else None for k, v in p.items()}
        got = mb.block_norm(q["residual"], q["y"], q["w_post"], q["w_pre"], q["gate"], 0.3, out=mb.BlockNormResult(q[first], q[second]))
        assert torch.equal(got.residual_out, want.residual_out) and torch.equal(got.normed, want.normed)


@pytest.mark.gpu
@pytest.mark.parametrize("T,d", [(7, 40), (9, 33), (2500, 64), (700, 1024), (5, 8200)])
def test_gradients_on_rows_that_are_read(cuda, T, d):
    bf = torch.bfloat16
    p = make(T, d, bf, bf, "full", True, True, seed=d)
    r = p["residual"]
    want = mb.block_norm_backward(p["d_res"], p["d_normed"], r, p["y"], p["w_post"], p["w_pre"], p["gate"], 0.3)
    L = mb.lib()
    nbytes = L.moe_b200_block_norm_backward_workspace_bytes(T, d)
    for places in (("d_res", "y", "gate"), ("residual", "d_normed", "y"), ("d_normed", "gate", "d_res"), ("d_res", "residual", "d_normed")):
        q = {k: v.clone() for k, v in p.items()}
        sums, ws = torch.empty((2, d), device="cuda"), torch.empty(nbytes, device="cuda", dtype=torch.uint8)
        out = [q[k] for k in places]
        status = L.moe_b200_block_norm_backward(
            q["d_res"].data_ptr(), q["d_normed"].data_ptr(), q["residual"].data_ptr(), d, 0, q["y"].data_ptr(), d, q["w_post"].data_ptr(),
            q["w_pre"].data_ptr(), q["gate"].data_ptr(), mb.GATE_FULL, 0.3, 1e-6, T, d, mb.BF16, out[0].data_ptr(), out[1].data_ptr(),
            sums[0].data_ptr(), sums[1].data_ptr(), out[2].data_ptr(), ws.data_ptr(), nbytes, torch.cuda.current_stream().cuda_stream or None)
        assert status == mb.OK
        for got, ref in zip((*out, *sums), (want.d_residual, want.d_y, want.d_gate, want.d_w_post, want.d_w_pre)):
            assert torch.equal(got, ref), places


@pytest.mark.gpu
def test_no_rows(cuda):
    p = make(0, 48, torch.bfloat16, torch.float32, "channel", True, True)
    f, b = run_both(p, 1.0, 1e-6)
    assert f.normed.shape == (0, 48) and b.d_y.shape == (0, 48)
    assert not b.d_w_post.any() and not b.d_w_pre.any() and not b.d_gate.any()
    assert b.d_gate.shape == (1, 48)


@pytest.mark.gpu
def test_same_bits_again_and_on_another_stream(cuda):
    p = make(300, 1024, torch.bfloat16, torch.bfloat16, "channel", True, True)
    a = run_both(p, 1.0, 1e-6)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    b = run_both(p, 1.0, 1e-6, stream=s)
    s.synchronize()
    for x, y in zip((*a[0], *a[1]), (*b[0], *b[1])):
        assert torch.equal(x, y)


@pytest.mark.gpu
def test_captured_and_replayed(cuda):
    p = make(64, 512, torch.bfloat16, torch.bfloat16, "token", True, True)
    run_both(p, 1.0, 1e-6)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run_both(p, 0.7, 1e-5)
    q = make(64, 512, torch.bfloat16, torch.bfloat16, "token", True, True, seed=9)
    for k in p:
        p[k].copy_(q[k])
    graph.replay()
    check(p, got=got)


@pytest.mark.gpu
def test_gradient_against_differences(cuda):
    """The gradients' dot product with a direction is the forward's difference
    quotient along it, in fp32 residuals: central differences of step h are off
    by O(h^2); y, the weights and the gate are 16-bit, so the direction moves
    the residual alone and h * direction stays representable in fp32."""
    g = torch.Generator(device="cuda").manual_seed(5)
    p = make(4, 96, torch.bfloat16, torch.float32, "token", True, True)
    v = torch.randn((4, 96), generator=g, device="cuda")
    h = 2.0 ** -4

    def loss(r):
        q = dict(p, residual=r)
        f = mb.block_norm(q["residual"], q["y"], q["w_post"], q["w_pre"], q["gate"])
        return ((f.residual_out.double() * p["d_res"].double()).sum() + (f.normed.double() * p["d_normed"].double()).sum()), f

    _, f0 = loss(p["residual"])
    b = mb.block_norm_backward(p["d_res"], p["d_normed"], f0.residual_out, p["y"], p["w_post"], p["w_pre"], p["gate"])
    up, down = loss(p["residual"] + h * v)[0], loss(p["residual"] - h * v)[0]
    slope = float((b.d_residual.double() * v.double()).sum())
    # normed is bf16: each of its 384 values is off by at most half a step of about 1, times its gradient
    noise = 2 * float((p["d_normed"].double().abs() * f0.normed.double().abs()).sum()) * half_step(torch.bfloat16) / (2 * h)
    third = h * h * float((p["d_normed"].double().abs() * p["w_pre"].double().abs()).sum())  # |n'''| is of order 1 here
    assert abs(float(up - down) / (2 * h) - slope) <= noise + third


# ------------------------------------------------------------- refusals ----

def cpu(T=4, d=16, dtype=torch.bfloat16):
    return torch.zeros((T, d), dtype=dtype), torch.ones((d,), dtype=dtype)


def test_refusals():
    x, w = cpu()
    bad = [
        lambda: mb.block_norm(x),                                                  # nothing to do
        lambda: mb.block_norm(x, None, w_post=w, w_pre=w),                         # post norm without a block
        lambda: mb.block_norm(x, x, w_pre=w[:8]),                                  # weight of another width
        lambda: mb.block_norm(x, x.float(), w_pre=w),                              # types
        lambda: mb.block_norm(x.double(), x, w_pre=w),
        lambda: mb.block_norm(x, x, w_pre=w.half()),
        lambda: mb.block_norm(x, x, w_pre=w, gate=torch.ones((4, 2), dtype=x.dtype)),
        lambda: mb.block_norm(x, x, w_pre=w, gate=torch.ones((4, 1))),             # gate of another type
        lambda: mb.block_norm(x, x.T.contiguous().T, w_pre=w),                     # columns apart
        lambda: mb.block_norm(x, x[:1].expand(4, 16), w_pre=w),                    # rows on one another
        lambda: mb.block_norm(x[0], w_pre=w),
        lambda: mb.block_norm(x, x, w_pre=w),                                      # not on a GPU
        lambda: mb.block_norm_backward(None, None, x, x),
        lambda: mb.block_norm_backward(x, None, x, x, w_pre=w),
        lambda: mb.block_norm_backward(x, x, x, x),
        lambda: mb.block_norm_backward(x[:, :8], x, x, x, w_pre=w),
    ]
    for f in bad:
        with pytest.raises(mb.MoEB200Error) as e:
            f()
        assert e.value.status == mb.ERR_INVALID_ARG


def test_c_refusals():
    L = mb.lib()
    p = 0x10000

    def fwd(y=p, ys=16, r=p, rs=16, wo=p, wn=p, ga=None, form=0, eps=1e-6, T=4, d=16, dt=1, ro=p, no=p):
        return L.moe_b200_block_norm(y, ys, r, rs, 0, wo, wn, ga, form, 1.0, eps, T, d, dt, ro, no, None)

    assert fwd(T=0) == mb.OK
    assert fwd(T=-1) == fwd(d=0) == fwd(dt=5) == fwd(form=4, ga=p) == fwd(form=1) == fwd(ga=p) == mb.ERR_INVALID_ARG
    assert fwd(eps=-1.0) == fwd(eps=float("nan")) == fwd(r=None) == fwd(ro=None) == fwd(no=None) == mb.ERR_INVALID_ARG
    assert fwd(y=None) == fwd(y=None, wo=None, wn=None) == fwd(rs=15) == fwd(ys=8) == mb.ERR_INVALID_ARG
    assert fwd(d=16385, rs=1 << 20, ys=1 << 20) == mb.ERR_UNSUPPORTED
    need = L.moe_b200_block_norm_backward_workspace_bytes(4, 16)
    assert need > 0 and need % 256 == 0
    assert L.moe_b200_block_norm_backward_workspace_bytes(-1, 16) == 0

    def bwd(dr=p, dn=p, ro=p, y=p, wo=p, wn=p, out=p, dy=p, dwo=p, dwn=p, ws=p, nb=need, T=4):
        return L.moe_b200_block_norm_backward(dr, dn, ro, 16, 0, y, 16, wo, wn, None, 0, 1.0, 1e-6, T, 16, 1, out, dy, dwo,
                                              dwn, None, ws, nb, None)

    assert bwd(dn=None) == bwd(ro=None) == bwd(out=None) == bwd(dy=None) == bwd(dwo=None) == bwd(dwn=None) == mb.ERR_INVALID_ARG
    assert bwd(dr=None, wn=None) == bwd(ws=p + 16) == mb.ERR_INVALID_ARG
    assert bwd(ws=None) == bwd(nb=need - 256) == mb.ERR_WORKSPACE
