"""GPU numerics of the grouped products and their gradients against 64 bits,
element by element.

Tolerances: a product of two 16-bit numbers is exact in fp32; the tensor core
adds with at least the 24 bits of fp32 but may cut instead of round, so each of
the n additions of a sum is off by at most 2^-23 of the largest partial sum,
itself at most sum |a||b|.  Bound: half a step of the 16-bit result plus
n 2^-23 sum |a||b| (plus half the smallest fp16 step)."""
import numpy as np
import pytest
import torch

import moe_b200 as mb


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def assert_close(got, a, b, name):
    """got against a @ b in 64 bits."""
    a, b = a.double(), b.double()
    ref, mag = a @ b, a.abs() @ b.abs()
    n, h = a.shape[1], half_step(got.dtype)
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 1e-38
    bound = h * ref.abs() + (1 + h) * n * 2.0 ** -23 * mag + tiny
    err = (got.double() - ref).abs()
    assert (err <= bound).all(), f"{name}: worst {float((err / bound).max()):.3g} of the bound"


def make(counts, K, N, dtype, E=None, seed=0, extra=0, lead=0):
    """Rows of the segments between `lead` rows before and `extra` rows behind them."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = lead + int(sum(counts)) + extra
    E = E or len(counts)
    x = torch.randn((rows, K), generator=g, device="cuda").to(dtype)
    dy = torch.randn((rows, N), generator=g, device="cuda").to(dtype)
    w = (torch.randn((E, N, K), generator=g, device="cuda") * 0.05).to(dtype)
    seg = torch.tensor(lead + np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda")
    return x, dy, w, seg


def check(x, dy, w, seg, seg_expert=None):
    y = mb.grouped_mm(x, seg, w, seg_expert)
    dx = mb.grouped_mm_dgrad(dy, seg, w, seg_expert)
    dw = mb.grouped_mm_wgrad(dy, x, seg)
    assert mb.device_status() == 0
    ss = seg.tolist()
    for s in range(len(ss) - 1):
        e = s if seg_expert is None else int(seg_expert[s])
        lo, hi = ss[s], ss[s + 1]
        if hi > lo:
            assert_close(y[lo:hi], x[lo:hi], w[e].T, f"y of {s}")
            assert_close(dx[lo:hi], dy[lo:hi], w[e], f"dx of {s}")
            assert_close(dw[s], dy[lo:hi].T, x[lo:hi], f"dw of {s}")
        else:
            assert not dw[s].any()
    return y, dx, dw


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("counts,K,N", [
    ([1], 8, 8),                                # the smallest call
    ([0, 1, 0, 15, 16, 17, 0], 64, 64),         # segment ends inside and on 16-row steps, empty ends
    ([63, 64, 65, 127, 128, 129], 72, 136),     # around the 64-row and 128-row tiles; odd widths
    ([200, 0, 77, 300], 320, 264),              # one column past the 256-wide tile
    ([5, 900, 3], 1096, 712),
    ([2] * 40, 200, 24),                        # more segments than a scan step
])
def test_products_and_gradients(cuda, dtype, counts, K, N):
    check(*make(counts, K, N, dtype, seed=len(counts) + K))


@pytest.mark.gpu
def test_more_tiles_than_sms_and_long_sums(cuda):
    """Several tiles a CTA (accumulators alternate, pipeline wraps) and one hot expert."""
    check(*make([3000, 10, 0, 500, 40, 129, 1, 64], 512, 1032, torch.bfloat16, seed=2))


@pytest.mark.gpu
def test_most_segments(cuda):
    """1024 segments of 0 to 40 rows."""
    counts = np.random.default_rng(1).integers(0, 41, size=1024)
    check(*make(list(counts), 40, 72, torch.bfloat16, seed=6))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [8, 300, 2000, 9000])
def test_pair_single_and_few_row_forms(cuda, rows):
    """The tile forms (chosen by the rows a segment has on average and
    the number of tiles), each with segments far from the average."""
    check(*make([rows, 3 * rows, 1, 0, rows // 2], 264, 520, torch.float16, seed=rows))
    check(*make([5 * rows + 3], 200, 136, torch.bfloat16, seed=rows))


@pytest.mark.gpu
@pytest.mark.parametrize("hot", [33, 40, 64, 100, 700])
@pytest.mark.parametrize("K,N", [(64, 72), (200, 264), (1024, 512)])
def test_long_segments_among_many_short_ones(cuda, hot, K, N):
    """Few rows a segment on average, and segments of more rows than that form's tile has."""
    check(*make([7, 0, hot] + [3] * 60 + [hot - 1, 0], K, N, torch.bfloat16, seed=hot))


@pytest.mark.gpu
def test_every_segment_empty(cuda):
    x, dy, w, seg = make([0, 0, 0], 64, 48, torch.bfloat16, extra=5)
    out = torch.full((5, 48), 7.0, dtype=x.dtype, device="cuda")
    mb.grouped_mm(x, seg, w, out=out)
    assert (out == 7).all()
    assert not mb.grouped_mm_wgrad(dy, x, seg).any()


@pytest.mark.gpu
def test_no_rows(cuda):
    x, dy, w, seg = make([0, 0], 64, 48, torch.float16)
    assert mb.grouped_mm(x, seg, w).shape == (0, 48)
    assert mb.grouped_mm_dgrad(dy, seg, w).shape == (0, 64)
    assert not mb.grouped_mm_wgrad(dy, x, seg).any()


@pytest.mark.gpu
def test_expert_map_and_experts_out_of_range(cuda):
    x, dy, w, seg = make([50, 0, 130, 20, 64, 1], 96, 80, torch.bfloat16, E=3, seed=5)
    se = torch.tensor([1, 0, 1, 2, 0, 2], dtype=torch.int32, device="cuda")
    check(x, dy, w, seg, se)
    se[2], se[4] = 3, -1
    ss = seg.tolist()
    y, dx = mb.grouped_mm(x, seg, w, se), mb.grouped_mm_dgrad(dy, seg, w, se)
    for s in (2, 4):
        assert not y[ss[s]:ss[s + 1]].any() and not dx[ss[s]:ss[s + 1]].any()
    assert_close(y[ss[3]:ss[4]], x[ss[3]:ss[4]], w[2].T, "y of 3")


@pytest.mark.gpu
@pytest.mark.parametrize("counts,K,N", [
    ([9, 20, 7, 0, 12], 72, 136),                # 32-row tiles
    ([100, 40, 129, 64, 1], 72, 136),            # narrow tiles
    ([300, 260, 130, 0, 600] * 3, 72, 1544),     # 128 x 256 tiles in the forward
    ([300, 260, 130, 0, 600] * 3, 1544, 72),     # and in dgrad
    ([5000, 5000, 3000], 72, 1544),              # SM pairs, the same
    ([5000, 5000, 3000], 1544, 72),
])
def test_rows_of_experts_out_of_range_may_hold_anything(cuda, counts, K, N):
    """A segment whose expert is outside [0, E) gives zeros whatever its rows
    hold (padding: NaN, infinities), and its neighbours are not touched."""
    n = len(counts)
    x, dy, w, seg = make(counts, K, N, torch.bfloat16, E=2, seed=n)
    ss = seg.tolist()
    for bad in (2, -1, 2 ** 31 - 1, -2 ** 31):
        experts = [s % 2 for s in range(n)]
        out = [0, n - 1]
        for i, s in enumerate(out):
            experts[s] = bad
            x[ss[s]:ss[s + 1]] = float("nan") if i else float("inf")
            dy[ss[s]:ss[s + 1]] = float("-inf") if i else float("nan")
        se = torch.tensor(experts, dtype=torch.int32, device="cuda")
        y, dx = mb.grouped_mm(x, seg, w, se), mb.grouped_mm_dgrad(dy, seg, w, se)
        assert mb.device_status() == 0
        for s in range(n):
            lo, hi = ss[s], ss[s + 1]
            if s in out:
                assert (y[lo:hi] == 0).all() and (dx[lo:hi] == 0).all()
            elif hi > lo:
                assert_close(y[lo:hi], x[lo:hi], w[experts[s]].T, f"y of {s}")
                assert_close(dx[lo:hi], dy[lo:hi], w[experts[s]], f"dx of {s}")


@pytest.mark.gpu
def test_rows_outside_the_segments(cuda):
    """Rows before and behind the segments: not written by the forward and
    dgrad, and what they hold (NaN here) reaches no sum of wgrad."""
    x, dy, w, seg = make([33, 7, 100], 128, 72, torch.bfloat16, extra=50, lead=9)
    lo, hi = int(seg[0]), int(seg[-1])
    for t in (x, dy):
        t[:lo] = float("nan")
        t[hi:] = float("inf")
    y = torch.full((x.shape[0], 72), 3.0, dtype=x.dtype, device="cuda")
    dx = torch.full((x.shape[0], 128), 3.0, dtype=x.dtype, device="cuda")
    mb.grouped_mm(x, seg, w, out=y)
    mb.grouped_mm_dgrad(dy, seg, w, out=dx)
    dw = mb.grouped_mm_wgrad(dy, x, seg)
    for t in (y, dx):
        assert (t[:lo] == 3).all() and (t[hi:] == 3).all() and torch.isfinite(t).all()
    ss = seg.tolist()
    for s in range(3):
        assert_close(dw[s], dy[ss[s]:ss[s + 1]].T, x[ss[s]:ss[s + 1]], f"dw of {s}")


@pytest.mark.gpu
def test_infinities_stay_with_their_expert(cuda):
    """A weight of infinity in one expert changes no other expert's rows, also
    where the reduced length ends inside a tile."""
    x, dy, w, seg = make([40, 40, 40], 72, 88, torch.bfloat16, seed=3)
    want = [t.clone() for t in (mb.grouped_mm(x, seg, w), mb.grouped_mm_dgrad(dy, seg, w))]
    w[1] = float("inf")
    got = mb.grouped_mm(x, seg, w), mb.grouped_mm_dgrad(dy, seg, w)
    for a, b in zip(got, want):
        assert torch.equal(a[:40], b[:40]) and torch.equal(a[80:], b[80:])


@pytest.mark.gpu
def test_offsets_outside_the_rows_are_held_inside(cuda):
    x, dy, w, seg = make([30, 30], 64, 64, torch.float16)
    want = mb.grouped_mm(x, seg, w)
    bad = torch.tensor([-100, 30, 1 << 30], dtype=torch.int32, device="cuda")
    assert torch.equal(mb.grouped_mm(x, bad, w), want)
    assert torch.equal(mb.grouped_mm_wgrad(dy, x, bad), mb.grouped_mm_wgrad(dy, x, seg))
    assert mb.device_status() == 0


@pytest.mark.gpu
def test_offsets_that_fall_are_held_ascending(cuda):
    """A start below an earlier one counts as that one, also 32 segments later."""
    counts = [7, 0, 40] + [3] * 40
    x, dy, w, seg = make(counts, 64, 72, torch.bfloat16)
    bad = seg.clone()
    bad[2] = 5        # inside segment 0: segment 1 is empty, segment 2 begins at 7 all the same
    seg[35] = seg[34]
    bad[35] = 0       # far back: segment 34 is empty and 35 begins where it did
    for got, want in ((mb.grouped_mm(x, bad, w), mb.grouped_mm(x, seg, w)),
                      (mb.grouped_mm_dgrad(dy, bad, w), mb.grouped_mm_dgrad(dy, seg, w)),
                      (mb.grouped_mm_wgrad(dy, x, bad), mb.grouped_mm_wgrad(dy, x, seg))):
        assert torch.equal(got, want)
    assert mb.device_status() == 0


@pytest.mark.gpu
def test_offsets_past_32_bits(cuda):
    """Rows and weights whose element offsets pass 2^31."""
    rows, K, N = 270000, 8192, 64
    x = torch.zeros((rows, K), dtype=torch.bfloat16, device="cuda")
    x[-100:] = torch.randn((100, K), device="cuda").bfloat16()
    w = (torch.randn((2, N, K), device="cuda") * 0.02).bfloat16()
    seg = torch.tensor([rows - 100, rows - 60, rows], dtype=torch.int32, device="cuda")
    y = mb.grouped_mm(x, seg, w)
    assert_close(y[-100:-60], x[-100:-60], w[0].T, "y")
    assert_close(y[-60:], x[-60:], w[1].T, "y")
    dy = torch.zeros((rows, N), dtype=torch.bfloat16, device="cuda")
    dy[-100:] = torch.randn((100, N), device="cuda").bfloat16()
    dx = mb.grouped_mm_dgrad(dy, seg, w, out=x.clone())
    assert_close(dx[-60:], dy[-60:], w[1], "dx")
    assert_close(mb.grouped_mm_wgrad(dy, x, seg)[1], dy[-60:].T, x[-60:], "dw")
    del x, dx
    E, N, K = 280, 2048, 4096  # 2.3e9 weights
    w = torch.zeros((E, N, K), dtype=torch.bfloat16, device="cuda")
    w[-1] = (torch.randn((N, K), device="cuda") * 0.02).bfloat16()
    se = torch.tensor([E - 1], dtype=torch.int32, device="cuda")
    seg = torch.tensor([0, 20], dtype=torch.int32, device="cuda")
    x = torch.randn((20, K), device="cuda").bfloat16()
    assert_close(mb.grouped_mm(x, seg, w, se), x, w[-1].T, "y")
    dy = torch.randn((20, N), device="cuda").bfloat16()
    assert_close(mb.grouped_mm_dgrad(dy, seg, w, se), dy, w[-1], "dx")


@pytest.mark.gpu
def test_sums_that_take_longer_than_a_wait(cuda):
    """One segment of 450 million rows: a tile takes 2.5 s, longer than a wait
    without regard to the sum's length.  All rows but the first and last 2000 are
    zeros, which add nothing, so the tolerance is that of 4000 rows."""
    rows, n = 450_000_000, 2000
    dy, x = (torch.zeros((rows, 8), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    g = torch.Generator(device="cuda").manual_seed(3)
    for t in (dy, x):
        for at in (slice(0, n), slice(rows - n, rows)):
            t[at] = torch.randn((n, 8), generator=g, device="cuda").bfloat16()
    dw = mb.grouped_mm_wgrad(dy, x, torch.tensor([0, rows], dtype=torch.int32, device="cuda"))
    assert mb.device_status() == 0
    ends = [torch.cat([t[:n], t[rows - n:]]) for t in (dy, x)]
    assert_close(dw[0], ends[0].T, ends[1], "dw")


@pytest.mark.gpu
def test_matches_the_two_product_ffn(cuda):
    """Two grouped products are the plain FFN, bit for bit."""
    x, _, w_up, seg = make([100, 0, 300, 17], 128, 96, torch.bfloat16)
    w_down = (torch.randn((4, 128, 96), device="cuda") * 0.05).bfloat16()
    mid, y = mb.grouped_ffn(x, seg, w_up, w_down)
    mine = mb.grouped_mm(x, seg, w_up)
    assert torch.equal(mine, mid) and torch.equal(mb.grouped_mm(mine, seg, w_down), y)


@pytest.mark.gpu
def test_streams_and_graphs(cuda):
    x, dy, w, seg = make([100, 20, 300], 256, 128, torch.bfloat16)
    want = mb.grouped_mm(x, seg, w), mb.grouped_mm_dgrad(dy, seg, w), mb.grouped_mm_wgrad(dy, x, seg)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (s1, s2):
        s.wait_stream(torch.cuda.current_stream())
    got = [(mb.grouped_mm(x, seg, w, stream=s), mb.grouped_mm_dgrad(dy, seg, w, stream=s), mb.grouped_mm_wgrad(dy, x, seg, stream=s))
           for s in (s1, s2, s1, s2)]
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = mb.grouped_mm(x, seg, w), mb.grouped_mm_dgrad(dy, seg, w), mb.grouped_mm_wgrad(dy, x, seg)
    seg.copy_(torch.tensor([0, 250, 251, 420], dtype=torch.int32))
    graph.replay()
    fresh = mb.grouped_mm(x, seg, w), mb.grouped_mm_dgrad(dy, seg, w), mb.grouped_mm_wgrad(dy, x, seg)
    assert all(torch.equal(a, b) for a, b in zip(again, fresh))
    assert mb.device_status() == 0


@pytest.mark.gpu
def test_result_on_the_rows_is_refused(cuda):
    """N = K: the shapes would allow it, but other tiles still read the rows."""
    x, dy, w, seg = make([30, 50], 64, 64, torch.bfloat16)
    for f in (lambda: mb.grouped_mm(x, seg, w, out=x), lambda: mb.grouped_mm_dgrad(dy, seg, w, out=dy),
              lambda: mb.grouped_mm_wgrad(w.view(128, 64), w.view(128, 64), seg, out=w)):
        with pytest.raises(mb.MoEB200Error, match="overlaps"):
            f()


# ------------------------------------------------------------- refusals ----

def test_refusals():
    x, dy = torch.zeros((4, 16)).half(), torch.zeros((4, 24)).half()
    w, seg = torch.zeros((2, 24, 16)).half(), torch.zeros(3, dtype=torch.int32)
    bad = [
        lambda: mb.grouped_mm(x, seg, w[:, :, :8]),
        lambda: mb.grouped_mm(x, seg.long(), w),
        lambda: mb.grouped_mm(x, seg[:1], w),
        lambda: mb.grouped_mm(x, torch.zeros(4, dtype=torch.int32), w),           # more segments than experts
        lambda: mb.grouped_mm(x, seg, w, seg_expert=torch.zeros(3, dtype=torch.int32)),
        lambda: mb.grouped_mm(x.float(), seg, w.float()),
        lambda: mb.grouped_mm(x, seg, w.bfloat16()),
        lambda: mb.grouped_mm(x, seg, w.transpose(1, 2).contiguous().transpose(1, 2)),
        lambda: mb.grouped_mm(x, seg, w, out=x),
        lambda: mb.grouped_mm_dgrad(x, seg, w),
        lambda: mb.grouped_mm_wgrad(dy[:3], x, seg),
        lambda: mb.grouped_mm_wgrad(dy.bfloat16(), x, seg),
        lambda: mb.grouped_mm(x, seg, w),                                         # not on a GPU
    ]
    for f in bad:
        with pytest.raises(mb.MoEB200Error) as e:
            f()
        assert e.value.status == mb.ERR_INVALID_ARG


def test_c_refusals():
    L = mb.lib()
    p = 0x10000

    def fwd(fn=L.moe_b200_grouped_mm, x=p, seg=p, nseg=2, rows=4, N=16, K=16, E=2, w=p, dt=1, y=p):
        return fn(x, seg, None, nseg, rows, N, K, E, w, dt, y, None)

    for fn in (L.moe_b200_grouped_mm, L.moe_b200_grouped_mm_dgrad):
        assert fwd(fn, rows=0) == mb.OK
        assert fwd(fn, rows=-1) == fwd(fn, nseg=0) == fwd(fn, N=0) == fwd(fn, K=0) == fwd(fn, E=0) == mb.ERR_INVALID_ARG
        assert fwd(fn, dt=3) == fwd(fn, x=None) == fwd(fn, seg=None) == fwd(fn, w=None) == fwd(fn, y=None) == mb.ERR_INVALID_ARG
        assert fwd(fn, x=p + 2) == fwd(fn, y=p + 8) == mb.ERR_INVALID_ARG
        assert fwd(fn, N=20) == fwd(fn, K=12) == fwd(fn, nseg=1025) == mb.ERR_UNSUPPORTED
    wg = L.moe_b200_grouped_mm_wgrad
    assert wg(p, None, p, 2, 4, 16, 16, 1, p, None) == wg(p, p, p, 2, 4, 16, 16, 1, None, None) == mb.ERR_INVALID_ARG
    assert wg(p, p, p, 2, 4, 16, 12, 1, p, None) == mb.ERR_UNSUPPORTED
