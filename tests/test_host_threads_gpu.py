"""C calls of one operator from several host threads at once, each thread with
sizes that ask for another amount of shared memory of the same kernel: every
call succeeds and gives the bits that it gives alone."""
import threading

import pytest
import torch

import moe_b200 as mb

pytestmark = pytest.mark.gpu
ROUNDS = 4000


def run_together(jobs):
    """Jobs: (function, its arguments without the stream, the tensors that it
    writes, the tensors that it reads), each in a thread and a stream of its own."""
    want = []
    for fn, args, out, _ in jobs:
        assert fn(*args, None) == mb.OK
        torch.cuda.synchronize()
        want.append([t.clone() for t in out])
        for t in out:
            t.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    start, failed, why = threading.Barrier(len(jobs)), [0] * len(jobs), set()

    def work(i):
        fn, args = jobs[i][:2]
        handle = streams[i].cuda_stream
        torch.cuda.set_device(0)
        start.wait()
        for _ in range(ROUNDS):
            if fn(*args, handle) != mb.OK:
                failed[i] += 1
                why.add(mb.lib().moe_b200_last_error())

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not any(failed), f"{failed} of {ROUNDS} calls failed: {why}"
    for (_, _, out, _), ref in zip(jobs, want):
        assert all(torch.equal(a, b) for a, b in zip(out, ref))
    assert mb.device_status() == 0


def rand(shape, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).bfloat16()


def ints(shape, top, seed, dtype=torch.int32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(0, top, shape, generator=g, device="cuda", dtype=dtype)


def empty(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, device="cuda", dtype=dtype)


def ptr(*tensors):
    return [t.data_ptr() for t in tensors]


@pytest.mark.parametrize("which", ["grouped_mm", "dgrad", "wgrad"])
def test_grouped_products(cuda, which):
    """Tables of 2 to 1024 segments, of which the last one has rows."""
    x, dy, w = rand((16, 64), 1), rand((16, 72), 2), rand((1024, 72, 64), 3, 0.05)

    def job(n):
        seg = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
        seg[-1] = 16
        if which == "wgrad":
            dw = empty(n, 72, 64)
            return mb.lib().moe_b200_grouped_mm_wgrad, (*ptr(dy, x, seg), n, 16, 72, 64, mb.BF16, *ptr(dw)), [dw], (seg, x, dy)
        fn, rows, out = ((mb.lib().moe_b200_grouped_mm, x, empty(16, 72)) if which == "grouped_mm" else
                         (mb.lib().moe_b200_grouped_mm_dgrad, dy, empty(16, 64)))
        return fn, (*ptr(rows, seg), None, n, 16, 72, 64, 1024, *ptr(w), mb.BF16, *ptr(out)), [out], (seg, rows, w)

    run_together([job(n) for n in (2, 1024 if which != "wgrad" else 64, 3, 700 if which != "wgrad" else 40)])


def test_4bit_products(cuda):
    def job(d, E):
        x, wq, ws, a = rand((3, d), d), ints((E, 32, d // 2), 256, d, torch.uint8), rand((E, 32, d // 32), 5, 0.01), ints((3, 2), E, 9)
        y = empty(6, 32)
        return (mb.lib().moe_b200_expert_linear_w4,
                (*ptr(x), 0, *ptr(a), 3, 2, E, d, 32, *ptr(wq, ws), None, 32, mb.ACT_NONE, mb.BF16, *ptr(y)), [y], (x, wq, ws, a))

    run_together([job(128, 4), job(2048, 4), job(256, 300), job(1024, 4)])


def test_norms(cuda):
    def job(T, d):
        y, r, w = rand((T, d), d), rand((T, d), d + 1), rand((d,), d + 2)
        out, n = empty(T, d), empty(T, d)
        return (mb.lib().moe_b200_block_norm,
                (*ptr(y), d, *ptr(r), d, 0, *ptr(w, w), None, mb.GATE_NONE, 1.0, 1e-6, T, d, mb.BF16, *ptr(out, n)), [out, n], (y, r, w))

    run_together([job(600, d) for d in (2816, 4096, 2816, 4096)])


def test_norm_gradients(cuda):
    def job(T, d):
        dr, dn, r, y, w = rand((T, d), 1), rand((T, d), 2), rand((T, d), 3), rand((T, d), 4), rand((d,), 5)
        d_r, d_y, d_post, d_pre = empty(T, d), empty(T, d), empty(d, dtype=torch.float32), empty(d, dtype=torch.float32)
        nbytes = mb.lib().moe_b200_block_norm_backward_workspace_bytes(T, d)
        ws = empty(nbytes, dtype=torch.uint8)
        return (mb.lib().moe_b200_block_norm_backward,
                (*ptr(dr, dn, r), d, 0, *ptr(y), d, *ptr(w, w), None, mb.GATE_NONE, 1.0, 1e-6, T, d, mb.BF16,
                 *ptr(d_r, d_y, d_post, d_pre), None, *ptr(ws), nbytes), [d_r, d_y, d_post, d_pre], (dr, dn, r, y, w, ws))

    run_together([job(40, d) for d in (2816, 4096, 2304, 4096)])


@pytest.mark.parametrize("op", ["pack", "ffn", "unpermute", "route"])
def test_layer(cuda, op):
    """The layer's own operators."""
    L = mb.lib()

    def job(T, d, E, K):
        x, g = rand((T, d), d), torch.Generator(device="cuda").manual_seed(d)
        asgn = torch.rand((T, E), generator=g, device="cuda").topk(K, dim=1).indices.to(torch.int32).contiguous()
        wts = torch.rand((T, K), generator=g, device="cuda")
        if op == "pack":
            nbytes = L.moe_b200_pack_workspace_bytes(T, K, E)
            ws, packed, pw = torch.zeros(nbytes, device="cuda", dtype=torch.uint8), empty(T * K, d), empty(T * K, dtype=torch.float32)
            idx = [empty(n, dtype=torch.int32) for n in (T * K, E, E + 1, T * K)]
            return (L.moe_b200_pack, (*ptr(x, asgn, wts), T, K, E, d, *ptr(packed, pw, *idx), *ptr(ws), nbytes), [packed, pw, *idx],
                    (x, asgn, wts, ws))
        if op == "route":
            r = mb.RouterWeights(torch.randn((d, E), generator=g, device="cuda") * d ** -0.5, torch.bfloat16)
            a, w = empty(T, K, dtype=torch.int32), empty(T, K, dtype=torch.float32)
            return L.moe_b200_route, (*ptr(x), T, d, E, K, mb.BF16, *ptr(r.buf), *ptr(a, w)), [a, w], (x, r)
        if op == "unpermute":
            y, pos, out = rand((T * K, d), 3), torch.randperm(T * K, generator=g, device="cuda").to(torch.int32), empty(T, d)
            return L.moe_b200_unpermute, (*ptr(y, wts, pos), T, K, d, mb.BF16, *ptr(out)), [out], (y, wts, pos)
        seg = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
        seg[-1] = T
        up, down, mid, y = rand((E, 32, 64), 4, 0.1), rand((E, 64, 32), 5, 0.1), empty(T, 32), empty(T, 64)
        x = rand((T, 64), 6)
        return (L.moe_b200_grouped_ffn, (*ptr(x, seg), None, E, T, 64, 32, E, *ptr(up, down), mb.BF16, *ptr(mid, y)), [mid, y],
                (x, seg, up, down))

    run_together([job(40, 256, 4, 1), job(40, 2048, 16, 4), job(40, 512, 100, 2), job(40, 1024, 128, 4)])


@pytest.mark.parametrize("op", ["grouped_mm", "dgrad", "wgrad", "w4", "norm", "norm_backward", "ffn", "route", "pack", "unpermute"])
def test_a_threads_first_use_of_the_gpu(cuda, op):
    """A call that is the first thing its host thread does on the device."""
    x, w, w2 = rand((16, 64), 1), rand((2, 64, 64), 2, 0.1), rand((2, 64, 64), 3, 0.1)
    one, seg, a = rand((64,), 4), torch.tensor([0, 7, 16], dtype=torch.int32, device="cuda"), ints((16, 1), 2, 5)
    wq, ws = ints((2, 64, 32), 256, 6, torch.uint8), rand((2, 64, 2), 7, 0.01)
    wts, pos = torch.ones(16, 1, device="cuda"), torch.arange(16, dtype=torch.int32, device="cuda")
    router, space = mb.RouterWeights(torch.randn(64, 8, device="cuda"), torch.bfloat16), mb.Workspace(16, 1, 2)
    calls = {
        "grouped_mm": lambda: mb.grouped_mm(x, seg, w),
        "dgrad": lambda: mb.grouped_mm_dgrad(x, seg, w),
        "wgrad": lambda: mb.grouped_mm_wgrad(x, x, seg),
        "w4": lambda: mb.expert_linear_w4(x, a, wq, ws),
        "norm": lambda: mb.block_norm(x, x, one, one).normed,
        "norm_backward": lambda: mb.block_norm_backward(x, x, x, x, one, one).d_y,
        "ffn": lambda: mb.grouped_ffn(x, seg, w, w2)[1],
        "route": lambda: mb.route(x, router, 2)[1],
        "pack": lambda: mb.pack(x, a, wts, 2, workspace=space).packed,
        "unpermute": lambda: mb.unpermute(x, wts, pos, 16, 1),
    }
    call, got = calls[op], []
    want = call()
    torch.cuda.synchronize()

    def work():
        try:
            got.append(call())
        except Exception as e:  # noqa: BLE001
            got.append(e)

    t = threading.Thread(target=work)
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert isinstance(got[0], torch.Tensor), got[0]
    assert torch.equal(got[0], want)
