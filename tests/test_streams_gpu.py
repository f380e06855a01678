"""Calls on another stream than the current one: what they allocate is memory
that no other stream still uses, and stays theirs until both streams are through
with it."""
import pytest
import torch

import moe_b200 as mb

pytestmark = pytest.mark.gpu

T, D = 4096, 2048  # results of 16 MB
SLEEP = 200_000_000  # clock cycles: about 0.1 s


def rand(shape, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).bfloat16()


def operators():
    x, y, w1 = rand((T, D), 1), rand((T, D), 2), rand((D,), 3)
    w, seg = rand((1, D, D), 4, 0.02), torch.tensor([0, T], dtype=torch.int32, device="cuda")
    wide = torch.tensor([0, 64, 128], dtype=torch.int32, device="cuda")
    a = torch.zeros((T, 1), dtype=torch.int32, device="cuda")
    xq, wq, ws = rand((T, 64), 5), torch.randint(0, 256, (1, D, 32), device="cuda", dtype=torch.uint8), rand((1, D, 2), 6, 0.01)
    return {"norm": lambda s: mb.block_norm(x, y, w1, w1, stream=s),
            "norm_backward": lambda s: mb.block_norm_backward(x, y, x, y, w1, w1, stream=s)[:2],
            "grouped_mm": lambda s: (mb.grouped_mm(x, seg, w, stream=s),),
            "dgrad": lambda s: (mb.grouped_mm_dgrad(x, seg, w, stream=s),),
            "wgrad": lambda s: (mb.grouped_mm_wgrad(x[:128], y[:128], wide, stream=s),),
            "w4": lambda s: (mb.expert_linear_w4(xq, a, wq, ws, stream=s),)}


def layer_operators():
    x, wts = rand((T, D), 1), torch.rand((T, 1), device="cuda")
    a = torch.randint(0, 4, (T, 1), device="cuda", dtype=torch.int32)
    up, down, seg = rand((1, D, D), 4, 0.02), rand((1, D, D), 5, 0.02), torch.tensor([0, T], dtype=torch.int32, device="cuda")
    gate_up, pos = rand((1, 2 * D, D), 6, 0.02), torch.arange(T, dtype=torch.int32, device="cuda")
    w_gate = torch.randn((D, 8), device="cuda")
    return {"pack": lambda s: mb.pack(x, a, wts, 4, stream=s)[:1],
            "ffn": lambda s: mb.grouped_ffn(x, seg, up, down, stream=s),
            "swiglu": lambda s: mb.grouped_swiglu(x, seg, gate_up, down, stream=s),
            "unpermute": lambda s: (mb.unpermute(x, wts, pos, T, 1, stream=s),),
            "weights": lambda s: mb.ffn_weights_from_reference(up, down, stream=s),
            "route": lambda s: mb.route(x, mb.RouterWeights(w_gate, torch.bfloat16, stream=s), 8, stream=s)}


@pytest.mark.parametrize("op", ["norm", "norm_backward", "grouped_mm", "dgrad", "wgrad", "w4",
                                "pack", "ffn", "swiglu", "unpermute", "weights", "route"])
@pytest.mark.parametrize("by_handle", [False, True])
def test_results_do_not_take_memory_that_the_current_stream_still_reads(cuda, op, by_handle):
    keep_what_is_read((operators() | layer_operators())[op], by_handle)


def keep_what_is_read(call, by_handle):
    side = torch.cuda.Stream()
    want = [t.clone() for t in call(None)]
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    # Tensors as large as the results, which the current stream reads 0.1 s from
    # now, and which are given back to the allocator meanwhile.
    sources = [torch.full_like(t, i + 1) for i, t in enumerate(want)]
    copies = [torch.empty_like(t) for t in want]
    torch.cuda.synchronize()
    torch.cuda._sleep(SLEEP)
    for a, b in zip(copies, sources):
        a.copy_(b)
    del b, sources
    got = call(side.cuda_stream if by_handle else side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    torch.cuda.synchronize()
    for i, c in enumerate(copies):
        assert (c == i + 1).all()


@pytest.mark.parametrize("op", ["norm", "norm_backward", "grouped_mm", "dgrad", "wgrad", "w4"])
def test_results_stay_until_both_streams_are_through(cuda, op):
    """The caller reads the results on the current stream and drops them; calls
    that follow on the other stream do not take their memory."""
    call = operators()[op]
    side = torch.cuda.Stream()
    want = [t.clone() for t in call(None)]
    torch.cuda.synchronize()
    got = call(side)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda._sleep(SLEEP)
    copies = [t.clone() for t in got]
    del got
    with torch.cuda.stream(side):
        for t in want:
            torch.zeros_like(t)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(copies, want))


@pytest.mark.parametrize("op", ["norm", "norm_backward", "grouped_mm", "dgrad", "wgrad", "w4"])
def test_another_stream_inside_a_capture(cuda, op):
    """Results allocated on a stream that has joined the capture belong to the graph."""
    call = operators()[op]
    side = torch.cuda.Stream()
    want = [t.clone() for t in call(None)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        side.wait_stream(torch.cuda.current_stream())
        got = call(side)
        torch.cuda.current_stream().wait_stream(side)
    others = [torch.full((64 << 20,), 7, dtype=torch.uint8, device="cuda") for _ in range(4)]
    with torch.cuda.stream(side):
        others += [torch.full((64 << 20,), 7, dtype=torch.uint8, device="cuda") for _ in range(4)]
    torch.cuda.synchronize()
    for t in got:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all((t == 7).all() for t in others)
