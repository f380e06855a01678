"""Host-side Python binding of libmoe_b200 (the sm_100a MoE packing library).

Mirrors the reference's packing operator interface (feiyang-cmu/15618-final,
include/moe/types.h:18-39 and include/moe/scatter.cuh:20-65):

  MoEParams, MoEBuffers, ScatterTimings   same fields and meaning
  make_scatter(name)                      "b200" -> B200Scatter; None for
                                          unknown names (src/scatter/factory.cu:17)
  B200Scatter.name() / workspace_bytes(p) / run(d_emb, d_asgn, d_wts, bufs, p, stream)

and adds functional entry points (pack, unpermute) over the same C ABI
(include/moe_b200.h).  Tensors are torch CUDA tensors; torch provides device
memory and streams only, every kernel is in libmoe_b200.so.  Where the
reference prints and exit(1)s on a bad shape or CUDA error
(include/moe/utils.cuh:14-22), this module raises MoEB200Error.

There is no CPU fallback: if the shared library is missing, importing the
library raises.
"""
from __future__ import annotations

import ctypes
import os
import sys
from dataclasses import dataclass
from typing import NamedTuple, Optional

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "lib", "libmoe_b200.so")

OK = 0
ERR_INVALID_ARG = 1
ERR_WORKSPACE = 2
ERR_UNSUPPORTED = 3
ERR_CUDA = 4
DEV_BAD_ASSIGNMENT = 0x10
DEV_WAIT_TIMEOUT = 0x20
DEV_BAD_WEIGHTS = 0x40
F16 = 0
BF16 = 1
MAX_EXPERTS = 1024
GATE_NONE, GATE_TOKEN, GATE_CHANNEL, GATE_FULL = 0, 1, 2, 3
ACT_NONE, ACT_SWIGLU = 0, 1


class MoEB200Error(RuntimeError):
    """A libmoe_b200 entry point returned an error status."""

    def __init__(self, status: int, msg: str):
        super().__init__(f"{msg} (status {status})")
        self.status = status


_lib = None


def lib() -> ctypes.CDLL:
    """Load libmoe_b200.so once; raise if it was not built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise MoEB200Error(ERR_CUDA, f"libmoe_b200.so not built at {LIB_PATH}; run __graft_entry__.build()")
    L = ctypes.CDLL(LIB_PATH)
    vp, sz, i32, cint = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int32, ctypes.c_int
    L.moe_b200_version.restype = cint
    L.moe_b200_status_string.restype = ctypes.c_char_p
    L.moe_b200_status_string.argtypes = [cint]
    L.moe_b200_last_error.restype = ctypes.c_char_p
    L.moe_b200_pack_workspace_bytes.restype = sz
    L.moe_b200_pack_workspace_bytes.argtypes = [cint, cint, cint]
    L.moe_b200_workspace_init.restype = cint
    L.moe_b200_workspace_init.argtypes = [vp, sz, vp]
    L.moe_b200_pack.restype = cint
    L.moe_b200_pack.argtypes = [vp, vp, vp, cint, cint, cint, cint,
                                vp, vp, vp, vp, vp, vp, vp, sz, vp]
    L.moe_b200_workspace_status.restype = cint
    L.moe_b200_workspace_status.argtypes = [vp, sz, vp, ctypes.POINTER(cint)]
    L.moe_b200_device_status.restype = cint
    L.moe_b200_device_status.argtypes = [vp, ctypes.POINTER(cint)]
    L.moe_b200_grouped_swiglu_gather.restype = cint
    L.moe_b200_grouped_swiglu_gather.argtypes = [vp, cint, vp, vp, vp, cint, cint, cint, cint, cint, vp, vp, cint,
                                                 vp, vp, vp]
    L.moe_b200_grouped_swiglu.restype = cint
    L.moe_b200_grouped_swiglu.argtypes = [vp, vp, vp, cint, cint, cint, cint, cint, vp, vp, cint, vp, vp, vp]
    L.moe_b200_grouped_ffn.restype = cint
    L.moe_b200_grouped_ffn.argtypes = [vp, vp, vp, cint, cint, cint, cint, cint, vp, vp, cint, vp, vp, vp]
    L.moe_b200_ffn_weights_from_reference.restype = cint
    L.moe_b200_ffn_weights_from_reference.argtypes = [vp, vp, cint, cint, cint, vp, vp, vp]
    L.moe_b200_router_weights_bytes.restype = sz
    L.moe_b200_router_weights_bytes.argtypes = [cint, cint, cint]
    L.moe_b200_router_prepare.restype = cint
    L.moe_b200_router_prepare.argtypes = [vp, cint, cint, cint, vp, vp]
    L.moe_b200_route.restype = cint
    L.moe_b200_route.argtypes = [vp, cint, cint, cint, cint, cint, vp, vp, vp, vp]
    L.moe_b200_ep_layout.restype = cint
    L.moe_b200_ep_layout.argtypes = [vp, cint, cint, cint, ctypes.POINTER(ctypes.c_int32), vp, vp, vp, vp, vp]
    u64 = ctypes.c_uint64
    L.moe_b200_ep_create.restype = cint
    L.moe_b200_ep_create.argtypes = [cint, cint, cint, cint, cint, cint, ctypes.POINTER(ctypes.c_int32), cint,
                                     ctypes.POINTER(vp)]
    L.moe_b200_ep_set_replicated.restype = cint
    L.moe_b200_ep_set_replicated.argtypes = [vp, ctypes.POINTER(ctypes.c_int32), cint]
    L.moe_b200_ep_local_experts.restype = cint
    L.moe_b200_ep_local_experts.argtypes = [vp, ctypes.POINTER(ctypes.c_int32)]
    L.moe_b200_ep_destroy.restype = cint
    L.moe_b200_ep_destroy.argtypes = [vp]
    L.moe_b200_ep_ipc_handle.restype = cint
    L.moe_b200_ep_ipc_handle.argtypes = [vp, vp]
    L.moe_b200_ep_connect.restype = cint
    L.moe_b200_ep_connect.argtypes = [vp, vp]
    L.moe_b200_ep_recv_rows.restype = vp
    L.moe_b200_ep_recv_rows.argtypes = [vp]
    L.moe_b200_ep_back_rows.restype = vp
    L.moe_b200_ep_back_rows.argtypes = [vp]
    L.moe_b200_ep_recv_capacity.restype = ctypes.c_int64
    L.moe_b200_ep_recv_capacity.argtypes = [vp]
    L.moe_b200_ep_dispatch.restype = cint
    L.moe_b200_ep_dispatch.argtypes = [vp, u64, vp, vp, vp, cint, vp, vp, vp, vp, vp, vp, sz, vp]
    L.moe_b200_ep_receive.restype = cint
    L.moe_b200_ep_receive.argtypes = [vp, u64, vp, vp, vp]
    L.moe_b200_ep_return_identity.restype = cint
    L.moe_b200_ep_return_identity.argtypes = [vp, u64, vp, vp]
    L.moe_b200_ep_ffn_return.restype = cint
    L.moe_b200_ep_ffn_return.argtypes = [vp, u64, vp, vp, cint, vp, vp, cint, vp, vp]
    L.moe_b200_ep_combine.restype = cint
    L.moe_b200_ep_combine.argtypes = [vp, u64, vp, vp, cint, cint, vp, vp]
    L.moe_b200_ep_step.restype = cint
    L.moe_b200_ep_step.argtypes = [vp, vp, vp, vp, cint, cint, vp, vp, cint, vp, vp, vp, vp, vp, vp, vp, sz, vp, vp]
    L.moe_b200_ep_epoch.restype = u64
    L.moe_b200_ep_epoch.argtypes = [vp]
    L.moe_b200_unpermute.restype = cint
    L.moe_b200_unpermute.argtypes = [vp, vp, vp, cint, cint, cint, cint, vp, vp]
    i64, f32 = ctypes.c_int64, ctypes.c_float
    L.moe_b200_block_norm.restype = cint
    L.moe_b200_block_norm.argtypes = [vp, i64, vp, i64, cint, vp, vp, vp, cint, f32, f32, cint, cint, cint, vp, vp, vp]
    L.moe_b200_block_norm_backward_workspace_bytes.restype = sz
    L.moe_b200_block_norm_backward_workspace_bytes.argtypes = [cint, cint]
    L.moe_b200_block_norm_backward.restype = cint
    L.moe_b200_block_norm_backward.argtypes = [vp, vp, vp, i64, cint, vp, i64, vp, vp, vp, cint, f32, f32, cint, cint,
                                               cint, vp, vp, vp, vp, vp, vp, sz, vp]
    for f in (L.moe_b200_grouped_mm, L.moe_b200_grouped_mm_dgrad):
        f.restype = cint
        f.argtypes = [vp, vp, vp, cint, cint, cint, cint, cint, vp, cint, vp, vp]
    L.moe_b200_grouped_mm_wgrad.restype = cint
    L.moe_b200_grouped_mm_wgrad.argtypes = [vp, vp, vp, cint, cint, cint, cint, cint, vp, vp]
    L.moe_b200_expert_linear_w4.restype = cint
    L.moe_b200_expert_linear_w4.argtypes = [vp, cint, vp, cint, cint, cint, cint, cint, vp, vp, vp, cint, cint, cint,
                                            vp, vp]
    _lib = L
    return L


def _check(status: int, what: str) -> None:
    if status != OK:
        L = lib()
        detail = L.moe_b200_last_error().decode() or L.moe_b200_status_string(status).decode()
        raise MoEB200Error(status, f"{what}: {detail}")


def _ptr(t) -> Optional[int]:
    if t is None:
        return None
    return t.data_ptr()


def _stream_handle(stream) -> Optional[int]:
    import torch
    if stream is None:
        stream = torch.cuda.current_stream()
    if isinstance(stream, int):
        return stream or None
    return stream.cuda_stream or None


def _other_stream(dev, stream):
    """`stream` (a torch stream or a raw handle) as a torch stream; None where
    it is the current one of `dev`."""
    import torch
    if stream is None:
        return None
    handle = _stream_handle(stream) or 0
    if handle == torch._C._cuda_getCurrentRawStream(dev.index):
        return None
    if not isinstance(stream, int):
        return stream
    return torch.cuda.ExternalStream(handle, device=dev) if handle else torch.cuda.default_stream(dev)


def _fresh(dev, stream, alloc):
    """alloc()'s tensors (or Nones), which a call will write on `stream`.
    Where that is another stream than the current one they are allocated on it,
    since memory that the current stream's earlier work still uses may be handed
    out to the current stream alone; and they are kept from reuse until the
    current stream, on which the caller goes on, is through with them too."""
    if stream is None:
        return alloc()
    import torch
    dev = torch.device(dev)
    if dev.index is None:
        dev = torch.device(dev.type, torch.cuda.current_device())
    other = _other_stream(dev, stream)
    if other is None:
        return alloc()
    with torch.cuda.stream(other):
        got = alloc()
    here = torch.cuda.current_stream(dev)
    for t in got:
        if t is not None:
            t.record_stream(here)
    return got


def _new(like, shape, dev, stream, dtype=None):
    """An empty tensor beside `like`, which a call will write on `stream`."""
    if stream is None:
        return like.new_empty(shape) if dtype is None else like.new_empty(shape, dtype=dtype)
    return _fresh(dev, stream, lambda: (like.new_empty(shape, dtype=dtype),))[0]


def _device_of(t):
    """The device that a call on this tensor runs on."""
    return t.device


def _on_device(dev, fn, *args):
    """fn(*args) with `dev` current."""
    torch = sys.modules["torch"]
    if torch._C._cuda_getDevice() == dev.index:
        return fn(*args)
    with torch.cuda.device(dev):
        return fn(*args)


def _enqueue(what, fn, dev, stream, *args):
    """Calls fn(*args, stream) with `dev` current (stream None: its current one)."""
    index = dev.index
    if index is None:
        raise MoEB200Error(ERR_INVALID_ARG, f"{what}: tensors must be on a CUDA device, got {dev}")
    cuda = sys.modules["torch"]._C  # (there are tensors, so it is loaded)
    handle = (cuda._cuda_getCurrentRawStream(index) or None) if stream is None else _stream_handle(stream)
    if cuda._cuda_getDevice() == index:
        status = fn(*args, handle)
    else:
        status = _on_device(dev, fn, *args, handle)
    if status != OK:
        _check(status, what)


# --------------------------------------------------------------------------
# The reference interface
# --------------------------------------------------------------------------

@dataclass
class MoEParams:
    """Problem sizes (reference include/moe/types.h:18-24)."""
    T: int
    K: int
    E: int
    d_model: int
    d_ffn: int = 0


@dataclass
class MoEBuffers:
    """Caller-owned device outputs + scratch (reference include/moe/types.h:28-39)."""
    packed: object
    packed_weights: object
    perm: object
    expert_count: object
    expert_start: object
    strategy_ws: object = None
    strategy_ws_bytes: int = 0


@dataclass
class ScatterTimings:
    """Per-stage times; 0 = not measured (reference include/moe/scatter.cuh:20-26)."""
    count_ms: float = 0.0
    prefix_ms: float = 0.0
    sort_ms: float = 0.0
    gather_ms: float = 0.0
    total_ms: float = 0.0


def allocate_buffers(p: MoEParams, device="cuda", dtype=None) -> MoEBuffers:
    """Allocate MoEBuffers the way the reference harnesses do
    (apps/bench_scatter.cu:98-113): expert_start has E+1 entries."""
    import torch
    dtype = dtype or torch.float16
    TK = p.T * p.K
    ws_bytes = pack_workspace_bytes(p.T, p.K, p.E)
    return MoEBuffers(
        packed=torch.empty((TK, p.d_model), dtype=dtype, device=device),
        packed_weights=torch.empty(TK, dtype=torch.float32, device=device),
        perm=torch.empty(TK, dtype=torch.int32, device=device),
        expert_count=torch.empty(p.E, dtype=torch.int32, device=device),
        expert_start=torch.empty(p.E + 1, dtype=torch.int32, device=device),
        strategy_ws=torch.empty(max(ws_bytes, 256), dtype=torch.uint8, device=device),
        strategy_ws_bytes=max(ws_bytes, 256),
    )


class B200Scatter:
    """The sm_100a packing strategy behind the reference's IScatter boundary."""

    def __init__(self):
        self._ws_key = None

    def name(self) -> str:
        return "b200"

    def workspace_bytes(self, p: MoEParams) -> int:
        return pack_workspace_bytes(p.T, p.K, p.E)

    def run(self, d_emb, d_asgn, d_wts, bufs: MoEBuffers, p: MoEParams, stream=None,
            slot_pos=None) -> ScatterTimings:
        dev = _device_of(d_emb)
        key = (_ptr(bufs.strategy_ws), bufs.strategy_ws_bytes, p.T, p.K, p.E)
        if key != self._ws_key:
            _enqueue("workspace_init", lib().moe_b200_workspace_init, dev, stream, _ptr(bufs.strategy_ws),
                     bufs.strategy_ws_bytes)
            self._ws_key = key
        _enqueue("pack", lib().moe_b200_pack, dev, stream,
                 _ptr(d_emb), _ptr(d_asgn), _ptr(d_wts), p.T, p.K, p.E, p.d_model,
                 _ptr(bufs.packed), _ptr(bufs.packed_weights), _ptr(bufs.perm),
                 _ptr(bufs.expert_count), _ptr(bufs.expert_start), _ptr(slot_pos),
                 _ptr(bufs.strategy_ws), bufs.strategy_ws_bytes)
        return ScatterTimings()


def make_scatter(name: str):
    """Factory (reference src/scatter/factory.cu:11-18): None for unknown names."""
    if name == "b200":
        return B200Scatter()
    return None


# --------------------------------------------------------------------------
# Functional API
# --------------------------------------------------------------------------

def pack_workspace_bytes(T: int, K: int, E: int) -> int:
    return int(lib().moe_b200_pack_workspace_bytes(T, K, E))


class PackResult(NamedTuple):
    packed: object
    packed_weights: object
    perm: object
    expert_count: object
    expert_start: object
    slot_pos: object


class Workspace:
    """A zero-filled packing workspace reused across calls (one per stream)."""

    def __init__(self, T: int, K: int, E: int, device="cuda", stream=None):
        import torch
        self.nbytes = max(pack_workspace_bytes(T, K, E), 256)
        self.buf, = _fresh(device, stream, lambda: (torch.empty(self.nbytes, dtype=torch.uint8, device=device),))
        self.shape = (T, K, E)
        _enqueue("workspace_init", lib().moe_b200_workspace_init, _device_of(self.buf), stream, self.buf.data_ptr(),
                 self.nbytes)

    def fits(self, T, K, E) -> bool:
        return pack_workspace_bytes(T, K, E) <= self.nbytes

    def device_status(self, stream=None) -> int:
        """Synchronise and return (and clear) the device condition bits."""
        import torch
        out = ctypes.c_int(0)
        with torch.cuda.device(_device_of(self.buf)):
            _check(lib().moe_b200_workspace_status(self.buf.data_ptr(), self.nbytes, _stream_handle(stream),
                                                   ctypes.byref(out)), "workspace_status")
        return out.value


def pack(emb, asgn, wts, E: int, workspace: Optional[Workspace] = None, out: Optional[PackResult] = None,
         stream=None, rows: bool = True) -> PackResult:
    """Stable pack of emb [T, d] (16-bit) by asgn [T, K] (int32); wts [T, K] fp32.
    rows=False: indices only (packed is None, no row copy)."""
    import torch
    T, d = emb.shape
    K = asgn.shape[1]
    TK = T * K
    dev = emb.device
    if workspace is None:
        workspace = Workspace(T, K, E, device=dev, stream=stream)
    if out is None:
        out = _fresh(dev, stream, lambda: PackResult(
            packed=torch.empty((TK, d), dtype=emb.dtype, device=dev) if rows else None,
            packed_weights=torch.empty(TK, dtype=torch.float32, device=dev) if wts is not None else None,
            perm=torch.empty(TK, dtype=torch.int32, device=dev),
            expert_count=torch.empty(E, dtype=torch.int32, device=dev),
            expert_start=torch.empty(E + 1, dtype=torch.int32, device=dev),
            slot_pos=torch.empty(TK, dtype=torch.int32, device=dev),
        ))
    _enqueue("pack", lib().moe_b200_pack, _device_of(emb), stream,
             _ptr(emb), _ptr(asgn), _ptr(wts), T, K, E, d,
             _ptr(out.packed), _ptr(out.packed_weights), _ptr(out.perm),
             _ptr(out.expert_count), _ptr(out.expert_start), _ptr(out.slot_pos),
             workspace.buf.data_ptr(), workspace.nbytes)
    return out


def device_status(stream=None) -> int:
    """Synchronise and return (and clear) the condition bits that workspace-less
    kernels (unpermute, grouped FFN) recorded on the current device."""
    out = ctypes.c_int(0)
    _check(lib().moe_b200_device_status(_stream_handle(stream), ctypes.byref(out)), "device_status")
    return out.value


def dtype_code(torch_dtype) -> int:
    import torch
    if torch_dtype == torch.float16:
        return F16
    if torch_dtype == torch.bfloat16:
        return BF16
    raise MoEB200Error(ERR_INVALID_ARG, f"unsupported dtype {torch_dtype}")


def unpermute(y, packed_weights, slot_pos, T: int, K: int, out=None, stream=None):
    """out[t] = round16(sum_k w[p] * y[p]), p = slot_pos[t*K + k]; fp32 accumulate."""
    import torch
    d = y.shape[1]
    if out is None:
        out, = _fresh(y.device, stream, lambda: (torch.empty((T, d), dtype=y.dtype, device=y.device),))
    _enqueue("unpermute", lib().moe_b200_unpermute, _device_of(y), stream, _ptr(y), _ptr(packed_weights), _ptr(slot_pos),
             T, K, d, dtype_code(y.dtype), _ptr(out))
    return out


def grouped_swiglu(x, seg_start, w_gate_up, w_down, seg_expert=None, h=None, y=None, stream=None,
                   row_token=None):
    """Grouped SwiGLU FFN over packed rows x [rows, d] (bf16/fp16).
    seg_start: int32 [nseg + 1] device offsets (e.g. expert_start from pack);
    w_gate_up [E, 2I, d], w_down [E, d, I].  Returns (h [rows, I], y [rows, d]).
    row_token (int32 [rows], e.g. perm from pack): x is then the token matrix
    [T, d] and packed row r is x[row_token[r]] (gathered, no packed copy)."""
    import torch
    if row_token is not None:
        T, d = x.shape
        rows = row_token.numel()
    else:
        rows, d = x.shape
    E, two_i, _ = w_gate_up.shape
    I = two_i // 2
    nseg = seg_start.numel() - 1
    if h is None:
        h, = _fresh(x.device, stream, lambda: (torch.empty((rows, I), dtype=x.dtype, device=x.device),))
    if y is None:
        y, = _fresh(x.device, stream, lambda: (torch.empty((rows, d), dtype=x.dtype, device=x.device),))
    if row_token is not None:
        _enqueue("grouped_swiglu_gather", lib().moe_b200_grouped_swiglu_gather, _device_of(x), stream, _ptr(x), T,
                 _ptr(row_token), _ptr(seg_start), _ptr(seg_expert), nseg, rows, d, I, E, _ptr(w_gate_up), _ptr(w_down),
                 dtype_code(x.dtype), _ptr(h), _ptr(y))
        return h, y
    _enqueue("grouped_swiglu", lib().moe_b200_grouped_swiglu, _device_of(x), stream, _ptr(x), _ptr(seg_start),
             _ptr(seg_expert), nseg, rows, d, I, E, _ptr(w_gate_up), _ptr(w_down), dtype_code(x.dtype), _ptr(h), _ptr(y))
    return h, y


def grouped_ffn(x, seg_start, w_up, w_down, seg_expert=None, mid=None, y=None, stream=None):
    """The reference's activation-free expert FFN, grouped, on packed rows
    x [rows, d]: mid = x . w_up[e]^T, y = mid . w_down[e]^T (fp32 accumulate,
    each rounded once).  w_up [E, F, d], w_down [E, d, F] (K-major; see
    ffn_weights_from_reference).  Returns (mid [rows, F], y [rows, d])."""
    import torch
    rows, d = x.shape
    E, F, _ = w_up.shape
    nseg = seg_start.numel() - 1
    if mid is None:
        mid, = _fresh(x.device, stream, lambda: (torch.empty((rows, F), dtype=x.dtype, device=x.device),))
    if y is None:
        y, = _fresh(x.device, stream, lambda: (torch.empty((rows, d), dtype=x.dtype, device=x.device),))
    _enqueue("grouped_ffn", lib().moe_b200_grouped_ffn, _device_of(x), stream, _ptr(x), _ptr(seg_start), _ptr(seg_expert),
             nseg, rows, d, F, E, _ptr(w_up), _ptr(w_down), dtype_code(x.dtype), _ptr(mid), _ptr(y))
    return mid, y


def ffn_weights_from_reference(w1, w2, stream=None):
    """The reference's expert weights W1 [E, d, F] / W2 [E, F, d] (row-major
    B operands, apps/bench_e2e.cu:281-292) in the layout grouped_ffn takes:
    (w_up [E, F, d], w_down [E, d, F]), transposed on the device."""
    import torch
    E, d, F = w1.shape
    # (a copy that contiguous() makes is read on `stream` too: made there)
    w_up, w_down, w1, w2 = _fresh(w1.device, stream, lambda: (
        torch.empty((E, F, d), dtype=w1.dtype, device=w1.device),
        torch.empty((E, d, F), dtype=w1.dtype, device=w1.device), w1.contiguous(), w2.contiguous()))
    _enqueue("ffn_weights_from_reference", lib().moe_b200_ffn_weights_from_reference, _device_of(w1), stream, _ptr(w1),
             _ptr(w2), E, d, F, _ptr(w_up), _ptr(w_down))
    return w_up, w_down


class RouterWeights:
    """Gate weights prepared for moe_b200_route: w_gate [d, E] fp32 on the
    device (row i = input feature i, as the reference's W_gate), split into
    16-bit pieces of the embeddings' dtype and transposed once."""

    def __init__(self, w_gate, dtype, stream=None):
        import torch
        if w_gate.dtype != torch.float32 or w_gate.dim() != 2:
            raise MoEB200Error(ERR_INVALID_ARG, "RouterWeights: w_gate must be a 2-D float32 tensor [d, E]")
        self.d, self.E = w_gate.shape
        self.dtype = dtype
        nbytes = lib().moe_b200_router_weights_bytes(self.d, self.E, dtype_code(dtype))
        if nbytes == 0:
            raise MoEB200Error(ERR_INVALID_ARG, f"RouterWeights: bad shape d={self.d} E={self.E}")
        self.buf, w_gate = _fresh(w_gate.device, stream, lambda: (
            torch.empty(nbytes, dtype=torch.uint8, device=w_gate.device), w_gate.contiguous()))
        _enqueue("router_prepare", lib().moe_b200_router_prepare, _device_of(w_gate), stream, _ptr(w_gate), self.d, self.E,
                 dtype_code(dtype), _ptr(self.buf))


def route(x, weights, K, out=None, stream=None):
    """Router on the tensor cores: x [T, d] (bf16/fp16), weights a
    RouterWeights of the same dtype.  Returns (assignments int32 [T, K],
    routing weights fp32 [T, K]): the K most probable experts of the softmax
    over all E logits, in descending probability, ties to the lower index."""
    import torch
    T, d = x.shape
    if out is None:
        out = _fresh(x.device, stream, lambda: (torch.empty((T, K), dtype=torch.int32, device=x.device),
                                                torch.empty((T, K), dtype=torch.float32, device=x.device)))
    _enqueue("route", lib().moe_b200_route, _device_of(x), stream, _ptr(x), T, d, weights.E, K, dtype_code(x.dtype),
             _ptr(weights.buf), _ptr(out[0]), _ptr(out[1]))
    return out


def ep_layout(all_counts, rank, expert_first, out=None, stream=None):
    """Device-side EP layout from all_counts [N, E] (int32, device).
    Returns (seg_start [N*L+1], seg_expert [N*L], send_counts [N], recv_counts [N])."""
    import torch
    N, E = all_counts.shape
    if not (0 <= rank < N) or len(expert_first) != N + 1:
        raise MoEB200Error(ERR_INVALID_ARG, f"ep_layout: rank {rank} / {len(expert_first)} bounds for {N} ranks")
    L = expert_first[rank + 1] - expert_first[rank]
    dev = all_counts.device
    if out is None:
        out = _fresh(dev, stream, lambda: (torch.empty(N * L + 1, dtype=torch.int32, device=dev),
                                           torch.empty(max(N * L, 1), dtype=torch.int32, device=dev),
                                           torch.empty(N, dtype=torch.int32, device=dev),
                                           torch.empty(N, dtype=torch.int32, device=dev)))
    first = (ctypes.c_int32 * (N + 1))(*expert_first)
    _enqueue("ep_layout", lib().moe_b200_ep_layout, _device_of(all_counts), stream, _ptr(all_counts), N, E, rank, first,
             _ptr(out[0]), _ptr(out[1]), _ptr(out[2]), _ptr(out[3]))
    return out


# --------------------------------------------------------------------------
# Norms around the block, expert products and their gradients, 4-bit weights
# --------------------------------------------------------------------------

def _refuse(what: str, why: str):
    raise MoEB200Error(ERR_INVALID_ARG, f"{what}: {why}")


def _rows(what, name, t, shape, dtype, strided=False):
    """Checks a tensor's shape, type and layout (strided: rows may lie apart)."""
    if t.shape == shape and t.dtype == dtype and t.is_contiguous():
        return
    if t.shape != shape or t.dtype != dtype:
        _refuse(what, f"{name} must be {dtype} {tuple(shape)}, got {t.dtype} {tuple(t.shape)}")
    if not (strided and t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= t.shape[1]):
        _refuse(what, f"{name} must be contiguous" + (" or have contiguous rows that do not overlap" if strided else ""))


def _same_device(what, *tensors):
    index = tensors[0].get_device()  # -1: the CPU
    for t in tensors:
        if t is not None and (t.get_device() != index or index < 0):
            _refuse(what, f"tensors must be on one CUDA device, got {tensors[0].device} and {t.device}")
    return tensors[0].device


def _row_stride(what, name, t, shape, dtype):
    """Elements from row to row of a tensor whose rows may lie apart."""
    if t.shape == shape and t.dtype == dtype and t.is_contiguous():
        return shape[1]
    _rows(what, name, t, shape, dtype, strided=True)
    return t.stride(0) if shape[0] > 1 else shape[1]


def _gate_form(what, gate, T, d, dtype):
    if gate is None:
        return GATE_NONE
    if gate.dtype != dtype or not gate.is_contiguous():
        _refuse(what, f"gate must be contiguous {dtype}")
    shape = tuple(gate.shape)
    if shape == (T, 1):  # a shape that broadcasts counts as broadcast, also where it is [T, d]
        return GATE_TOKEN
    if shape in ((1, d), (d,)):
        return GATE_CHANNEL
    if shape == (T, d):
        return GATE_FULL
    _refuse(what, f"gate must be ({T}, 1), (1, {d}), ({d},) or ({T}, {d}), got {shape}")


class BlockNormResult(NamedTuple):
    residual_out: object
    normed: object


class BlockNormGrads(NamedTuple):
    d_residual: object
    d_y: object
    d_w_post: object
    d_w_pre: object
    d_gate: object


def _check_block_norm(what, residual, y, w_post, w_pre, gate):
    """The checks both directions share: (T, d, dtype, its code, residual is
    fp32, gate form, row strides of residual and y)."""
    import torch
    if residual.dim() != 2:
        _refuse(what, "the residual must be [T, d]")
    some = y if y is not None else w_pre
    if some is None:
        _refuse(what, "nothing to do without y and w_pre")
    dtype = some.dtype
    code = BF16 if dtype == torch.bfloat16 else dtype_code(dtype)
    shape = residual.shape
    T, d = shape
    res_dtype = residual.dtype
    res32 = res_dtype == torch.float32
    if not res32 and res_dtype != dtype:
        _refuse(what, f"the residual must be {dtype} or float32, got {res_dtype}")
    res_stride, y_stride = d, 0
    if not residual.is_contiguous():
        res_stride = _row_stride(what, "the residual", residual, shape, res_dtype)
    if y is not None:
        y_stride = _row_stride(what, "y", y, shape, dtype)
        if w_post is not None:
            _rows(what, "w_post", w_post, (d,), dtype)
    elif w_post is not None or gate is not None:
        _refuse(what, "w_post and gate need y")
    if w_pre is not None:
        _rows(what, "w_pre", w_pre, (d,), dtype)
    form = GATE_NONE if gate is None else _gate_form(what, gate, T, d, dtype)
    return T, d, dtype, code, int(res32), form, res_stride, y_stride


def block_norm(residual, y=None, w_post=None, w_pre=None, gate=None, scale=1.0, eps=1e-6, out=None, stream=None):
    """Norms behind and before a block, fused with its gate and residual scale:
      z = rms(y) * w_post (w_post None: y);  residual_out = residual + scale * gate * z
      normed = rms(residual_out) * w_pre (w_pre None: None)
    residual [T, d] 16-bit or float32, y [T, d] 16-bit (None: residual_out is
    the residual), gate [T, 1], [1, d] / [d] or [T, d].  residual and y may be
    row-strided.  out: a BlockNormResult of contiguous tensors to write, each
    of its own or the rows of residual, y or a [T, d] gate of its width."""
    import torch
    T, d, dtype, code, res32, form, res_stride, y_stride = _check_block_norm("block_norm", residual, y, w_post, w_pre,
                                                                              gate)
    dev = _same_device("block_norm", residual, y, w_post, w_pre, gate)
    if out is None:
        like, plain = torch.empty_like, torch.contiguous_format

        def alloc():
            return BlockNormResult(
                like(residual, memory_format=plain) if y is not None else None,
                like(residual, dtype=dtype, memory_format=plain) if w_pre is not None else None)

        out = alloc() if stream is None else _fresh(dev, stream, alloc)
    else:
        if (out.residual_out is None) != (y is None) or (out.normed is None) != (w_pre is None):
            _refuse("block_norm", "out needs residual_out with y and normed with w_pre, and neither without")
        _same_device("block_norm", residual, *out)
        if y is not None:
            _rows("block_norm", "out.residual_out", out.residual_out, (T, d), residual.dtype)
        if w_pre is not None:
            _rows("block_norm", "out.normed", out.normed, (T, d), dtype)
    if T == 0:
        return out if y is not None else BlockNormResult(residual, out.normed)
    _enqueue("block_norm", lib().moe_b200_block_norm, dev, stream,
             _ptr(y), y_stride, _ptr(residual), res_stride, res32, _ptr(w_post), _ptr(w_pre), _ptr(gate), form, scale,
             eps, T, d, code, _ptr(out.residual_out), _ptr(out.normed))
    return out if y is not None else BlockNormResult(residual, out.normed)


def block_norm_backward(d_residual_out, d_normed, residual_out, y=None, w_post=None, w_pre=None, gate=None, scale=1.0,
                        eps=1e-6, stream=None):
    """Gradients of block_norm from those of its results (d_residual_out None:
    zero; d_normed None without w_pre) and its stored residual_out.  Returns
    BlockNormGrads: d_residual in the residual's type, d_y 16-bit, d_w_post and
    d_w_pre float32 [d], d_gate float32 [T, 1] or the gate's [1, d] / [d], or
    16-bit [T, d]."""
    import torch
    what = "block_norm_backward"
    T, d, dtype, code, res32, form, res_stride, y_stride = _check_block_norm(what, residual_out, y, w_post, w_pre, gate)
    if (d_normed is None) != (w_pre is None):
        _refuse(what, "d_normed and w_pre go together")
    if d_residual_out is None and w_pre is None:
        _refuse(what, "no gradient given")
    if d_residual_out is not None:
        _rows(what, "d_residual_out", d_residual_out, (T, d), residual_out.dtype)
    if d_normed is not None:
        _rows(what, "d_normed", d_normed, (T, d), dtype)
    dev = _same_device(what, residual_out, d_residual_out, d_normed, y, w_post, w_pre, gate)
    # of the tensors' device: the size follows its number of SMs
    nbytes = int(_on_device(dev, lib().moe_b200_block_norm_backward_workspace_bytes, T, d))

    like, plain = torch.empty_like, torch.contiguous_format
    f32 = torch.float32

    def alloc():
        return BlockNormGrads(
            like(residual_out, memory_format=plain),
            like(y, memory_format=plain) if y is not None else None,
            like(w_post, dtype=f32) if w_post is not None else None,
            like(w_pre, dtype=f32) if w_pre is not None else None,
            None if gate is None else like(gate) if form == GATE_FULL else like(gate, dtype=f32))

    got = alloc() if stream is None else _fresh(dev, stream, alloc)
    if T == 0:  # sums over no token
        with torch.cuda.stream(_other_stream(dev, stream)):
            for t in got[2:]:
                if t is not None:
                    t.zero_()
        return got
    ws = _new(residual_out, (max(nbytes, 256),), dev, stream, torch.uint8)
    _enqueue(what, lib().moe_b200_block_norm_backward, dev, stream,
             _ptr(d_residual_out), _ptr(d_normed), _ptr(residual_out), res_stride, res32, _ptr(y), y_stride,
             _ptr(w_post), _ptr(w_pre), _ptr(gate), form, scale, eps, T, d, code, _ptr(got.d_residual),
             _ptr(got.d_y), _ptr(got.d_w_post), _ptr(got.d_w_pre), _ptr(got.d_gate), _ptr(ws), nbytes)
    return got


def _grouped_mm(what, fn, rows_in, seg_start, w, seg_expert, out, stream, forward):
    import torch
    if rows_in.dim() != 2 or w.dim() != 3 or seg_start.dim() != 1 or seg_start.numel() < 2:
        _refuse(what, "rows must be 2-D, w [E, N, K] and seg_start [nseg + 1]")
    E, N, K = w.shape
    rows = rows_in.shape[0]
    width_in, width_out = (K, N) if forward else (N, K)
    nseg = seg_start.numel() - 1
    dtype = rows_in.dtype
    code = dtype_code(dtype)
    _rows(what, "rows", rows_in, (rows, width_in), dtype)
    _rows(what, "w", w, (E, N, K), dtype)
    _rows(what, "seg_start", seg_start, (nseg + 1,), torch.int32)
    if seg_expert is not None:
        _rows(what, "seg_expert", seg_expert, (nseg,), torch.int32)
    elif nseg > E:
        _refuse(what, f"{nseg} segments for {E} experts need seg_expert")
    dev = _same_device(what, rows_in, seg_start, w, seg_expert, out)
    if out is None:
        out = _new(rows_in, (rows, width_out), dev, stream)
    else:
        _rows(what, "out", out, (rows, width_out), dtype)
    _enqueue(what, fn, dev, stream, _ptr(rows_in), _ptr(seg_start), _ptr(seg_expert), nseg, rows, N, K, E,
             _ptr(w), code, _ptr(out))
    return out


def grouped_mm(x, seg_start, w, seg_expert=None, out=None, stream=None):
    """One product per expert: y[r] = w[e] . x[r] for the rows r of segment s
    (rows seg_start[s] .. seg_start[s+1] - 1, e = seg_expert[s] or s).
    x [rows, K], w [E, N, K] -> [rows, N]; rows outside every segment are not
    written."""
    return _grouped_mm("grouped_mm", lib().moe_b200_grouped_mm, x, seg_start, w, seg_expert, out, stream, True)


def grouped_mm_dgrad(dy, seg_start, w, seg_expert=None, out=None, stream=None):
    """Gradient of grouped_mm for its rows: dx[r] = w[e]^T . dy[r];
    dy [rows, N], w [E, N, K] -> [rows, K]."""
    return _grouped_mm("grouped_mm_dgrad", lib().moe_b200_grouped_mm_dgrad, dy, seg_start, w, seg_expert, out, stream,
                       False)


def grouped_mm_wgrad(dy, x, seg_start, out=None, stream=None):
    """Gradient of grouped_mm for its weights: dw[s] = sum over the segment's
    rows of dy[r] x[r]^T; dy [rows, N], x [rows, K] -> [nseg, N, K], zeros for
    empty segments (segments that share an expert are to be added up by the
    caller)."""
    import torch
    what = "grouped_mm_wgrad"
    if dy.dim() != 2 or x.dim() != 2 or seg_start.dim() != 1 or seg_start.numel() < 2:
        _refuse(what, "dy and x must be 2-D and seg_start [nseg + 1]")
    rows, N = dy.shape
    K = x.shape[1]
    nseg = seg_start.numel() - 1
    dtype = x.dtype
    code = dtype_code(dtype)
    _rows(what, "dy", dy, (rows, N), dtype)
    _rows(what, "x", x, (rows, K), dtype)
    _rows(what, "seg_start", seg_start, (nseg + 1,), torch.int32)
    dev = _same_device(what, x, dy, seg_start, out)
    if out is None:
        out = _new(x, (nseg, N, K), dev, stream)
    else:
        _rows(what, "out", out, (nseg, N, K), dtype)
    _enqueue(what, lib().moe_b200_grouped_mm_wgrad, dev, stream, _ptr(dy), _ptr(x), _ptr(seg_start), nseg, rows,
             N, K, code, _ptr(out))
    return out


def expert_linear_w4(x, asgn, w_q, w_scale, w_zero=None, act=None, out=None, stream=None):
    """Products of few tokens with 4-bit expert weights, slot (t, k) with
    expert asgn[t, k] (int32; -1: no expert, a row of zeros).
      x       [T, d], or [T, K, d] with a row of its own for each slot
      w_q     uint8 [E, N, d/2] (even column in the low half of a byte)
      w_scale [E, N, d/group] of x's type, group 32, 64 or 128
      w_zero  uint8 [E, N, d/group], None: 8
      act     None, or "swiglu": silu(y[:, :N/2]) * y[:, N/2:]
    Returns [T*K, N] (swiglu [T*K, N/2]); combine a down product's rows with
    unpermute and slot_pos = arange(T*K).  At most 4096 slots T*K and 1024
    experts; N a multiple of 8 (swiglu: 16)."""
    import torch
    what = "expert_linear_w4"
    if act not in (None, "swiglu"):
        _refuse(what, f"act must be None or 'swiglu', got {act!r}")
    if asgn.dim() != 2 or w_q.dim() != 3 or w_scale.dim() != 3 or x.dim() not in (2, 3):
        _refuse(what, "x must be [T, d] or [T, K, d], asgn [T, K], w_q and w_scale 3-D")
    T, K = asgn.shape
    E, N, half = w_q.shape
    d = 2 * half
    dtype = x.dtype
    code = dtype_code(dtype)
    _rows(what, "x", x, (T, d) if x.dim() == 2 else (T, K, d), dtype)
    _rows(what, "asgn", asgn, (T, K), torch.int32)
    _rows(what, "w_q", w_q, (E, N, half), torch.uint8)
    groups = w_scale.shape[2]
    if groups < 1 or d % groups != 0:
        _refuse(what, f"w_scale has {groups} groups for d={d}")
    _rows(what, "w_scale", w_scale, (E, N, groups), dtype)
    if w_zero is not None:
        _rows(what, "w_zero", w_zero, (E, N, groups), torch.uint8)
    n_out = N // 2 if act else N
    dev = _same_device(what, x, asgn, w_q, w_scale, w_zero, out)
    if out is None:
        out = _new(x, (T * K, n_out), dev, stream)
    else:
        _rows(what, "out", out, (T * K, n_out), dtype)
    _enqueue(what, lib().moe_b200_expert_linear_w4, dev, stream,
             _ptr(x), int(x.dim() == 3), _ptr(asgn), T, K, E, d, N, _ptr(w_q), _ptr(w_scale), _ptr(w_zero), d // groups,
             ACT_SWIGLU if act else ACT_NONE, code, _ptr(out))
    return out
