"""Host-side mirror of the reference's `strix::kernels` launchers for the MoE path, over the C ABI.

Same function names, argument order and meaning as kernels/moe_router.hpp, kernels/moe_grouped.hpp,
kernels/linear_q4.hpp, kernels/linear_q8.hpp and kernels/swiglu.hpp; a failed precondition raises `Error` (the
reference throws strix::Error) carrying the library's message.  Tensors are torch CUDA tensors used purely as device
memory: BF16 activations may be passed as torch.bfloat16 or as raw uint16/int16 bit tensors.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import enum
import struct
from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib


class Error(RuntimeError):
    """A failed precondition or launch; the reference's strix::Error (common/check.hpp:29-32)."""

    def __init__(self, code: int, message: str):
        super().__init__(message)
        self.code = code


class GpuFatalError(Error):
    """A sticky CUDA error: the context is gone (common/check.hpp:36-39)."""


class Act(enum.IntEnum):  # kernels/norm.hpp:20
    F32 = 0
    BF16 = 1
    F16_STAGED = 2  # not in the reference: F16 laid out by stage_f16 for a tensor-core operand
    F16_TILED = 3   # not in the reference: the tile-blocked form made by stage_f16_tiles


class MoeMath(enum.IntEnum):  # kernels/moe_grouped.hpp:39
    F32 = 0
    WmmaBf16 = 1
    WmmaF16 = 2
    WmmaF16Narrow = 3
    WmmaF16Wide = 4
    WmmaF16Wide256 = 5
    WmmaF16F32Partials = 6  # not in the reference: WmmaF16 with the combine's per-slot dots kept in FP32


LAUNCHES = 0  # kernels of this library launched through this module (the benchmark's gpu_launches)


def _count(n: int = 1) -> None:
    global LAUNCHES
    LAUNCHES += n


def _check(rc: int) -> None:
    _count()
    if rc != 0:
        msg = _lib.load().sxb_last_error().decode()
        raise (GpuFatalError if rc == 3 else Error)(rc, msg)


def _ptr(t) -> Optional[int]:
    if t is None:
        return None
    if isinstance(t, int):
        return t
    if not t.is_cuda:
        raise Error(1, "strixite_b200.kernels: tensors must live on a CUDA device (no CPU path exists)")
    return t.data_ptr()


def _stream(stream) -> int:
    if stream is None:
        if torch.cuda.is_initialized():  # the handle itself: the Stream object around it costs 3 us a call, a fifth of a one-token pass's host time
            return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())
        return torch.cuda.current_stream().cuda_stream
    return stream if isinstance(stream, int) else stream.cuda_stream


def _within(stream, device):
    """The context in which what a call allocates, clears and reads itself is ordered with the kernels that it gives to `stream`."""
    if stream is None or device.type != "cuda":
        return contextlib.nullcontext()
    if isinstance(stream, int):
        stream = torch.cuda.ExternalStream(stream, device) if stream else torch.cuda.default_stream(device)
    return torch.cuda.stream(stream)


def _handed(stream, *tensors):
    """What was allocated within `stream` goes to the caller, whose current stream may still use it when it is let go."""
    if stream is not None and tensors[0].is_cuda:
        for t in tensors:
            t.record_stream(torch.cuda.current_stream(t.device))


@dataclass
class QDeviceView:
    """A quantized matrix on the device: Q4DeviceView / Q8DeviceView (runtime/q4_device.hpp:14-19) plus its bit width."""

    q: torch.Tensor       # uint8 [N, K/2] (Q4) or [N, K] (Q8)
    scale: torch.Tensor   # BF16 bits [N, K/G]
    minv: torch.Tensor    # BF16 bits [N, K/G]
    N: int
    K: int
    G: int
    bits: int = 4

    def c(self) -> _lib.SxbQView:
        return _lib.SxbQView(self.q.data_ptr(), self.scale.data_ptr(), self.minv.data_ptr(), self.N, self.K, self.G)

    def bytes(self) -> int:
        return self.q.numel() + 2 * self.scale.numel() + 2 * self.minv.numel()

    def rows(self, lo: int, hi: int) -> "QDeviceView":
        """The view of rows [lo, hi) (e.g. one rank's experts of a stacked matrix)."""
        return QDeviceView(self.q[lo:hi], self.scale[lo:hi], self.minv[lo:hi], hi - lo, self.K, self.G, self.bits)


class QRawView:
    """A quantized matrix given by raw device pointers (e.g. a view into a loaded strixw file): the same interface as
    QDeviceView for the launchers."""

    def __init__(self, view: "_lib.SxbQView", bits: int, keepalive=None):
        self.view, self.bits, self.keepalive = view, bits, keepalive
        self.N, self.K, self.G = view.N, view.K, view.G

    def c(self) -> "_lib.SxbQView":
        return self.view

    def bytes(self) -> int:
        return self.N * self.K * self.bits // 8 + 4 * self.N * (self.K // self.G)


def _b(w: QDeviceView) -> str:
    if w.bits not in (4, 8):
        raise Error(1, f"experts have {w.bits} bits, expected 4 or 8")
    return f"q{w.bits}"


# ---- kernels/moe_router.hpp -----------------------------------------------------------------------------------

def moe_router(logits, ld, M, E, k, shared_logit, shared_ld, shared_id, ids, coef, act, err, stream=None):
    _check(_lib.load().sxb_moe_router(_ptr(logits), ld, M, E, k, _ptr(shared_logit), shared_ld, shared_id, _ptr(ids),
                                      _ptr(coef), int(act), _ptr(err), _stream(stream)))


def check_router_error(err, what: str):
    _check(_lib.load().sxb_check_router_error(_ptr(err), what.encode()))


def report_router_error(e, what: str):
    _check(_lib.load().sxb_report_router_error((C.c_uint32 * 3)(*[int(v) for v in e]), what.encode()))


def moe_shared_add(y, s, gate_logit, gate_ld, M, N, gate_index, act, err, stream=None):
    _check(_lib.load().sxb_moe_shared_add(_ptr(y), _ptr(s), _ptr(gate_logit), gate_ld, M, N, gate_index, int(act),
                                          _ptr(err), _stream(stream)))


def moe_shared_add_inject(y, s, gate_logit, gate_ld, M, N, gate_index, x, w_in, H, act, err, stream=None):
    _check(_lib.load().sxb_moe_shared_add_inject(_ptr(y), _ptr(s), _ptr(gate_logit), gate_ld, M, N, gate_index, _ptr(x),
                                                 _ptr(w_in), H, int(act), _ptr(err), _stream(stream)))


# ---- kernels/linear.hpp, kernels/linear_wmma.hpp: the router-logits projection; the residual add ----------------

def linear_bf16w(x, w, y, M, N, K, act, out_act=None, stream=None):
    _check(_lib.load().sxb_linear_bf16w(_ptr(x), _ptr(w), _ptr(y), M, N, K, int(act), int(act if out_act is None else out_act),
                                        _stream(stream)))


def _w_act(w) -> int:
    return int(Act.F32 if w.dtype == torch.float32 else Act.BF16)


def router_logits(x, w, bias, logits, stream=None):
    """logits [M, ld] FP32 = x [M, K] BF16 * w [N, K]^T (FP32 or BF16) + bias [N]: the streaming (decode) form."""
    M, K = x.shape
    N = w.shape[0]
    _check(_lib.load().sxb_router_logits(_ptr(x), _ptr(w), _w_act(w), _ptr(bias), M, N, K, _ptr(logits), logits.stride(0),
                                         _stream(stream)))


@dataclass
class RouterPlanes:
    """A router weight prepared for the tensor-core projection: `planes` BF16 planes [planes][Npad][K]."""

    data: torch.Tensor
    planes: int
    N: int
    K: int


def router_prepare(w: torch.Tensor, planes: Optional[int] = None, stream=None) -> RouterPlanes:
    """Splits w [N, K] (FP32: 3 planes carry every bit of it, 2 planes 16 bits; BF16: 1 plane) once, at load time."""
    N, K = w.shape
    if planes is None:
        planes = 3 if w.dtype == torch.float32 else 1
    nbytes = _lib.load().sxb_router_planes_bytes(N, K, planes)
    if nbytes == 0:
        _check(1)
    data = torch.empty(nbytes // 2, dtype=torch.int16, device=w.device)
    _check(_lib.load().sxb_router_prepare(_ptr(w), _w_act(w), N, K, planes, _ptr(data), _stream(stream)))
    return RouterPlanes(data, planes, N, K)


def router_logits_wmma(x, rp: RouterPlanes, bias, logits, stream=None):
    """The same projection on the tcgen05 tensor cores (prefill)."""
    M = x.shape[0]
    _check(_lib.load().sxb_router_logits_wmma(_ptr(x), _ptr(rp.data), rp.planes, _ptr(bias), M, rp.N, rp.K, _ptr(logits),
                                              logits.stride(0), _stream(stream)))


def residual_add(x, y, out, stream=None):
    """out = bf16(x + y); x, out BF16 (out may be x), y FP32 or BF16."""
    _check(_lib.load().sxb_residual_add(_ptr(x), _ptr(y), int(Act.F32 if y.dtype == torch.float32 else Act.BF16), _ptr(out),
                                        x.numel(), _stream(stream)))


def check_dense_status(what: str):
    _check(_lib.load().sxb_check_dense_status(what.encode()))


def set_wait_limit(ns: int):
    _check(_lib.load().sxb_set_wait_limit(int(ns)))


def linear_qw_wmma(x, w: QDeviceView, y, M, act, out_act=None, stream=None):
    fn = getattr(_lib.load(), f"sxb_linear_{_b(w)}_wmma")
    _check(fn(_ptr(x), C.byref(w.c()), _ptr(y), M, int(act), int(Act.BF16 if out_act is None else out_act), _stream(stream)))


def linear_qw_wmma_swiglu(x, w: QDeviceView, h, M, act, h_f16=0, stream=None):
    fn = getattr(_lib.load(), f"sxb_linear_{_b(w)}_wmma_swiglu")
    _check(fn(_ptr(x), C.byref(w.c()), _ptr(h), M, int(act), int(h_f16), _stream(stream)))


def hc_inject(x, w_in, y, T, H, d, act, stream=None):
    """kernels/hc.hpp:52-54: X[t, s*d + j] += w_in[t, s] * y[t, j], in place."""
    _check(_lib.load().sxb_hc_inject(_ptr(x), _ptr(w_in), _ptr(y), T, H, d, int(act), _stream(stream)))


def hc_mix_down(x, w: QDeviceView, T, H, d, r, inject, eps, h, w_in, inv, act, stream=None):
    """kernels/hc.hpp:36-42: X [T, H*d] -> h [T, r], w_in [T, H] (inject), inv [T, H]; w [r (+ H), H*d] Q4 or Q8."""
    fn = getattr(_lib.load(), f"sxb_hc_mix_down_{_b(w)}")
    _check(fn(_ptr(x), C.byref(w.c()), T, H, d, r, int(bool(inject)), C.c_float(eps), _ptr(h), _ptr(w_in), _ptr(inv), int(act),
              _stream(stream)))


def hc_mix_up(h, w_up: QDeviceView, x, norm_w, inv, T, H, d, u, act, stream=None):
    """kernels/hc.hpp:44-50: u [T, d] from h [T, r], the streams X, the hc_norm weight and inv; w_up [H*d, r] CHUNK-MAJOR."""
    fn = getattr(_lib.load(), f"sxb_hc_mix_up_{_b(w_up)}")
    _check(fn(_ptr(h), C.byref(w_up.c()), _ptr(x), _ptr(norm_w), _ptr(inv), T, H, d, _ptr(u), int(act), _stream(stream)))


def hc_wmma_workspace_bytes(T, H, d, R, bits, G) -> int:
    """kernels/hc_wmma.hpp:29-30: bytes of device workspace hc_mix_down_wmma needs for T tokens and R = r (+ H) weight rows."""
    n = _lib.load().sxb_hc_mix_down_wmma_workspace_bytes(T, H, d, R, int(bits), G)
    if n == 0:
        _check(1)
    return n


def hc_mix_down_wmma(x, w: QDeviceView, T, H, d, r, inject, eps, h, w_in, inv, ws, act, stream=None, inv_ready=False):
    """kernels/hc_wmma.hpp:34-39: hc_mix_down on the tensor cores (F16 operands, FP32 accumulation); ws: a uint8 tensor of
    hc_wmma_workspace_bytes, 256-byte aligned."""
    fn = getattr(_lib.load(), f"sxb_hc_mix_down_wmma_{_b(w)}")
    _check(fn(_ptr(x), C.byref(w.c()), T, H, d, r, int(bool(inject)), C.c_float(eps), _ptr(h), _ptr(w_in), _ptr(inv), _ptr(ws),
              ws.numel() * ws.element_size(), int(act), int(bool(inv_ready)), _stream(stream)))


def hc_inject_inv(x, w_in, y, T, H, d, eps, inv, act, stream=None):
    """kernels/hc_wmma.hpp:40-43: hc_inject and the next mix's inv [T, H] of the updated X, in one pass."""
    _check(_lib.load().sxb_hc_inject_inv(_ptr(x), _ptr(w_in), _ptr(y), T, H, d, C.c_float(eps), _ptr(inv), int(act), _stream(stream)))


def hc_mix_up_wmma_workspace_bytes(T, H, d, r, bits, G) -> int:
    n = _lib.load().sxb_hc_mix_up_wmma_workspace_bytes(T, H, d, r, int(bits), G)
    if n == 0:
        _check(1)
    return n


def hc_mix_up_wmma(h, w_up: QDeviceView, x, norm_w, inv, T, H, d, u, ws, act, stream=None):
    """kernels/hc_wmma.hpp:45-49: hc_mix_up on the tensor cores; w_up [H*d, r] CHUNK-MAJOR; ws: a uint8 tensor of
    hc_mix_up_wmma_workspace_bytes."""
    fn = getattr(_lib.load(), f"sxb_hc_mix_up_wmma_{_b(w_up)}")
    _check(fn(_ptr(h), C.byref(w_up.c()), _ptr(x), _ptr(norm_w), _ptr(inv), T, H, d, _ptr(u), _ptr(ws), ws.numel() * ws.element_size(),
              int(act), _stream(stream)))


def to_chunk_major(w: QDeviceView, stream=None) -> QDeviceView:
    """formats/q4.hpp:55 to_chunk_major on the device: a new view with the same codes, scales and mins chunk-major."""
    q, sc, mn = torch.empty_like(w.q), torch.empty_like(w.scale), torch.empty_like(w.minv)
    _check(_lib.load().sxb_to_chunk_major(C.byref(w.c()), w.bits, _ptr(q), _ptr(sc), _ptr(mn), _stream(stream)))
    return QDeviceView(q, sc, mn, w.N, w.K, w.G, w.bits)


# ---- kernels/moe_grouped.hpp ----------------------------------------------------------------------------------

def moe_route_workspace_bytes(M, A, E) -> int:
    n = _lib.load().sxb_moe_route_workspace_bytes(M, A, E)
    if n == 0:
        _check(1)
    return n


TC_TILES = ()  # rows of the tile lists beside those of 8 and 128 slots: none


def route_layout(M, A, E) -> dict:
    out = (C.c_int64 * 8)()
    _check(_lib.load().sxb_route_layout(M, A, E, out))
    keys = ["header", "offsets", "slots", "tile8_bucket", "tile8_start", "tile128_bucket", "tile128_start", "total"]
    return dict(zip(keys, list(out)))


def moe_group_routes(ids, M, A, E, ws, ws_bytes, err, stream=None):
    _count(2 if M * A > 2048 else 0)  # the multi-CTA pack is three launches
    _check(_lib.load().sxb_moe_group_routes(_ptr(ids), M, A, E, _ptr(ws), ws_bytes, _ptr(err), _stream(stream)))


def moe_route_small(logits, ld, M, E_total, k, e_lo, E_local, ids, coef, ws, ws_bytes, router_err, expert_err, stream=None):
    """moe_router + moe_group_routes[_ep] (M * k <= 2048 slots): one launch of one CTA up to 32 tokens, two above."""
    _count(1 if M > 32 else 0)
    _check(_lib.load().sxb_moe_route_small(_ptr(logits), ld, M, E_total, k, e_lo, E_local, _ptr(ids), _ptr(coef), _ptr(ws),
                                           ws_bytes, _ptr(router_err), _ptr(expert_err), _stream(stream)))


def check_grouped_status(ws, what: str):
    _check(_lib.load().sxb_check_grouped_status(_ptr(ws), what.encode()))


def moe_group_routes_ep(ids, M, A, E_total, e_lo, E_local, ws, ws_bytes, err, stream=None):
    _count(2 if M * A > 2048 else 0)
    _check(_lib.load().sxb_moe_group_routes_ep(_ptr(ids), M, A, E_total, e_lo, E_local, _ptr(ws), ws_bytes, _ptr(err),
                                               _stream(stream)))


def linear_qw_experts_gather_grouped(x, w: QDeviceView, E, ws, ws_bytes, M, A, y, act, math, stream=None):
    fn = getattr(_lib.load(), f"sxb_linear_{_b(w)}_experts_gather_grouped")
    _check(fn(_ptr(x), C.byref(w.c()), E, _ptr(ws), ws_bytes, M, A, _ptr(y), int(act), int(math), _stream(stream)))


def linear_qw_experts_gather_grouped_swiglu(x, w: QDeviceView, E, ws, ws_bytes, M, A, h, act, math, stream=None,
                                            h_f16=False):
    fn = getattr(_lib.load(), f"sxb_linear_{_b(w)}_experts_gather_grouped_swiglu")
    _check(fn(_ptr(x), C.byref(w.c()), E, _ptr(ws), ws_bytes, M, A, _ptr(h), int(act), int(math), _stream(stream),
              int(h_f16)))


@dataclass
class MoeSharedAdd:  # kernels/moe_grouped.hpp:75-81
    s: torch.Tensor
    gate_logit: object  # tensor or raw pointer to token 0's gate logit
    gate_ld: int
    gate_index: int
    err: torch.Tensor

    def c(self) -> _lib.SxbMoeSharedAdd:
        return _lib.SxbMoeSharedAdd(_ptr(self.s), _ptr(self.gate_logit), self.gate_ld, self.gate_index, _ptr(self.err))


def linear_qw_experts_combine_grouped(h, w: QDeviceView, E, ids, coef, ws, ws_bytes, partial, M, A, y, act, math,
                                      stream=None, shared: Optional[MoeSharedAdd] = None, h_f16=False, out_act=None):
    fn = getattr(_lib.load(), f"sxb_linear_{_b(w)}_experts_combine_grouped")
    sh = C.byref(shared.c()) if shared is not None else None
    _count(1)  # the per-slot dots, then the reduce
    _check(fn(_ptr(h), C.byref(w.c()), E, _ptr(ids), _ptr(coef), _ptr(ws), ws_bytes, _ptr(partial), M, A, _ptr(y),
              int(act), int(act if out_act is None else out_act), int(math), _stream(stream), sh, int(h_f16)))


def linear_qw_experts_combine_grouped_ep(h, w: QDeviceView, E_local, E_total, e_lo, ids, coef, ws, ws_bytes, partial, M,
                                         A, y, act, math, stream=None, h_f16=False, out_act=None):
    fn = getattr(_lib.load(), f"sxb_linear_{_b(w)}_experts_combine_grouped_ep")
    _count(1)
    _check(fn(_ptr(h), C.byref(w.c()), E_local, E_total, e_lo, _ptr(ids), _ptr(coef), _ptr(ws), ws_bytes, _ptr(partial),
              M, A, _ptr(y), int(act), int(act if out_act is None else out_act), int(math), _stream(stream), int(h_f16)))


# ---- kernels/linear_q4.hpp, kernels/linear_q8.hpp, runtime/qweight.hpp -----------------------------------------

def linear_qw(x, w: QDeviceView, y, M, act, out_act=None, stream=None):
    fn = getattr(_lib.load(), f"sxb_linear_{_b(w)}")
    _check(fn(_ptr(x), C.byref(w.c()), _ptr(y), M, int(act), int(act if out_act is None else out_act), _stream(stream)))


def linear_q4(x, w, y, M, act, out_act=None, stream=None):
    linear_qw(x, w, y, M, act, out_act, stream)


linear_q8 = linear_q4


def linear_qw_experts_gather(x, w: QDeviceView, E, ids, M, A, y, act, err, stream=None):
    fn = getattr(_lib.load(), f"sxb_linear_{_b(w)}_experts_gather")
    _check(fn(_ptr(x), C.byref(w.c()), E, _ptr(ids), M, A, _ptr(y), int(act), _ptr(err), _stream(stream)))


def linear_qw_experts_gather_swiglu(x, w: QDeviceView, E, ids, M, A, h, act, err, stream=None):
    fn = getattr(_lib.load(), f"sxb_linear_{_b(w)}_experts_gather_swiglu")
    _check(fn(_ptr(x), C.byref(w.c()), E, _ptr(ids), M, A, _ptr(h), int(act), _ptr(err), _stream(stream)))


def linear_qw_experts_combine(h, w: QDeviceView, E, ids, coef, M, A, y, act, err, stream=None, out_act=None):
    fn = getattr(_lib.load(), f"sxb_linear_{_b(w)}_experts_combine")
    _check(fn(_ptr(h), C.byref(w.c()), E, _ptr(ids), _ptr(coef), M, A, _ptr(y), int(act),
              int(act if out_act is None else out_act), _ptr(err), _stream(stream)))


def check_expert_error(err, what: str):
    _check(_lib.load().sxb_check_expert_error(_ptr(err), what.encode()))


def report_expert_error(e, what: str):
    _check(_lib.load().sxb_report_expert_error((C.c_uint32 * 3)(*[int(v) for v in e]), what.encode()))


def stage_f16(x, M, K, bits, xh, stream=None):
    """x [M, K] BF16 -> xh [M, K] F16 in the k order of a `bits`-bit tensor-core weight operand."""
    _check(_lib.load().sxb_stage_f16(_ptr(x), M, K, bits, _ptr(xh), _stream(stream)))


def stage_f16_tiles(x, ws, ws_bytes, M, A, E, K, bits, xs, stream=None):
    """x [M, K] BF16 -> xs, the tile-blocked F16 operand form for the tiles of grouping workspace ws."""
    _check(_lib.load().sxb_stage_f16_tiles(_ptr(x), _ptr(ws), ws_bytes, M, A, E, K, bits, _ptr(xs), _stream(stream)))


# ---- kernels/swiglu.hpp ---------------------------------------------------------------------------------------

def swiglu(gu, h, rows, I, act, stream=None):
    _check(_lib.load().sxb_swiglu(_ptr(gu), _ptr(h), rows, I, int(act), _stream(stream)))


# ---- formats/q4.hpp, formats/q8.hpp (on the device) -----------------------------------------------------------

def quantize(w: torch.Tensor, G: int, bits: int, err: Optional[torch.Tensor] = None, stream=None) -> QDeviceView:
    """quantize_q4 / quantize_q8 (formats/q4.hpp:32, formats/q8.hpp:32) of an FP32 [N, K] tensor on the device."""
    if w.dtype != torch.float32 or w.dim() != 2 or not w.is_contiguous():
        raise Error(1, "quantize: w must be a contiguous FP32 [N, K] tensor")
    N, K = w.shape
    if bits not in (4, 8) or G not in (32, 64, 128) or K % G:
        raise Error(1, f"quantize: bits = {bits}, G = {G}, K = {K} unsupported")
    with _within(stream, w.device):
        q = torch.empty((N, K // 2 if bits == 4 else K), dtype=torch.uint8, device=w.device)
        scale = torch.empty((N, K // G), dtype=torch.int16, device=w.device)
        minv = torch.empty((N, K // G), dtype=torch.int16, device=w.device)
        own = err is None
        if own:
            err = torch.zeros(4, dtype=torch.int32, device=w.device)
        _check(_lib.load().sxb_quantize(_ptr(w), N, K, G, bits, _ptr(q), _ptr(scale), _ptr(minv), _ptr(err), _stream(stream)))
        if own and int(err[0].item()) != 0:
            raise Error(1, f"quantize: non-finite weight at [{int(err[1])}, {int(err[2])}]")
    _handed(stream, q, scale, minv)
    return QDeviceView(q, scale, minv, N, K, G, bits)


# ---- attention over a paged key-value cache (no counterpart among the launchers mirrored above) -------------------

def _on(dev, what: str, **tensors):
    """Refuses what the kernels would take for something else: {name: (tensor, dtypes)} on another device than the cache's, of another type, or
    not contiguous along its last dimension."""
    for name, (t, dtypes) in tensors.items():
        if t is None:
            continue
        if t.device != dev or t.dtype not in dtypes or (t.dim() and t.stride(-1) != 1 and t.shape[-1] != 1):
            raise Error(1, f"{what}: {name} is {t.dtype} on {t.device} with strides {tuple(t.stride())}, expected {' or '.join(map(str, dtypes))} on {dev}, "
                           "its last dimension contiguous")


_I32, _F32, _ROWS = (torch.int32,), (torch.float32,), (torch.bfloat16, torch.float32)
_BF16 = (torch.bfloat16,)
_WORDS = (torch.int32, torch.uint32)


class KvCache:
    """A pool of pages of keys and values (SxbKvCache).  k, v: BF16 [n_pages, n_kv, page, D] (bits 16), or uint8 codes of that shape (8) or
    [n_pages, n_kv, page, D / 2] (4) with k_sm, v_sm [n_pages, n_kv, page, D / G, 2] BF16, a group's scale and min.  The first three
    dimensions may have any strides, the same ones (in rows) for all: a transposed view of [n_pages, page, n_kv, D] is fine."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, bits: int, G: int = 0, k_sm: Optional[torch.Tensor] = None, v_sm: Optional[torch.Tensor] = None):
        if bits not in (16, 8, 4):
            raise Error(1, f"KvCache: {bits} bits unsupported (16 = BF16, 8 or 4)")
        if k.dim() != 4 or v.shape != k.shape:
            raise Error(1, f"KvCache: k {tuple(k.shape)} and v {tuple(v.shape)}, expected the same [n_pages, n_kv, page, D]")
        if not k.is_cuda:
            raise Error(1, "KvCache: the cache must live on a CUDA device (no CPU path exists)")
        self.n_pages, self.n_kv, self.page = k.shape[:3]
        self.D = k.shape[3] * (2 if bits == 4 else 1)
        self.bits, self.G, self.device = bits, (self.D if bits == 16 else G), k.device
        codes = _BF16 if bits == 16 else (torch.uint8,)
        _on(k.device, "KvCache", k=(k, codes), v=(v, codes))
        parts = [(k, k.shape[3]), (v, k.shape[3])]
        if bits != 16:
            if G not in (32, 64, 128) or G > self.D:
                raise Error(1, f"KvCache: group size {G} unsupported (32, 64 or 128, at most D = {self.D})")
            groups = self.D // G
            for name, t in (("k_sm", k_sm), ("v_sm", v_sm)):
                if t is None or tuple(t.shape) != (*k.shape[:3], groups, 2) or t.stride(3) != 2:
                    raise Error(1, f"KvCache: {name} is {None if t is None else tuple(t.shape)}, expected {(*k.shape[:3], groups, 2)}, a row's groups contiguous")
            _on(k.device, "KvCache", k_sm=(k_sm, _BF16), v_sm=(v_sm, _BF16))
            parts += [(k_sm, 2 * groups), (v_sm, 2 * groups)]
        elif k_sm is not None or v_sm is not None:
            raise Error(1, "KvCache: a BF16 cache has no scales")
        rows = None
        for t, n in parts:
            # a dimension of one has no stride to speak of
            here = tuple(t.stride(i) / n if t.shape[i] > 1 else 1 for i in range(3))
            if any(r != int(r) or r < 1 for r in here) or (rows is not None and here != rows):
                raise Error(1, f"KvCache: strides {tuple(t.stride())} are not whole rows of {n}, or not those of k")
            rows = here
        self.k, self.v, self.k_sm, self.v_sm = k, v, k_sm, v_sm
        self._c = _lib.SxbKvCache(k.data_ptr(), v.data_ptr(), _ptr(k_sm), _ptr(v_sm), self.n_pages, self.n_kv, self.page, self.D, self.G,
                                  *[int(r) for r in rows], bits)
        self.index, self._at = k.get_device(), C.addressof(self._c)

    @classmethod
    def empty(cls, n_pages: int, n_kv: int, page: int, D: int, bits: int, G: int = 64, device="cuda") -> "KvCache":
        """A pool of zeros."""
        def zeros(*shape, dtype):
            return torch.zeros((n_pages, n_kv, page, *shape), dtype=dtype, device=device)
        if bits == 16:
            return cls(zeros(D, dtype=torch.bfloat16), zeros(D, dtype=torch.bfloat16), 16)
        n = D // 2 if bits == 4 else D
        return cls(zeros(n, dtype=torch.uint8), zeros(n, dtype=torch.uint8), bits, G, zeros(D // G, 2, dtype=torch.bfloat16),
                   zeros(D // G, 2, dtype=torch.bfloat16))

    def bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_sm, self.v_sm) if t is not None)


# The argument blocks of include/strix_b200.h, field for field (native alignment): packed and passed as one pointer, a call of twenty arguments costs
# ctypes more than the smallest kernel takes.
_WRITE_ARGS = struct.Struct("@PqqqPPPqPPPqqqPPqPfii")
_READ_ARGS = struct.Struct("@PPPPqqqqPPPi")
_DECODE_ARGS = struct.Struct("@PqqqPPqqPPqqPqPPNPqff")


def _rows(t: torch.Tensor) -> int:
    """Elements from one row of a matrix to the next."""
    return t.shape[1] if t.is_contiguous() else t.stride(0)


def _refuse(cache, what, **tensors):
    """A call's tensors are not what the kernels take them for: says which one."""
    if cache.index != torch.cuda.current_device():
        raise Error(1, f"{what}: the cache lives on {cache.device}, the current device is {torch.cuda.current_device()}")
    _on(cache.device, what, **tensors)
    raise Error(1, f"{what}: a vector is not contiguous, or the shapes do not fit: " + ", ".join(f"{n} {tuple(t.shape)}" for n, (t, _) in tensors.items() if t is not None))


def _places_ok(cache, seq, pos, pages, err, T):
    dev = cache.index
    return (seq.dtype is torch.int32 and pos.dtype is torch.int32 and pages.dtype is torch.int32 and err.dtype in _WORDS and seq.get_device() == dev
            and pos.get_device() == dev and pages.get_device() == dev and err.get_device() == dev and seq.is_contiguous() and pos.is_contiguous()
            and err.is_contiguous() and pages.dim() == 2 and (pages.is_contiguous() or pages.stride(1) == 1) and seq.numel() == T and pos.numel() == T
            and err.numel() >= 3)


def attn_qkv_write(qkv, cache: KvCache, seq, pos, pages, q_out, err, q_norm=None, k_norm=None, eps=1e-6, inv_freq=None, interleaved=False, stream=None):
    """sxb_attn_qkv_write: qkv [T, (n_q + 2 n_kv) D] BF16 or FP32 -> queries normed and rotated into q_out [T, n_q D] BF16, keys and values into the
    cache at position pos [T] of sequence seq [T] (int32; seq < 0: a padding row), pages [n_seq, n_cols] int32.  q_norm, k_norm [D] FP32 or None;
    inv_freq [rot / 2] FP32 or None.  err: 3 or more zeroed int32."""
    T, width = qkv.shape
    D, dev, dt = cache.D, cache.index, qkv.dtype
    n_q = width // D - 2 * cache.n_kv
    rot = qn = kn = fr = 0
    ok = (dev == torch._C._cuda_getDevice() and dt in _ROWS and q_out.dtype is torch.bfloat16 and qkv.get_device() == dev and q_out.get_device() == dev
          and width % D == 0 and n_q >= 1 and q_out.shape == (T, n_q * D) and (qkv.is_contiguous() or qkv.stride(1) == 1)
          and (q_out.is_contiguous() or q_out.stride(1) == 1) and _places_ok(cache, seq, pos, pages, err, T))
    if q_norm is not None:
        ok = ok and q_norm.dtype is torch.float32 and q_norm.get_device() == dev and q_norm.is_contiguous() and q_norm.numel() == D
        qn = q_norm.data_ptr()
    if k_norm is not None:
        ok = ok and k_norm.dtype is torch.float32 and k_norm.get_device() == dev and k_norm.is_contiguous() and k_norm.numel() == D
        kn = k_norm.data_ptr()
    if inv_freq is not None:
        ok = ok and inv_freq.dtype is torch.float32 and inv_freq.get_device() == dev and inv_freq.is_contiguous()
        rot, fr = 2 * inv_freq.numel(), inv_freq.data_ptr()
    if not ok:
        _refuse(cache, "attn_qkv_write", qkv=(qkv, _ROWS), q_out=(q_out, _BF16), q_norm=(q_norm, _F32), k_norm=(k_norm, _F32), inv_freq=(inv_freq, _F32),
                seq=(seq, _I32), pos=(pos, _I32), pages=(pages, _I32), err=(err, _WORDS))
    n_seq, n_cols = pages.shape
    _check(_lib.load().sxb_attn_qkv_write(_WRITE_ARGS.pack(
        qkv.data_ptr(), _rows(qkv), T, n_q, qn, kn, fr, rot, seq.data_ptr(), pos.data_ptr(), pages.data_ptr(), _rows(pages), n_cols, n_seq, cache._at,
        q_out.data_ptr(), _rows(q_out), err.data_ptr(), eps, dt is torch.bfloat16, bool(interleaved)), _stream(stream)))


def kv_read(cache: KvCache, seq, pos, pages, k_out, v_out, err, stream=None):
    """sxb_kv_read: positions pos [T] of sequences seq [T] of the cache -> k_out, v_out [T, n_kv, D], BF16 or FP32."""
    T, dev, dt = seq.shape[0], cache.index, k_out.dtype
    shape = (T, cache.n_kv, cache.D)
    if not (dev == torch._C._cuda_getDevice() and dt in _ROWS and v_out.dtype is dt and k_out.get_device() == dev and v_out.get_device() == dev
            and k_out.shape == shape and v_out.shape == shape and k_out.is_contiguous() and v_out.is_contiguous()
            and _places_ok(cache, seq, pos, pages, err, T)):
        _refuse(cache, "kv_read", k_out=(k_out, _ROWS), v_out=(v_out, (dt,)), seq=(seq, _I32), pos=(pos, _I32), pages=(pages, _I32), err=(err, _WORDS))
    n_seq, n_cols = pages.shape
    _check(_lib.load().sxb_kv_read(_READ_ARGS.pack(
        cache._at, seq.data_ptr(), pos.data_ptr(), pages.data_ptr(), _rows(pages), n_cols, n_seq, T, k_out.data_ptr(), v_out.data_ptr(), err.data_ptr(),
        dt is torch.bfloat16), _stream(stream)))


def attn_decode_workspace_bytes(cache: KvCache, n_q: int, max_q: int) -> int:
    """Bytes of workspace that attn_decode needs on the current device; zeroed once before its first use."""
    n = _lib.load().sxb_attn_decode_workspace_bytes(n_q, cache.n_kv, cache.D, cache.bits, max_q)
    if n == 0:
        _check(1)
    return n


def attn_decode(q, cache: KvCache, pages, q_start, kv_len, max_q, out, ws, err, scale=None, softcap=0.0, window=0, lse=None, stream=None):
    """sxb_attn_decode: q [T, n_q D] BF16, rows q_start[b] .. q_start[b + 1] - 1 (int32 [B + 1]) the new tokens of sequence b, kv_len [B] int32 its
    keys, their own included -> out [T, n_q D] BF16, lse [T, n_q] FP32.  scale: None = D ** -0.5; softcap, window: 0 = none.  max_q: a
    sequence's largest count of new tokens."""
    T, width = q.shape
    D, dev, B = cache.D, cache.index, kv_len.shape[0]
    n_q = width // D
    if not (dev == torch._C._cuda_getDevice() and q.dtype is torch.bfloat16 and out.dtype is torch.bfloat16 and pages.dtype is torch.int32
            and q_start.dtype is torch.int32 and kv_len.dtype is torch.int32 and err.dtype in _WORDS and q.get_device() == dev and out.get_device() == dev
            and pages.get_device() == dev and q_start.get_device() == dev and kv_len.get_device() == dev and ws.get_device() == dev
            and err.get_device() == dev and width % D == 0 and out.shape == (T, width) and pages.dim() == 2 and pages.shape[0] >= B
            and q_start.numel() == B + 1 and (q.is_contiguous() or q.stride(1) == 1) and (out.is_contiguous() or out.stride(1) == 1)
            and (pages.is_contiguous() or pages.stride(1) == 1) and q_start.is_contiguous() and kv_len.is_contiguous() and ws.is_contiguous()
            and err.is_contiguous() and err.numel() >= 3
            and (lse is None or (lse.dtype is torch.float32 and lse.get_device() == dev and lse.shape == (T, n_q) and lse.is_contiguous()))):
        _refuse(cache, "attn_decode", q=(q, _BF16), out=(out, _BF16), pages=(pages, _I32), q_start=(q_start, _I32), kv_len=(kv_len, _I32), lse=(lse, _F32),
                ws=(ws, (ws.dtype,)), err=(err, _WORDS))
    rows = max_q * (n_q // cache.n_kv)
    tile = 8 if rows <= 8 else 16 if rows <= 16 or cache.bits != 16 or D == 256 else 32
    if tile * D > 1024:
        _count()  # the parts of split sequences are joined by a second kernel
    _check(_lib.load().sxb_attn_decode(_DECODE_ARGS.pack(
        q.data_ptr(), _rows(q), T, n_q, cache._at, pages.data_ptr(), _rows(pages), pages.shape[1], q_start.data_ptr(), kv_len.data_ptr(), B, max_q,
        out.data_ptr(), _rows(out), 0 if lse is None else lse.data_ptr(), ws.data_ptr(), ws.numel() * ws.element_size(), err.data_ptr(), window,
        D ** -0.5 if scale is None else scale, softcap), _stream(stream)))


def check_attn_error(err, what: str):
    _check(_lib.load().sxb_check_attn_error(_ptr(err), what.encode()))


def report_attn_error(e, what: str):
    _check(_lib.load().sxb_report_attn_error((C.c_uint32 * 3)(*[int(v) for v in e]), what.encode()))


# ---- around the head: norm into 8-bit codes, products of 8-bit floating point, verification of drafts ---------------------

F8 = torch.float8_e4m3fn
_F8_BLOCK = 128
_NORM_ARGS = struct.Struct("@PPPPPPPqqqqqqqqfiii")
_LINEAR_F8_ARGS = struct.Struct("@PPPPqqqqi")
_VERIFY_ARGS = struct.Struct("@PPqqqqqPPPPPPPPPNPii")


def _blocks(n: int) -> int:
    return -(-n // _F8_BLOCK)


def _refuse_all(dev, what, **tensors):
    """A call's tensors are not what the kernels take them for: says which one."""
    if dev != torch.cuda.current_device():
        raise Error(1, f"{what}: the tensors live on device {dev}, the current device is {torch.cuda.current_device()}")
    _on(torch.device("cuda", dev), what, **tensors)
    raise Error(1, f"{what}: a vector is not contiguous, or the shapes do not fit: " + ", ".join(f"{n} {tuple(t.shape)}" for n, (t, _) in tensors.items() if t is not None))


def _ld(t, what: str, name: str) -> int:
    """The row stride of a tensor that is not contiguous.  (The wrappers below ask for no strides of those that are: each costs 0.17 us.)"""
    if t.dim() != 2 or (t.stride(1) != 1 and t.shape[1] != 1):
        raise Error(1, f"{what}: {name} is {tuple(t.shape)} with strides {tuple(t.stride())}, expected two dimensions, the last one contiguous")
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _matrix(t, what: str, name: str):
    if t.dim() != 2:
        raise Error(1, f"{what}: {name} is {tuple(t.shape)}, expected two dimensions")
    return t.shape


class F8View:
    """A weight in 8-bit floating point (SxbF8View): codes q [N, K] float8_e4m3fn, contiguous, scale [ceil(N / 128), ceil(K / 128)] FP32."""

    def __init__(self, q: torch.Tensor, scale: torch.Tensor):
        if q.dim() != 2 or q.dtype != F8 or not q.is_contiguous():
            raise Error(1, f"F8View: q is {tuple(q.shape)} of {q.dtype}, expected contiguous [N, K] of {F8}")
        self.N, self.K = q.shape
        if scale.dtype != torch.float32 or tuple(scale.shape) != (_blocks(self.N), _blocks(self.K)) or not scale.is_contiguous() or scale.device != q.device:
            raise Error(1, f"F8View: scale is {tuple(scale.shape)} of {scale.dtype} on {scale.device}, expected contiguous {(_blocks(self.N), _blocks(self.K))} FP32 on {q.device}")
        if not q.is_cuda:
            raise Error(1, "F8View: the weight must live on a CUDA device (no CPU path exists)")
        self.q, self.scale, self.device, self.index, self.blocks = q, scale, q.device, q.get_device(), _blocks(self.K)
        self._c = _lib.SxbF8View(q.data_ptr(), scale.data_ptr(), self.N, self.K)
        self._at = C.addressof(self._c)

    def bytes(self) -> int:
        return self.q.numel() + 4 * self.scale.numel()


def quantize_f8(w: torch.Tensor, err: Optional[torch.Tensor] = None, stream=None) -> F8View:
    """sxb_quantize_f8 of a contiguous FP32 or BF16 [N, K] tensor: codes and a scale for each block of 128 x 128."""
    if w.dtype not in _ROWS or w.dim() != 2 or not w.is_contiguous():
        raise Error(1, "quantize_f8: w must be a contiguous FP32 or BF16 [N, K] tensor")
    if w.is_cuda and w.get_device() != torch.cuda.current_device():
        raise Error(1, f"quantize_f8: w lives on device {w.get_device()}, the current device is {torch.cuda.current_device()}")
    if err is not None and (err.device != w.device or err.dtype not in _WORDS or not err.is_contiguous() or err.numel() < 3):
        raise Error(1, f"quantize_f8: err is {err.dtype} {tuple(err.shape)} on {err.device}, expected 3 or more contiguous int32 on {w.device}")
    N, K = w.shape
    with _within(stream, w.device):
        q = torch.empty((N, K), dtype=torch.uint8, device=w.device).view(F8)
        scale = torch.empty((_blocks(N), _blocks(K)), dtype=torch.float32, device=w.device)
        own = err is None
        if own:
            err = torch.zeros(4, dtype=torch.int32, device=w.device)
        _check(_lib.load().sxb_quantize_f8(_ptr(w), _w_act(w), N, K, _ptr(q), _ptr(scale), _ptr(err), _stream(stream)))
        if own and int(err[0].item()) != 0:
            raise Error(1, f"quantize_f8: non-finite weight at [{int(err[1])}, {int(err[2])}]")
    _handed(stream, q, scale)
    return F8View(q, scale)


def add_norm(x, y=None, weight=None, eps=1e-6, total=None, out=None, codes=None, scales=None, norm=True, stream=None):
    """sxb_add_norm: s = x + y in x's type (x [T, d] BF16 or FP32, y BF16, FP32 or None) -> total (may be x or y), its norm times weight [d] FP32 (None: 1) -> out
    BF16, codes float8_e4m3fn with scales [T, ceil(d / 128)] FP32; each of them or None.  norm=False: s itself in the place of its norm."""
    T, d = shape = _matrix(x, "add_norm", "x")
    dev, dt = x.get_device(), x.dtype
    ok = dev == torch._C._cuda_getDevice() and dt in _ROWS
    x_ld = d if x.is_contiguous() else _ld(x, "add_norm", "x")
    yp = wp = tp = op = cp = sp = y_bf16 = 0
    y_ld = t_ld = o_ld = c_ld = s_ld = d
    if y is not None:
        ok = ok and y.dtype in _ROWS and y.get_device() == dev and y.shape == shape
        yp, y_bf16 = y.data_ptr(), y.dtype is torch.bfloat16
        if not y.is_contiguous():
            y_ld = _ld(y, "add_norm", "y")
    if weight is not None:
        ok = ok and weight.dtype is torch.float32 and weight.get_device() == dev and weight.is_contiguous() and weight.numel() == d
        wp = weight.data_ptr()
    if total is not None:
        ok = ok and total.dtype is dt and total.get_device() == dev and total.shape == shape
        tp = total.data_ptr()
        if not total.is_contiguous():
            t_ld = _ld(total, "add_norm", "total")
    if out is not None:
        ok = ok and out.dtype is torch.bfloat16 and out.get_device() == dev and out.shape == shape
        op = out.data_ptr()
        if not out.is_contiguous():
            o_ld = _ld(out, "add_norm", "out")
    if codes is not None:
        ok = ok and codes.dtype is F8 and codes.get_device() == dev and codes.shape == shape
        cp = codes.data_ptr()
        if not codes.is_contiguous():
            c_ld = _ld(codes, "add_norm", "codes")
    if scales is not None:
        s_ld = -(-d // _F8_BLOCK)
        ok = ok and scales.dtype is torch.float32 and scales.get_device() == dev and scales.shape == (T, s_ld)
        sp = scales.data_ptr()
        if not scales.is_contiguous():
            s_ld = _ld(scales, "add_norm", "scales")
    if not ok:
        _refuse_all(dev, "add_norm", x=(x, _ROWS), y=(y, _ROWS), weight=(weight, _F32), total=(total, (dt,)), out=(out, _BF16), codes=(codes, (F8,)), scales=(scales, _F32))
    _check(_lib.load().sxb_add_norm(_NORM_ARGS.pack(
        x.data_ptr(), yp, wp, tp, op, cp, sp, T, d, x_ld, y_ld, t_ld, o_ld, c_ld, s_ld, eps, dt is torch.bfloat16, y_bf16, bool(norm)),
        torch._C._cuda_getCurrentRawStream(dev) if stream is None else _stream(stream)))


def linear_f8(x, x_scale, w: F8View, y, stream=None):
    """sxb_linear_f8: y [M, N] BF16 or FP32 = x [M, K] float8_e4m3fn (scales x_scale [M, ceil(K / 128)] FP32) times w^T."""
    M, K = _matrix(x, "linear_f8", "x")
    dev, dt = w.index, y.dtype
    if not (dev == torch._C._cuda_getDevice() and x.dtype is F8 and x_scale.dtype is torch.float32 and dt in _ROWS and x.get_device() == dev and x_scale.get_device() == dev
            and y.get_device() == dev and K == w.K and x_scale.shape == (M, w.blocks) and y.shape == (M, w.N)):
        _refuse_all(dev, "linear_f8", x=(x, (F8,)), x_scale=(x_scale, _F32), w=(w.q, (F8,)), y=(y, _ROWS))
    _check(_lib.load().sxb_linear_f8(_LINEAR_F8_ARGS.pack(
        x.data_ptr(), x_scale.data_ptr(), w._at, y.data_ptr(), M, K if x.is_contiguous() else _ld(x, "linear_f8", "x"),
        w.blocks if x_scale.is_contiguous() else _ld(x_scale, "linear_f8", "x_scale"), w.N if y.is_contiguous() else _ld(y, "linear_f8", "y"),
        dt is torch.bfloat16), torch._C._cuda_getCurrentRawStream(dev) if stream is None else _stream(stream)))


def verify_drafts_workspace_bytes(T: int, B: int, V: int) -> int:
    """Bytes of workspace that verify_drafts needs for T rows of B sequences over V tokens."""
    n = _lib.load().sxb_verify_drafts_workspace_bytes(T, B, V)
    if n == 0:
        _check(1)
    return n


def verify_drafts(logits, ids, q_start, u, u_pick, next_ids, n_new, ws, err, draft_logits=None, temperature=None, logp=None, stream=None):
    """sxb_verify_drafts: rows q_start[b] .. q_start[b + 1] - 1 (int32 [B + 1]) are sequence b's: the tokens ids [T] int32 fed there, the drafted ones behind the first, the target's
    logits [T, V] BF16 or FP32, the drafter's (or None: its tokens are all that is known of it), random numbers u [T] and u_pick [B] FP32, temperature [B] FP32 (None: 1; 0: greedy)
    -> next_ids [T] int32 (-1 behind the last), n_new [B] int32, logp [T] FP32 or None.  err: 3 or more zeroed int32."""
    T, V = shape = _matrix(logits, "verify_drafts", "logits")
    dev, B = logits.get_device(), n_new.numel()
    ok = (dev == torch._C._cuda_getDevice() and logits.dtype in _ROWS and ids.dtype is torch.int32 and ids.get_device() == dev
          and ids.numel() == T and ids.is_contiguous() and q_start.dtype is torch.int32 and q_start.get_device() == dev and q_start.numel() == B + 1 and q_start.is_contiguous()
          and u.dtype is torch.float32 and u.get_device() == dev and u.numel() == T and u.is_contiguous() and u_pick.dtype is torch.float32 and u_pick.get_device() == dev
          and u_pick.numel() == B and u_pick.is_contiguous() and next_ids.dtype is torch.int32 and next_ids.get_device() == dev and next_ids.numel() == T and next_ids.is_contiguous()
          and n_new.dtype is torch.int32 and n_new.get_device() == dev and n_new.is_contiguous() and ws.get_device() == dev and ws.is_contiguous()
          and err.get_device() == dev and err.dtype in _WORDS and err.is_contiguous() and err.numel() >= 3)
    dp = tp = lp = d_bf16 = 0
    ld = V if logits.is_contiguous() else _ld(logits, "verify_drafts", "logits")
    dld = V
    if draft_logits is not None:
        d = draft_logits
        ok = ok and d.dtype in _ROWS and d.get_device() == dev and d.shape == shape
        dp, d_bf16 = d.data_ptr(), d.dtype is torch.bfloat16
        if not d.is_contiguous():
            dld = _ld(d, "verify_drafts", "draft_logits")
    if temperature is not None:
        ok = ok and temperature.dtype is torch.float32 and temperature.get_device() == dev and temperature.numel() == B and temperature.is_contiguous()
        tp = temperature.data_ptr()
    if logp is not None:
        ok = ok and logp.dtype is torch.float32 and logp.get_device() == dev and logp.numel() == T and logp.is_contiguous()
        lp = logp.data_ptr()
    if not ok:
        _refuse_all(dev, "verify_drafts", logits=(logits, _ROWS), draft_logits=(draft_logits, _ROWS), ids=(ids, _I32), q_start=(q_start, _I32), u=(u, _F32), u_pick=(u_pick, _F32),
                    temperature=(temperature, _F32), next_ids=(next_ids, _I32), n_new=(n_new, _I32), logp=(logp, _F32), ws=(ws, (ws.dtype,)), err=(err, _WORDS))
    _count()  # two launches
    _check(_lib.load().sxb_verify_drafts(_VERIFY_ARGS.pack(
        logits.data_ptr(), dp, ld, dld, T, V, B, ids.data_ptr(), q_start.data_ptr(), u.data_ptr(), u_pick.data_ptr(), tp,
        next_ids.data_ptr(), n_new.data_ptr(), lp, ws.data_ptr(), ws.nbytes, err.data_ptr(), logits.dtype is torch.bfloat16, d_bf16),
        torch._C._cuda_getCurrentRawStream(dev) if stream is None else _stream(stream)))


def check_verify_error(err, what: str):
    _check(_lib.load().sxb_check_verify_error(_ptr(err), what.encode()))


def report_verify_error(e, what: str):
    _check(_lib.load().sxb_report_verify_error((C.c_uint32 * 3)(*[int(v) for v in e]), what.encode()))


# ---- the whole block as one call ------------------------------------------------------------------------------

def _layer_args(x, logits, y, gate_up, down, E, A, ids, coef, ws, ws_bytes, h, partial, router_err, expert_err, xs, math, E_total,
                e_lo, shared_gate_up, shared_down, sh_gu, sh_h, sh_y, sh_xs):
    M = x.shape[0]
    gu, dn = gate_up.c(), down.c()
    a = _lib.SxbMoeLayerArgs()
    a.M, a.E, a.A, a.E_total, a.e_lo = M, E, A, (E if E_total is None else E_total), e_lo
    a.gate_up, a.down, a.gate_up_bits, a.down_bits = C.pointer(gu), C.pointer(dn), gate_up.bits, down.bits
    keep = [gu, dn]
    if shared_gate_up is not None:
        sgu, sdn = shared_gate_up.c(), shared_down.c()
        keep += [sgu, sdn]
        a.shared_gate_up, a.shared_down, a.shared_bits = C.pointer(sgu), C.pointer(sdn), shared_gate_up.bits
    a.x, a.logits, a.logits_ld, a.y = _ptr(x), _ptr(logits), (logits.stride(0) if logits is not None else 0), _ptr(y)
    a.out_act = int(Act.F32 if y.dtype == torch.float32 else Act.BF16)
    a.math = -1 if math is None else int(math)
    a.ids, a.coef, a.ws, a.ws_bytes, a.h, a.partial = _ptr(ids), _ptr(coef), _ptr(ws), ws_bytes, _ptr(h), _ptr(partial)
    a.xs = _ptr(xs) if xs is not None else None
    for name, t in (("sh_gu", sh_gu), ("sh_h", sh_h), ("sh_y", sh_y), ("sh_xs", sh_xs)):
        setattr(a, name, _ptr(t) if t is not None else None)
    a.router_err, a.expert_err = _ptr(router_err), _ptr(expert_err)
    return a, keep


def moe_layer(x, logits, y, gate_up: QDeviceView, down: QDeviceView, E, A, ids, coef, ws, ws_bytes, h, partial, router_err,
              expert_err, xs=None, math=None, E_total=None, e_lo=0, shared_gate_up: Optional[QDeviceView] = None,
              shared_down: Optional[QDeviceView] = None, sh_gu=None, sh_h=None, sh_y=None, sh_xs=None, stream=None, side=None):
    """sxb_moe_layer: router, grouping, gate/up + SwiGLU, down + combine (+ shared expert) enqueued by one C call.
    x [M, d] BF16, logits [M, ld] FP32 (None: ids / coef already hold the routes), y [M, d] BF16 or FP32; the rest are the
    caller's work buffers.  side: a second stream for the shared expert's launches on the streaming path."""
    a, keep = _layer_args(x, logits, y, gate_up, down, E, A, ids, coef, ws, ws_bytes, h, partial, router_err, expert_err, xs, math,
                          E_total, e_lo, shared_gate_up, shared_down, sh_gu, sh_h, sh_y, sh_xs)
    M, small = x.shape[0], x.shape[0] * A <= 2048
    merged = logits is not None and small and M <= 32  # router and pack in one launch
    tc = (M >= 256) if math is None else int(math) >= int(MoeMath.WmmaF16)
    _count(int(logits is not None) + (1 if small else 3) - int(merged) + int(tc) + (3 if shared_gate_up is not None else 0) + 2)
    if side is None:
        _check(_lib.load().sxb_moe_layer(C.byref(a), _stream(stream)))
    else:
        _check(_lib.load().sxb_moe_layer_two_streams(C.byref(a), _stream(stream), _stream(side)))


# ---- expert parallelism over the C ABI (no counterpart in the reference) ------------------------------------------

def ep_unique_id() -> bytes:
    buf = (C.c_uint8 * 128)()
    _check(_lib.load().sxb_ep_unique_id(buf))
    return bytes(buf)


class EpContext:
    """A rank's expert-parallel context (sxb_ep_create): NCCL communicator, exchange buffers, peer mappings.
    return_path: 0 reduce-scatter, 1 peer stores of FP32 pieces, 2 of F16 pieces."""

    def __init__(self, unique_id: bytes, world: int, rank: int, T: int, d: int, A: int, return_path: int = 1):
        self.handle = C.c_void_p()
        idb = (C.c_uint8 * 128).from_buffer_copy(unique_id)
        _check(_lib.load().sxb_ep_create(idb, world, rank, T, d, A, return_path, C.byref(self.handle)))
        self.world, self.rank, self.T, self.return_path = world, rank, T, return_path

    def layer(self, x_loc, logits_loc, y_loc, gate_up: QDeviceView, down: QDeviceView, E_local, E_total, e_lo, A, ids, coef, ws,
              ws_bytes, h, partial, router_err, expert_err, xs=None, math=None, stream=None):
        """sxb_moe_layer_ep on this rank's rows; ids / coef / ws / h / partial / xs are sized for all T rows."""
        a, keep = _layer_args(x_loc, logits_loc, y_loc, gate_up, down, E_local, A, ids, coef, ws, ws_bytes, h, partial, router_err,
                              expert_err, xs, math, E_total, e_lo, None, None, None, None, None, None)
        _count(9)
        _check(_lib.load().sxb_moe_layer_ep(self.handle, C.byref(a), _stream(stream)))

    def set_timing(self, on: bool):
        _check(_lib.load().sxb_ep_set_timing(self.handle, int(on)))

    def timing(self) -> dict:
        ms = (C.c_float * 5)()
        n = C.c_int()
        _check(_lib.load().sxb_ep_timing(self.handle, ms, C.byref(n)))
        names = ("route", "gather_wait", "experts", "return", "sum")
        return {"layers": n.value, **{k: float(v) for k, v in zip(names, ms)}}

    def close(self):
        if self.handle:
            _lib.load().sxb_ep_destroy(self.handle)
            self.handle = C.c_void_p()
