"""Tensor-level wrappers over the C ABI.

Each function takes contiguous CUDA tensors, allocates its outputs through the
torch caching allocator (so `torch.cuda.max_memory_allocated` accounts for
them, as it does for the reference's `torch.empty` outputs,
fused_forward.py:216-217), makes the tensors' device current and enqueues the
native kernels on that device's current torch stream.
"""
from __future__ import annotations

import ctypes
from array import array
from functools import lru_cache
from operator import attrgetter

import torch

from . import _lib
from ._lib import BF16, F32, LAYOUT_PACKED128, LAYOUT_STD, W1_ROWS, W1_T  # noqa: F401

# Tile-order group (in 128-row tiles) where the caller passes none; the value
# the C side uses for the GEMMs it launches without one (kDefaultGroupM).
DEFAULT_GROUP_M = 32


def dtype_code(dtype: torch.dtype) -> int:
    if dtype == torch.bfloat16:
        return BF16
    if dtype == torch.float32:
        return F32
    raise TypeError(f"swiglu_b200 supports torch.bfloat16 and torch.float32, got {dtype}")


def _p(t: torch.Tensor | None) -> ctypes.c_void_p:
    return ctypes.c_void_p(0 if t is None else t.data_ptr())


# Stream-K workspace per (device index, stream handle): registered with the
# library the first time a stream is used, zero-filled by a memset ordered on
# that stream, and kept for the life of the process.
STREAM_WORKSPACE_BYTES = 48 << 20
_workspaces: dict[tuple[int, int], torch.Tensor] = {}
_stream_k = True


def _stream(dev: torch.device) -> ctypes.c_void_p:
    """Handle of `dev`'s current torch stream (the caller has made `dev`
    current), with its stream-K workspace registered."""
    s = torch.cuda.current_stream(dev).cuda_stream
    key = (dev.index, s)
    # No registration inside a graph capture: the buffer would belong to the
    # graph's private memory pool.
    if _stream_k and key not in _workspaces and not torch.cuda.is_current_stream_capturing():
        buf = torch.zeros(STREAM_WORKSPACE_BYTES, dtype=torch.uint8, device=dev)
        _lib.call("swiglu_b200_set_stream_workspace", _p(buf), buf.numel(), ctypes.c_void_p(s))
        _workspaces[key] = buf
    return ctypes.c_void_p(s)


# How the backward forms dW2 (read by the recompute Functions and the
# tensor-parallel block):
#   "prologue"  (default) dW2 recomputes h inside its operand prologue, before
#               the grad_h GEMM overwrites preact: no [M, H] buffer anywhere
#               in the backward (swiglu_recompute.py:71-73 without the h
#               temporary the reference materialises);
#   "emit_h"    the grad_h GEMM's epilogue also writes h of the preact it
#               replaces to a transient [M, H] buffer and dW2 = grad_y^T h is
#               a plain GEMM: faster by the difference of the two dW2 kernels
#               (about 0.26 ms of a 7.8 ms step at M=11136 D=3584 H=14336),
#               for one [M, H] buffer between the two GEMMs.
DW2_MODES = ("prologue", "emit_h")
_dw2_mode = "prologue"


def set_dw2_mode(mode: str) -> None:
    global _dw2_mode
    if mode not in DW2_MODES:
        raise ValueError(f"dW2 mode must be one of {DW2_MODES}, got {mode!r}")
    _dw2_mode = mode


def dw2_mode() -> str:
    return _dw2_mode


def set_stream_k(enabled: bool) -> None:
    """Enables (default) or disables the stream-K tail of the 2-SM GEMMs for
    later calls. Disabling unregisters every workspace this module registered;
    the kernels then run unsplit (results differ in f32 summation order)."""
    global _stream_k
    _stream_k = bool(enabled)
    if not enabled:
        for (index, s) in list(_workspaces):
            with torch.cuda.device(index):
                _lib.call("swiglu_b200_set_stream_workspace", None, 0, ctypes.c_void_p(s))
                torch.cuda.synchronize()
        _workspaces.clear()


# Launch trace: with a list installed by trace_launches(), every kernel entry
# point called through this module also records a CUDA event before and after
# its launch on the launching stream and appends (entry point, start, end).
# The events cost no device time worth measuring, so a caller (bench.py) can
# time each kernel inside the very steps it times as a whole.
_trace: list | None = None


def trace_launches(records: list | None) -> None:
    """Install `records` (a list) to collect (entry point, start event, end
    event) per launch from now on; None stops tracing."""
    global _trace
    _trace = records


def _call(dev: torch.device, name: str, *args) -> None:
    if _trace is None:
        _lib.call(name, *args)
        return
    st = torch.cuda.current_stream(dev)
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    e0.record(st)
    _lib.call(name, *args)
    e1.record(st)
    _trace.append((name, e0, e1))


def _check_cuda(*ts: torch.Tensor) -> torch.device:
    dev = None
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError("swiglu_b200 kernels take CUDA tensors (there is no CPU path)")
        if not t.is_contiguous():
            raise ValueError("swiglu_b200 kernels take contiguous tensors")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError(f"tensors on different devices: {dev} vs {t.device}")
    return dev


def _same_dtype(*ts: torch.Tensor) -> torch.dtype:
    dt = None
    for t in ts:
        if t is None:
            continue
        if dt is None:
            dt = t.dtype
        elif t.dtype != dt:
            raise TypeError(f"mixed dtypes {dt} and {t.dtype}")
    return dt


def swiglu_fwd(x: torch.Tensor, w: torch.Tensor, *, w_form: int, layout: int,
               h_from_rounded: bool, want_h: bool = True, want_preact: bool = True,
               group_size_m: int = DEFAULT_GROUP_M, preact_out: torch.Tensor | None = None,
               h_out: torch.Tensor | None = None):
    """(preact [M, 2H] or None, h [M, H] or None) for preact = x . W1^T in one
    launch. want_preact=False is the no-save (inference) forward. preact_out /
    h_out: contiguous buffers to write into instead of new ones."""
    assert want_h or want_preact
    dev = _check_cuda(x, w, preact_out, h_out)
    dt = _same_dtype(x, w, preact_out, h_out)
    M, K = x.shape
    if w_form == W1_ROWS:
        n2, K2 = w.shape
    else:
        K2, n2 = w.shape
    assert K == K2 and n2 % 2 == 0, f"shape mismatch x{tuple(x.shape)} w{tuple(w.shape)}"
    H = n2 // 2
    if preact_out is not None:
        assert want_preact and preact_out.shape == (M, n2)
    if h_out is not None:
        assert want_h and h_out.shape == (M, H)
    preact = (preact_out if preact_out is not None else torch.empty((M, n2), device=dev, dtype=dt)) \
        if want_preact else None
    h = (h_out if h_out is not None else torch.empty((M, H), device=dev, dtype=dt)) if want_h else None
    with torch.cuda.device(dev):
        _call(dev, "swiglu_b200_fused_matmul_swiglu_save_preact", _p(x), _p(w), _p(preact), _p(h),
              M, K, H, dtype_code(dt), w_form, layout, int(bool(h_from_rounded)),
              int(group_size_m), _stream(dev))
    return preact, h


def matmul(a: torch.Tensor, b: torch.Tensor, *, a_t: bool, b_t: bool,
           out_dtype: torch.dtype | None = None, out: torch.Tensor | None = None,
           group_size_m: int = DEFAULT_GROUP_M, tile_n: int = 0) -> torch.Tensor:
    """C = op(a) . op(b); op(a) = a.T if a_t, op(b) = b.T if b_t. tile_n = 512
    asks the 2-SM kernel for 256 x 512 output tiles (long-K GEMMs), 256 for
    256 x 256; 0 chooses by size (512 from 8 waves of 256 x 512 tiles)."""
    dev = _check_cuda(a, b, out)
    dt = _same_dtype(a, b)
    M, K = (a.shape[1], a.shape[0]) if a_t else tuple(a.shape)
    Kb, N = (b.shape[1], b.shape[0]) if b_t else tuple(b.shape)
    assert K == Kb, f"inner dimensions differ: {K} vs {Kb}"
    odt = out_dtype or dt
    if out is None:
        out = torch.empty((M, N), device=dev, dtype=odt)
    else:
        assert out.shape == (M, N) and out.dtype == odt
    with torch.cuda.device(dev):
        _call(dev, "swiglu_b200_matmul_tiled", _p(a), _p(b), _p(out), M, N, K, int(a_t), int(b_t),
              dtype_code(dt), dtype_code(odt), int(group_size_m), int(tile_n), _stream(dev))
    return out


def bwd_dw2(grad_y: torch.Tensor, preact: torch.Tensor, *, layout: int,
            out: torch.Tensor | None = None) -> torch.Tensor:
    """dW2 [Dout, H] = grad_y^T . swiglu(preact), h recomputed in the GEMM prologue."""
    dev = _check_cuda(grad_y, preact, out)
    dt = _same_dtype(grad_y, preact)
    M, Dout = grad_y.shape
    M2, n2 = preact.shape
    assert M == M2 and n2 % 2 == 0
    H = n2 // 2
    if out is None:
        out = torch.empty((Dout, H), device=dev, dtype=dt)
    with torch.cuda.device(dev):
        _call(dev, "swiglu_b200_bwd_dw2", _p(grad_y), _p(preact), _p(out), M, H, Dout,
              dtype_code(dt), layout, _stream(dev))
    return out


def bwd_grad_preact_inplace(grad_y: torch.Tensor, w2: torch.Tensor, preact: torch.Tensor, *,
                            layout: int, h_out: torch.Tensor | None = None) -> torch.Tensor:
    """preact <- grad_preact, from grad_h = grad_y . W2 formed tile by tile (never stored).
    With `h_out` ([M, H]) the same epilogue also writes h = swiglu(preact) of
    the values it replaces."""
    dev = _check_cuda(grad_y, w2, preact, h_out)
    dt = _same_dtype(grad_y, w2, preact, h_out)
    M, Dout = grad_y.shape
    Dout2, H = w2.shape
    assert Dout == Dout2 and preact.shape == (M, 2 * H)
    with torch.cuda.device(dev):
        if h_out is None:
            _call(dev, "swiglu_b200_bwd_grad_preact_inplace", _p(grad_y), _p(w2), _p(preact), M, H, Dout,
                  dtype_code(dt), layout, _stream(dev))
        else:
            assert h_out.shape == (M, H)
            _call(dev, "swiglu_b200_bwd_grad_preact_inplace_emit_h", _p(grad_y), _p(w2), _p(preact),
                  _p(h_out), M, H, Dout, dtype_code(dt), layout, _stream(dev))
    return preact


def forward_logic(preact: torch.Tensor, *, layout: int) -> torch.Tensor:
    dev = _check_cuda(preact)
    M, n2 = preact.shape
    assert n2 % 2 == 0
    H = n2 // 2
    h = torch.empty((M, H), device=dev, dtype=preact.dtype)
    with torch.cuda.device(dev):
        _call(dev, "swiglu_b200_forward_logic", _p(preact), _p(h), M, H, dtype_code(preact.dtype),
              layout, _stream(dev))
    return h


def backward_logic(preact: torch.Tensor, grad_h: torch.Tensor, *, layout: int,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    dev = _check_cuda(preact, grad_h, out)
    dt = _same_dtype(preact, grad_h)
    M, n2 = preact.shape
    H = n2 // 2
    assert grad_h.shape == (M, H), f"grad_h {tuple(grad_h.shape)} vs preact {tuple(preact.shape)}"
    if out is None:
        out = torch.empty_like(preact)
    with torch.cuda.device(dev):
        _call(dev, "swiglu_b200_backward_logic", _p(preact), _p(grad_h), _p(out), M, H, dtype_code(dt),
              layout, _stream(dev))
    return out


def pack_chunked(w: torch.Tensor, block_n_half: int, *, unpack: bool) -> torch.Tensor:
    dev = _check_cuda(w)
    K, n2 = w.shape
    out = torch.empty_like(w)
    with torch.cuda.device(dev):
        _call(dev, "swiglu_b200_pack_weight_chunked", _p(w), _p(out), K, n2 // 2, int(block_n_half),
              dtype_code(w.dtype), int(bool(unpack)), _stream(dev))
    return out


def device_status(device: torch.device | int | None = None, clear: bool = True) -> int:
    """Pipeline-timeout bits recorded by the kernels on `device` (0 = healthy)."""
    with torch.cuda.device(device if device is not None else torch.cuda.current_device()):
        return _lib.device_status(clear)


# ------------------------------------------------------------ e4m3 (FP8) path
def quantize_rows_e4m3(t: torch.Tensor):
    """(q, scale): row-scaled e4m3 copy of a bf16 [R, C] matrix, q [R, C]
    (torch.float8_e4m3fn) and the f32 dequantisation factor scale [R]
    (row r holds e4m3(v * 448 / amax_r), scale_r = amax_r / 448)."""
    dev = _check_cuda(t)
    if t.dtype != torch.bfloat16 or t.dim() != 2:
        raise TypeError("quantize_rows_e4m3 takes a 2-D bf16 tensor")
    R, C = t.shape
    q = torch.empty((R, C), device=dev, dtype=torch.float8_e4m3fn)
    s = torch.empty((R,), device=dev, dtype=torch.float32)
    with torch.cuda.device(dev):
        _call(dev, "swiglu_b200_quantize_rows_e4m3", _p(t), _p(q), _p(s), R, C, BF16, _stream(dev))
    return q, s


def swiglu_fwd_e4m3(xq: torch.Tensor, x_scale: torch.Tensor, wq: torch.Tensor, w_scale: torch.Tensor, *,
                    layout: int, h_from_rounded: bool, want_h: bool = True, want_preact: bool = True,
                    group_size_m: int = DEFAULT_GROUP_M):
    """(preact [M, 2H] or None, h [M, H] or None) in bf16 from e4m3 x [M, K]
    and W1 [2H, K] (rows in `layout` order) with their row scales."""
    assert want_h or want_preact
    dev = _check_cuda(xq, x_scale, wq, w_scale)
    M, K = xq.shape
    n2, K2 = wq.shape
    assert K == K2 and n2 % 2 == 0 and x_scale.shape == (M,) and w_scale.shape == (n2,)
    H = n2 // 2
    preact = torch.empty((M, n2), device=dev, dtype=torch.bfloat16) if want_preact else None
    h = torch.empty((M, H), device=dev, dtype=torch.bfloat16) if want_h else None
    with torch.cuda.device(dev):
        _call(dev, "swiglu_b200_fused_matmul_swiglu_e4m3", _p(xq), _p(x_scale), _p(wq), _p(w_scale),
              _p(preact), _p(h), M, K, H, layout, int(bool(h_from_rounded)), int(group_size_m), _stream(dev))
    return preact, h


def matmul_e4m3(aq: torch.Tensor, a_scale: torch.Tensor, bq: torch.Tensor, b_scale: torch.Tensor, *,
                out_dtype: torch.dtype = torch.bfloat16, group_size_m: int = DEFAULT_GROUP_M) -> torch.Tensor:
    """C [M, N] = A . B^T for e4m3 A [M, K] and B [N, K] with their row scales."""
    dev = _check_cuda(aq, a_scale, bq, b_scale)
    M, K = aq.shape
    N, K2 = bq.shape
    assert K == K2 and a_scale.shape == (M,) and b_scale.shape == (N,)
    out = torch.empty((M, N), device=dev, dtype=out_dtype)
    with torch.cuda.device(dev):
        _call(dev, "swiglu_b200_matmul_e4m3", _p(aq), _p(a_scale), _p(bq), _p(b_scale), _p(out), M, N, K,
              dtype_code(out_dtype), int(group_size_m), _stream(dev))
    return out


# ----------------------------------------------------------- helpers of the calls below
# These calls are also made for single tokens, where the host's time is what a
# user waits for: outputs come from new_empty (0.5 us less than torch.empty with
# keywords), checks take one pass, sizes of workspaces are looked up once.
_CODES = {torch.bfloat16: BF16, torch.float32: F32}


def _launch(dev: torch.device, name: str, *args) -> None:
    """`name(*args, stream)` with `dev` current, on its current torch stream."""
    index = dev.index
    stream = torch._C._cuda_getCurrentRawStream(index)
    if torch._C._cuda_getDevice() != index:
        with torch.cuda.device(dev):
            _call(dev, name, *args, stream)
    elif _trace is not None:
        _call(dev, name, *args, stream)
    else:
        status = getattr(_lib.load(), name)(*args, stream)
        if status:
            _lib.check(status)


@lru_cache(maxsize=None)
def _num_sms(index: int) -> int:
    return torch.cuda.get_device_properties(index).multi_processor_count


def _query(name: str, *args) -> int:
    n = ctypes.c_int64(0)
    _lib.call(name, *args, ctypes.byref(n))
    return n.value


@lru_cache(maxsize=1024)
def _rmsnorm_bwd_floats(M: int, D: int, sms: int) -> int:
    return _query("swiglu_b200_rmsnorm_bwd_workspace", M, D, sms)


@lru_cache(maxsize=1024)
def _grad_norm_doubles(count: int, sms: int) -> int:
    return _query("swiglu_b200_grad_norm_workspace", count, sms)


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


# ------------------------------------------------------------ residual RMS norm
def _check_norm(x: torch.Tensor, weight: torch.Tensor, *same: torch.Tensor | None):
    """(device, M, D, dtype codes of x and weight) of a norm's arguments; `same`
    are the tensors of x's shape and type."""
    shape, dtype, dev = x.shape, x.dtype, x.device
    ok = len(shape) == 2 and shape[1] >= 1 and weight.shape == shape[1:]
    ok = ok and x.is_cuda and x.is_contiguous() and weight.device == dev and weight.is_contiguous()
    for t in same:
        if t is not None:
            ok = ok and t.shape == shape and t.dtype == dtype and t.device == dev and t.is_contiguous()
    if not ok:
        _check_cuda(x, weight, *same)
        if len(shape) != 2 or shape[1] < 1:
            raise ValueError(f"the norm takes rows [M, D] with D >= 1, got {tuple(shape)}")
        if weight.shape != shape[1:]:
            raise ValueError(f"weight {tuple(weight.shape)} does not match rows of {shape[1]}")
        for t in same:
            if t is not None and t.shape != shape:
                raise ValueError(f"shapes differ: {tuple(t.shape)} and {tuple(shape)}")
        _same_dtype(x, *same)
    return dev, shape[0], shape[1], dtype_code(dtype), dtype_code(weight.dtype)


def rmsnorm_fwd(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, *, eps: float = 1e-6):
    """(y, s, rstd): the residual RMS norm of rows x [M, D] (bf16 or f32).
    s = x + residual rounded to x's dtype (x itself without a residual),
    rstd [M] = (mean s^2 + eps)^-1/2 in f32, y = s * rstd * weight in x's dtype.
    weight [D] may be bf16 or f32."""
    dev, M, D, dt, wdt = _check_norm(x, weight, residual)
    y = torch.empty_like(x)
    s = x if residual is None else torch.empty_like(x)
    rstd = x.new_empty(M, dtype=torch.float32)
    _launch(dev, "swiglu_b200_rmsnorm_fwd", x.data_ptr(), _ptr(residual), weight.data_ptr(), y.data_ptr(),
            s.data_ptr(), rstd.data_ptr(), M, D, ctypes.byref(ctypes.c_float(float(eps))), dt, wdt)
    return y, s, rstd


def rmsnorm_fwd_e4m3(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, *,
                     eps: float = 1e-6):
    """(q, scale, s, rstd): rmsnorm_fwd with y as row-scaled e4m3 (q [M, D],
    f32 scale [M], as quantize_rows_e4m3 gives them, but from the f32 y)."""
    dev, M, D, dt, wdt = _check_norm(x, weight, residual)
    q = x.new_empty((M, D), dtype=torch.float8_e4m3fn)
    scale = x.new_empty(M, dtype=torch.float32)
    s = x if residual is None else torch.empty_like(x)
    rstd = torch.empty_like(scale)
    _launch(dev, "swiglu_b200_rmsnorm_fwd_e4m3", x.data_ptr(), _ptr(residual), weight.data_ptr(), q.data_ptr(),
            scale.data_ptr(), s.data_ptr(), rstd.data_ptr(), M, D, ctypes.byref(ctypes.c_float(float(eps))), dt, wdt)
    return q, scale, s, rstd


def rmsnorm_bwd(dy: torch.Tensor, s: torch.Tensor, weight: torch.Tensor, rstd: torch.Tensor,
                ds: torch.Tensor | None = None):
    """(dx, dweight) of the norm: dx [M, D] is the gradient of x and of the
    residual alike (ds, the gradient of s from its other uses, is added),
    dweight [D] in weight's dtype. s and rstd as the forward returned them."""
    dev, M, D, dt, wdt = _check_norm(s, weight, dy, ds)
    if rstd.device != dev or rstd.dtype != torch.float32 or rstd.shape != (M,) or not rstd.is_contiguous():
        raise ValueError("rstd must be the forward's f32 [M] tensor")
    dx = torch.empty_like(s)
    dweight = torch.empty_like(weight)
    floats = _rmsnorm_bwd_floats(M, D, _num_sms(dev.index))
    ws = s.new_empty(floats, dtype=torch.float32)
    _launch(dev, "swiglu_b200_rmsnorm_bwd", dy.data_ptr(), s.data_ptr(), weight.data_ptr(), rstd.data_ptr(),
            _ptr(ds), dx.data_ptr(), dweight.data_ptr(), ws.data_ptr(), floats, M, D, dt, wdt)
    return dx, dweight


# --------------------------------------------------- gradient norm and clipping
def _check_dense(t: torch.Tensor, dev: torch.device) -> None:
    """Raises unless t's values fill one stretch of memory of `dev`, in whatever
    order of dimensions."""
    if not t.is_cuda:
        raise ValueError("swiglu_b200 kernels take CUDA tensors (there is no CPU path)")
    if t.device != dev:
        raise ValueError(f"tensors on different devices: {dev} vs {t.device}")
    if not t.permute(sorted(range(t.dim()), key=t.stride, reverse=True)).is_contiguous():
        raise ValueError("a gradient's values must fill one stretch of memory")


_dtype_of, _shape_of = attrgetter("dtype"), attrgetter("shape")


class _GradList:
    """Host arrays of a list of gradients, checked. (With map() over the methods
    instead of a loop over the tensors: 0.3 us less a tensor.)"""

    def __init__(self, tensors, out=None):
        T = torch.Tensor
        tensors = self.tensors = list(tensors)
        if not tensors:
            raise ValueError("no gradients given")
        dev = self.dev = tensors[0].device
        index = tensors[0].get_device()  # -1 on the CPU
        contiguous = all(map(T.is_contiguous, tensors))
        if index < 0 or not contiguous or any(map(index.__ne__, map(T.get_device, tensors))):
            for t in tensors:
                _check_dense(t, dev)
        dtypes = list(map(_dtype_of, tensors))
        try:
            self.dtypes = array("i", map(_CODES.__getitem__, dtypes))
        except KeyError as e:
            dtype_code(e.args[0])  # raises
        self.sizes = array("q", map(T.numel, tensors))
        self.grads = array("Q", map(T.data_ptr, tensors))
        self.out, self.outs = tensors, self.grads
        if out is not None:
            out = self.out = list(out)
            if len(out) != len(tensors):
                raise ValueError(f"{len(out)} outputs for {len(tensors)} gradients")
            if list(map(_shape_of, out)) != list(map(_shape_of, tensors)) or list(map(_dtype_of, out)) != dtypes:
                raise ValueError("an output differs from its gradient in shape or dtype")
            if (not contiguous or not all(map(T.is_contiguous, out))
                    or any(map(index.__ne__, map(T.get_device, out)))):
                for t, o in zip(tensors, out):
                    _check_dense(o, dev)
                    if o.stride() != t.stride():
                        raise ValueError("an output's strides differ from its gradient's")
            self.outs = array("Q", map(T.data_ptr, out))

    def args(self, with_outs: bool):
        a = [self.grads.buffer_info()[0]]
        if with_outs:
            a.append(self.outs.buffer_info()[0])
        return (*a, self.sizes.buffer_info()[0], self.dtypes.buffer_info()[0], len(self.tensors))

    def workspace(self) -> torch.Tensor:
        doubles = _grad_norm_doubles(len(self.tensors), _num_sms(self.dev.index))
        return self.tensors[0].new_empty(doubles, dtype=torch.float64)

    def norm(self) -> torch.Tensor:
        return self.tensors[0].new_empty((), dtype=torch.float32)

    def written(self) -> None:
        torch.autograd.graph.increment_version(self.out)


def grad_norm(tensors) -> torch.Tensor:
    """The 2-norm (f32, a 0-dim tensor on their device) of all the values of a
    list of bf16 / f32 tensors on one device (contiguous in some order of their
    dimensions)."""
    g = _GradList(tensors)
    norm = g.norm()
    ws = g.workspace()
    _launch(g.dev, "swiglu_b200_grad_norm", *g.args(False), ws.data_ptr(), ws.numel(), norm.data_ptr())
    return norm


def clip_grad_norm_(tensors, max_norm: float, *, out=None) -> torch.Tensor:
    """Scales the gradients by min(1, max_norm / (norm + 1e-6)), norm being
    grad_norm(tensors), and returns the norm (before clipping, on the device:
    nothing here waits for it). In place, or into the tensors `out`. A tensor
    that is written may not share memory with another one of the call."""
    g = _GradList(tensors, out)
    norm = g.norm()
    ws = g.workspace()
    _launch(g.dev, "swiglu_b200_clip_grad_norm", *g.args(True), ctypes.byref(ctypes.c_double(float(max_norm))),
            ws.data_ptr(), ws.numel(), norm.data_ptr())
    g.written()
    return norm


def clip_grads_by_norm_(tensors, norm: torch.Tensor, max_norm: float, *, out=None) -> None:
    """clip_grad_norm_ with a norm that is already known: an f32 tensor of one
    value on the gradients' device (reduced over ranks, for instance)."""
    g = _GradList(tensors, out)
    if norm.device != g.dev or norm.dtype != torch.float32 or norm.numel() != 1:
        raise ValueError("norm must be one f32 value on the gradients' device")
    _launch(g.dev, "swiglu_b200_clip_grads_by_norm", *g.args(True), norm.data_ptr(),
            ctypes.byref(ctypes.c_double(float(max_norm))))
    g.written()


# ------------------------------------------------------------------- MXFP4 path
def mxfp4_scale_shape(rows: int, cols: int) -> tuple[int, int, int, int, int]:
    """Shape of the scale tensor of a [rows, cols] MXFP4 matrix: tiles of 128
    rows by 4 blocks; the byte of (row, block) is element [row // 128,
    block // 4, row % 32, (row % 128) // 32, block % 4]."""
    return (-(-rows // 128), -(-cols // 128), 32, 4, 4)


def _check_mx(q: torch.Tensor, scale: torch.Tensor) -> tuple[int, int]:
    if q.dtype != torch.uint8 or scale.dtype != torch.uint8 or q.dim() != 2:
        raise TypeError("an MXFP4 matrix is a uint8 [R, K / 2] tensor of codes and a uint8 tensor of scales")
    R, K = q.shape[0], 2 * q.shape[1]
    if scale.shape != mxfp4_scale_shape(R, K):
        raise ValueError(f"scales {tuple(scale.shape)} do not fit a [{R}, {K}] matrix: {mxfp4_scale_shape(R, K)}")
    return R, K


def quantize_mxfp4(t: torch.Tensor):
    """(q, scale): MXFP4 copy of a bf16 or f32 [R, K] matrix, K % 32 == 0: q
    uint8 [R, K / 2] (two e2m1 codes a byte, the even column low) and the e8m0
    scale bytes in the product's tiles (mxfp4_scale_shape)."""
    dev = _check_cuda(t)
    if t.dim() != 2:
        raise ValueError(f"quantize_mxfp4 takes a matrix, got {tuple(t.shape)}")
    R, K = t.shape
    if K % 32:
        raise ValueError(f"{K} columns are not a multiple of 32")
    dt = dtype_code(t.dtype)
    q = t.new_empty((R, K // 2), dtype=torch.uint8)
    scale = q.new_empty(mxfp4_scale_shape(R, K))
    _launch(dev, "swiglu_b200_quantize_mxfp4", t.data_ptr(), q.data_ptr(), scale.data_ptr(), R, K, dt)
    return q, scale


def dequantize_mxfp4(q: torch.Tensor, scale: torch.Tensor, *, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The [R, K] values of an MXFP4 matrix, in bf16 or f32 (exact)."""
    dev = _check_cuda(q, scale)
    R, K = _check_mx(q, scale)
    dt = dtype_code(dtype)
    out = q.new_empty((R, K), dtype=dtype)
    _launch(dev, "swiglu_b200_dequantize_mxfp4", q.data_ptr(), scale.data_ptr(), out.data_ptr(), R, K, dt)
    return out


def matmul_mxfp4(aq: torch.Tensor, a_scale: torch.Tensor, bq: torch.Tensor, b_scale: torch.Tensor, *,
                 out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """C [M, N] = A . B^T for MXFP4 A [M, K] and B [N, K] with their scales;
    N % 8 == 0. Scale bytes past the last column must be 0, as quantize_mxfp4
    writes them; those past the last row may hold anything."""
    dev = _check_cuda(aq, a_scale, bq, b_scale)
    M, K = _check_mx(aq, a_scale)
    N, K2 = _check_mx(bq, b_scale)
    if K != K2:
        raise ValueError(f"inner dimensions differ: {K} vs {K2}")
    dt = dtype_code(out_dtype)
    out = aq.new_empty((M, N), dtype=out_dtype)
    _launch(dev, "swiglu_b200_matmul_mxfp4", aq.data_ptr(), a_scale.data_ptr(), bq.data_ptr(), b_scale.data_ptr(),
            out.data_ptr(), M, N, K, dt)
    return out


def swiglu_fwd_mxfp4(xq: torch.Tensor, x_scale: torch.Tensor, wq: torch.Tensor, w_scale: torch.Tensor, *, layout: int,
                     want_h: bool = True, want_preact: bool = True):
    """(preact [M, 2H] or None, h [M, H] or None) in bf16 from MXFP4 x [M, K]
    and W1 [2H, K] (rows in `layout` order); h from the rounded preact.
    H % 128 == 0."""
    assert want_h or want_preact
    dev = _check_cuda(xq, x_scale, wq, w_scale)
    M, K = _check_mx(xq, x_scale)
    n2, K2 = _check_mx(wq, w_scale)
    if K != K2 or n2 % 256:
        raise ValueError(f"x [{M}, {K}] and W1 [{n2}, {K2}]: inner dimensions must agree and H be a multiple of 128")
    H = n2 // 2
    # Few rows take two launches, with preact between them.
    fused = ctypes.c_int(0)
    if not want_preact:
        _lib.call("swiglu_b200_fused_matmul_swiglu_mxfp4_plan", M, K, H, _num_sms(dev.index), ctypes.byref(fused))
    preact = None if fused.value else xq.new_empty((M, n2), dtype=torch.bfloat16)
    h = xq.new_empty((M, H), dtype=torch.bfloat16) if want_h else None
    _launch(dev, "swiglu_b200_fused_matmul_swiglu_mxfp4", xq.data_ptr(), x_scale.data_ptr(), wq.data_ptr(),
            w_scale.data_ptr(), _ptr(preact), _ptr(h), M, K, H, layout)
    return preact if want_preact else None, h
