"""Writes stay inside the outputs, and offsets beyond 2^31 elements are right.

The C entry points are called on buffers with guard values on both sides of
every output, at ragged sizes; the large cases check sampled rows against the
64-bit forms (bounds as in the operators' own tests)."""
import ctypes

import pytest
import torch

from oracle import operators as O
from swiglu_b200 import _lib, ops

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24
GUARD = 256


class Guarded:
    """A buffer of `numel` elements with guards around it."""

    def __init__(self, numel, dtype):
        size = torch.empty(0, dtype=dtype).element_size()
        self.raw = torch.full((numel * size + 2 * GUARD,), 0xA5, dtype=torch.uint8, device=DEV)
        self.bytes = numel * size
        self.t = self.raw[GUARD:GUARD + self.bytes].view(dtype)
        self.ptr = self.t.data_ptr()

    def intact(self):
        return bool((self.raw[:GUARD] == 0xA5).all()) and bool((self.raw[GUARD + self.bytes:] == 0xA5).all())


def _code(dt):
    return _lib.F32 if dt == F32 else _lib.BF16


@pytest.mark.parametrize("M,D", [(1, 1), (1, 7), (3, 33), (5, 1001), (2, 4099), (37, 264), (9, 3584), (2, 65544), (700, 520), (1201, 1029), (1203, 4100)])
@pytest.mark.parametrize("dt", [BF, F32])
def test_norm_writes_stay_inside(M, D, dt):
    x, r = torch.randn(M, D, device=DEV).to(dt), torch.randn(M, D, device=DEV).to(dt)
    w = torch.ones(D, device=DEV, dtype=dt)
    y, s, rstd = Guarded(M * D, dt), Guarded(M * D, dt), Guarded(M, F32)
    q, sc = Guarded(M * D, torch.uint8), Guarded(M, F32)
    eps = ctypes.byref(ctypes.c_float(1e-6))
    _lib.call("swiglu_b200_rmsnorm_fwd", x.data_ptr(), r.data_ptr(), w.data_ptr(), y.ptr, s.ptr, rstd.ptr, M, D, eps,
              _code(dt), _code(dt), None)
    _lib.call("swiglu_b200_rmsnorm_fwd_e4m3", x.data_ptr(), r.data_ptr(), w.data_ptr(), q.ptr, sc.ptr, s.ptr, rstd.ptr,
              M, D, eps, _code(dt), _code(dt), None)
    n = ctypes.c_int64(0)
    _lib.call("swiglu_b200_rmsnorm_bwd_workspace", M, D, ops._num_sms(0), ctypes.byref(n))
    ws, dx, dw = Guarded(n.value, F32), Guarded(M * D, dt), Guarded(D, dt)
    _lib.call("swiglu_b200_rmsnorm_bwd", r.data_ptr(), s.ptr, w.data_ptr(), rstd.ptr, x.data_ptr(), dx.ptr, dw.ptr,
              ws.ptr, n.value, M, D, _code(dt), _code(dt), None)
    torch.cuda.synchronize()
    for b in (y, s, rstd, q, sc, ws, dx, dw):
        assert b.intact()
    with pytest.raises(_lib.SwigluError, match="workspace"):
        _lib.call("swiglu_b200_rmsnorm_bwd", r.data_ptr(), s.ptr, w.data_ptr(), rstd.ptr, x.data_ptr(), dx.ptr, dw.ptr,
                  ws.ptr, n.value - 1, M, D, _code(dt), _code(dt), None)


@pytest.mark.parametrize("R,K", [(1, 32), (65, 96), (129, 288), (63, 3616), (200, 512)])
@pytest.mark.parametrize("dt", [BF, F32])
def test_mxfp4_writes_stay_inside(R, K, dt):
    t = torch.randn(R, K, device=DEV).to(dt)
    shape = ops.mxfp4_scale_shape(R, K)
    q, sc, back = Guarded(R * K // 2, torch.uint8), Guarded(shape[0] * shape[1] * 512, torch.uint8), Guarded(R * K, dt)
    _lib.call("swiglu_b200_quantize_mxfp4", t.data_ptr(), q.ptr, sc.ptr, R, K, _code(dt), None)
    _lib.call("swiglu_b200_dequantize_mxfp4", q.ptr, sc.ptr, back.ptr, R, K, _code(dt), None)
    for M, out in ((1, F32), (7, BF), (130, F32), (700, BF)):
        a, asc = ops.quantize_mxfp4(torch.randn(M, K, device=DEV))
        N = -(-R // 8) * 8
        b, bsc = ops.quantize_mxfp4(torch.randn(N, K, device=DEV))
        c = Guarded(M * N, out)
        _lib.call("swiglu_b200_matmul_mxfp4", a.data_ptr(), asc.data_ptr(), b.data_ptr(), bsc.data_ptr(), c.ptr, M, N, K,
                  _code(out), None)
        torch.cuda.synchronize()
        assert c.intact()
    torch.cuda.synchronize()
    assert q.intact() and sc.intact() and back.intact()
    assert ops.device_status(0) == 0


def test_norm_beyond_2_31_elements():
    M, D = 270000, 8192                      # 2.2e9 elements
    x = torch.empty(M, D, device=DEV, dtype=BF)
    for i in range(0, M, 30000):
        x[i:i + 30000] = torch.randn(30000, D, device=DEV)
    w = (1 + 0.1 * torch.randn(D, device=DEV)).to(BF)
    y, s, rstd = ops.rmsnorm_fwd(x, w)
    q, scale, _, _ = ops.rmsnorm_fwd_e4m3(x, w)
    rows = torch.tensor([0, 1, 131071, 262143, 262144, 262145, M - 1])
    ry, _, rr = O.rmsnorm(x[rows].cpu(), w.cpu())
    steps = (D / 32 + 48) * U
    assert torch.all((y[rows].cpu().double() - ry).abs() <= (2 ** -8 + steps) * ry.abs())
    assert torch.all((rstd[rows].cpu().double() - rr).abs() <= steps * rr)
    v = q[rows].float().cpu().double() * scale[rows].cpu().double()[:, None]
    assert torch.all((v - ry).abs() <= torch.maximum(ry.abs() * 2 ** -4, scale[rows].cpu().double()[:, None] * 2 ** -10)
                     * (1 + 2 * steps) + 2 * steps * ry.abs())
    del q, y
    dx, dw = ops.rmsnorm_bwd(x, x, w, rstd)
    rx, _ = O.rmsnorm_grad(x[rows].cpu(), x[rows].cpu(), w.cpu(), rstd[rows].cpu())
    size = (x[rows].cpu().double() * w.cpu().double()).abs() * rr[:, None] * 40
    assert torch.all((dx[rows].cpu().double() - rx).abs() <= 2 ** -8 * rx.abs() + steps * size)
    del dx
    n = ops.grad_norm([x])
    want = sum(x[i:i + 30000].double().square().sum() for i in range(0, M, 30000)).sqrt().cpu()
    assert abs(n.cpu().double() - want) <= 34 * U * want
    keep = x[rows].clone()
    ops.clip_grad_norm_([x], 0.5 * float(want))
    assert torch.all((x[rows].float() - 0.5 * keep.float()).abs() <= (2 ** -8 + 2.0 ** -18) * 0.5 * keep.float().abs())


def test_mxfp4_beyond_2_31_elements():
    R, K = 300000, 8192
    t = torch.empty(R, K, device=DEV, dtype=BF)
    for i in range(0, R, 30000):
        t[i:i + 30000] = torch.randn(30000, K, device=DEV)
    q, scale = ops.quantize_mxfp4(t)
    back = ops.dequantize_mxfp4(q, scale)
    rows = torch.tensor([0, 127, 128, 262143, 262144, R - 1])
    want = O.mx_values(*O.mx_quantize(t[rows].cpu()))
    assert torch.equal(back[rows].cpu().double(), want)
    del back, t
    b, bsc = ops.quantize_mxfp4(torch.randn(7168, K, device=DEV) * K ** -0.5)
    c = ops.matmul_mxfp4(q, scale, b, bsc)                     # 2.15e9 outputs
    bv = ops.dequantize_mxfp4(b, bsc, dtype=F32).double().cpu()
    ref, mass = want @ bv.t(), want.abs() @ bv.abs().t()
    assert torch.all((c[rows].cpu().double() - ref).abs() <= 2 ** -8 * ref.abs() + (K / 64 + 8) * 2.0 ** -22 * mass)
    assert ops.device_status(0) == 0
