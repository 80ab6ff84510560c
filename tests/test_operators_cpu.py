"""The C entry points of the norm, MXFP4 and gradient-norm operators refuse bad
calls before they touch a device, and the 64-bit restatements they are tested
against agree with themselves. No GPU."""
import ctypes
from array import array

import pytest
import torch

from oracle import operators as O
from swiglu_b200 import _lib, ops

P = 256


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _eps(v=1e-6):
    return ctypes.byref(ctypes.c_float(v))


def _said(lib, rc, status, text):
    assert rc == status
    assert text in lib.swiglu_b200_last_error_message(), lib.swiglu_b200_last_error_message()


def test_norm_refusals(lib):
    f = lib.swiglu_b200_rmsnorm_fwd
    _said(lib, f(P, None, P, P, P, P, 4, 0, _eps(), 1, 1, None), 1, b"at least one column")
    _said(lib, f(P, None, P, P, P, P, -1, 8, _eps(), 1, 1, None), 1, b"dimensions")
    _said(lib, f(P, None, P, P, P, P, 4, 8, _eps(), 2, 1, None), 1, b"dtype")
    _said(lib, f(P, None, P, P, P, P, 4, 8, _eps(), 1, 9, None), 1, b"dtype")
    _said(lib, f(P, None, P, P, P, P, 4, 8, _eps(-1.0), 1, 1, None), 1, b"eps")
    _said(lib, f(P, None, P, P, P, P, 4, 8, _eps(float("nan")), 1, 1, None), 1, b"eps")
    _said(lib, f(P, None, P, P, P, P, 4, 8, None, 1, 1, None), 1, b"null")
    _said(lib, f(None, None, P, P, P, P, 4, 8, _eps(), 1, 1, None), 1, b"null")
    _said(lib, f(P, P, P, P, None, P, 4, 8, _eps(), 1, 1, None), 1, b"null")       # a residual needs s
    _said(lib, f(P + 1, None, P, P, P, P, 4, 8, _eps(), 1, 1, None), 2, b"aligned")
    assert f(None, None, None, None, None, None, 0, 8, _eps(), 1, 1, None) == 0    # no rows
    g = lib.swiglu_b200_rmsnorm_fwd_e4m3
    _said(lib, g(P, None, P, P, None, P, P, 4, 8, _eps(), 1, 1, None), 1, b"null")
    b = lib.swiglu_b200_rmsnorm_bwd
    _said(lib, b(P, P, P, P, None, P, None, P, 10, 4, 8, 1, 1, None), 1, b"null")
    _said(lib, b(P, P, P, P, None, None, P, P, 10, 4, 8, 1, 1, None), 1, b"null")
    _said(lib, b(P, P, P, P, None, P, P, P + 4, 10, 4, 8, 1, 1, None), 2, b"16 bytes")
    n = ctypes.c_int64(-1)
    assert lib.swiglu_b200_rmsnorm_bwd_workspace(0, 8, 148, ctypes.byref(n)) == 0
    _said(lib, lib.swiglu_b200_rmsnorm_bwd_workspace(4, 0, 148, ctypes.byref(n)), 1, b"positive")


def _arrays(ptrs, sizes, dtypes):
    return array("Q", ptrs), array("q", sizes), array("i", dtypes)


def test_clip_refusals(lib):
    mn = ctypes.byref(ctypes.c_double(1.0))

    def clip(ptrs, outs, sizes, dtypes, max_norm=mn, ws=P, norm=P):
        g, s, d = _arrays(ptrs, sizes, dtypes)
        o = array("Q", outs)
        return lib.swiglu_b200_clip_grad_norm(g.buffer_info()[0], o.buffer_info()[0], s.buffer_info()[0],
                                              d.buffer_info()[0], len(ptrs), max_norm, ws, 1 << 20, norm, None)

    _said(lib, clip([P], [P], [8], [5]), 1, b"dtype")
    _said(lib, clip([P], [P], [-1], [0]), 1, b"size")
    _said(lib, clip([P], [P], [1 << 50], [0]), 1, b"size")
    _said(lib, clip([0], [P], [8], [0]), 1, b"null")
    _said(lib, clip([P], [0], [8], [0]), 1, b"null")
    _said(lib, clip([P + 2], [P + 2], [8], [0]), 2, b"aligned")
    _said(lib, clip([P], [P], [8], [0], norm=None), 1, b"null")
    _said(lib, clip([P], [P], [8], [0], max_norm=None), 1, b"null")
    _said(lib, clip([P], [P], [8], [0], max_norm=ctypes.byref(ctypes.c_double(-0.5))), 1, b"max_norm")
    _said(lib, clip([P], [P], [8], [0], max_norm=ctypes.byref(ctypes.c_double(float("nan")))), 1, b"max_norm")
    _said(lib, clip([P, P], [P, P], [8, 8], [0, 0]), 1, b"overlaps")               # the same tensor twice
    _said(lib, clip([P, 512], [P, P + 28], [8, 8], [0, 0]), 1, b"overlaps")        # two outputs share a value
    _said(lib, clip([P], [P + 4], [8], [0]), 1, b"overlaps")                       # shifted in place
    _said(lib, clip([P, 512], [1024, P], [8, 8], [0, 0]), 1, b"overlaps")          # an output over another's input
    n = ctypes.c_int64(0)
    assert lib.swiglu_b200_grad_norm_workspace(0, 148, ctypes.byref(n)) == 0 and n.value == 1
    assert lib.swiglu_b200_grad_norm_workspace(300, 148, ctypes.byref(n)) == 0 and 3 * 148 <= n.value <= 3 * 148 * 8


def test_mxfp4_refusals(lib):
    q, d, m = lib.swiglu_b200_quantize_mxfp4, lib.swiglu_b200_dequantize_mxfp4, lib.swiglu_b200_matmul_mxfp4
    for f in (q, d):
        _said(lib, f(P, P, P, 4, 40, 1, None), 1, b"multiple of 32")
        _said(lib, f(P, P, P, 4, 64, 3, None), 1, b"dtype")
        _said(lib, f(P, None, P, 4, 64, 1, None), 1, b"null")
        _said(lib, f(P + 8, P, P, 4, 64, 1, None), 2, b"16-byte")
        _said(lib, f(P, P, P, 1 << 30, 1 << 20, 1, None), 1, b"too large")
        assert f(None, None, None, 0, 64, 1, None) == 0
    _said(lib, m(P, P, P, P, P, 4, 8, 48, 1, None), 1, b"multiple of 32")
    _said(lib, m(P, P, P, P, P, 4, 12, 64, 1, None), 1, b"multiple of 8")
    _said(lib, m(P, P, P, P, P, 4, 8, 0, 1, None), 1, b"positive")
    _said(lib, m(P, P, P, None, P, 4, 8, 64, 1, None), 1, b"null")
    _said(lib, m(P, P, P, P, P + 4, 4, 8, 64, 1, None), 2, b"16-byte")
    assert m(None, None, None, None, None, 0, 8, 64, 1, None) == 0


def test_mxfp4_swiglu_refusals_and_plan(lib):
    f, plan = lib.swiglu_b200_fused_matmul_swiglu_mxfp4, lib.swiglu_b200_fused_matmul_swiglu_mxfp4_plan
    _said(lib, f(P, P, P, P, P, P, 4, 64, 96, 0, None), 1, b"multiple of 128")
    _said(lib, f(P, P, P, P, P, P, 4, 40, 128, 0, None), 1, b"multiple of 32")
    _said(lib, f(P, P, P, P, P, P, 4, 64, 128, 2, None), 1, b"layout")
    _said(lib, f(P, P, P, P, None, None, 4, 64, 128, 0, None), 1, b"null")
    _said(lib, f(P, P, P, P, P, P + 2, 4, 64, 128, 0, None), 2, b"16-byte")
    assert f(None, None, None, None, None, None, 0, 64, 128, 0, None) == 0
    fused = ctypes.c_int(-1)
    for M, K, H, want in [(11136, 3584, 14336, 1), (1, 3584, 14336, 0), (64, 1024, 2816, 0), (4096, 1024, 2816, 1)]:
        assert plan(M, K, H, 148, ctypes.byref(fused)) == 0 and fused.value == want, (M, K, H)
    _said(lib, plan(4, 64, 128, 0, ctypes.byref(fused)), 1, b"num_sms")


def test_python_refusals_without_a_device():
    t = torch.ones(4, 64)
    for call in (lambda: ops.rmsnorm_fwd(t, t[0]), lambda: ops.quantize_mxfp4(t), lambda: ops.grad_norm([t]),
                 lambda: ops.clip_grad_norm_([t], 1.0)):
        with pytest.raises(ValueError):
            call()


def test_mx_restatement():
    """The format's own statements: a value on the grid is kept, an error is at
    most half the local spacing (a saturated value: up to the block's top)."""
    g = torch.Generator().manual_seed(0)
    t = torch.randn(64, 96, generator=g) * torch.logspace(-8, 8, 64)[:, None]
    code, byte = O.mx_quantize(t)
    v = O.mx_values(code, byte)
    unit = torch.pow(torch.tensor(2.0, dtype=torch.float64), byte.double() - 127).repeat_interleave(32, 1)
    a = t.double().abs() / unit
    assert a.max() < 8
    step = torch.where(a < 2, 0.25, torch.where(a < 4, 0.5, 1.0)).double()
    assert torch.all(((v - t.double()).abs() / unit)[a <= 6] <= step[a <= 6])
    again = O.mx_quantize(v.float())
    assert torch.equal(O.mx_values(*again), v)
    tiles = O.mx_tiles(byte)
    assert tuple(tiles.shape) == ops.mxfp4_scale_shape(64, 96)
    assert tiles[0, 0, 5, 1, 2] == byte[37, 2]
