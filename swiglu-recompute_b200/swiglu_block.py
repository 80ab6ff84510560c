"""Pre-norm SwiGLU block: residual RMS norm, then the recompute MLP.

    s = x + residual                       (the residual stream, returned)
    y = MLP(RMSNorm(s))                    (added to the stream by the next block)

A stack passes (y, s) from block to block. The MLP's operands are bf16, row-
scaled e4m3 or MXFP4 (`precision`); the backward is the bf16 (or f32) recompute
backward in every case. In the spirit of the MLP, which does not keep h, the
block does not keep the norm's output: it saves the stream s, one f32 value a
row and preact, and forms the norm's output again in its backward.

The reference has the MLP alone (swiglu_recompute.py:81-98).
"""

from __future__ import annotations

import torch
import torch.nn as nn

from swiglu_b200 import ops
from swiglu_b200.library import kernels
from swiglu_b200.ops import LAYOUT_STD, W1_ROWS
from swiglu_recompute import _first_derivative_only, _flatten_rows, _mxfp4_gemm1, _recompute_backward

PRECISIONS = ("bf16", "e4m3", "mxfp4")


class _MLPPart:
    """What _recompute_backward asks of a Function's context, for the MLP inside
    the block's."""

    def __init__(self, needs_input_grad, consumed):
        self.needs_input_grad = needs_input_grad
        self._preact_consumed = consumed


def _same_stream(x, residual):
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"residual {tuple(residual.shape)} {residual.dtype} does not match x "
                         f"{tuple(x.shape)} {x.dtype}")


class RMSNormResidualFunction(torch.autograd.Function):
    """(y, s) = residual RMS norm of x [..., D]; without a residual, y alone."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        ctx.set_materialize_grads(False)
        x2 = _flatten_rows(x)
        r2 = None if residual is None else _flatten_rows(residual)
        w = weight.contiguous()
        y, s, rstd = kernels().rmsnorm_fwd(x2, w, r2, eps)
        if any(ctx.needs_input_grad[:3]):
            ctx.save_for_backward(s, w, rstd)
        ctx.x_shape = x.shape
        y = y.reshape(x.shape)
        return y if residual is None else (y, s.reshape(x.shape))

    @staticmethod
    @_first_derivative_only
    def backward(ctx, dy, ds=None):
        s, w, rstd = ctx.saved_tensors
        if dy is None:
            return ds, None, ds, None
        d2 = None if ds is None else _flatten_rows(ds).to(s.dtype)
        dx, dw = kernels().rmsnorm_bwd(_flatten_rows(dy).to(s.dtype), s, w, rstd, d2)
        dx = dx.reshape(ctx.x_shape)
        need = ctx.needs_input_grad
        return dx if need[0] else None, dw if need[1] else None, dx if need[2] else None, None


class PreNormSwiGLUFunction(torch.autograd.Function):
    """(y, s) of the block; without a residual, y alone (s is x). With grad=False
    nothing is kept for a backward and preact is not written (a Function's forward
    cannot see torch.no_grad itself)."""

    @staticmethod
    def forward(ctx, x, residual, weight, W1, W2, eps, precision, grad=True):
        ctx.set_materialize_grads(False)
        # The quantisers take f32 as well, but the backward is that of a bf16 block.
        if precision != "bf16" and not x.dtype == W1.dtype == W2.dtype == torch.bfloat16:
            raise TypeError(f"{precision} operands go with a bf16 stream and bf16 parameters, got {x.dtype}, "
                            f"{W1.dtype}, {W2.dtype}")
        x2 = _flatten_rows(x)
        r2 = None if residual is None else _flatten_rows(residual)
        g, W1c, W2c = weight.contiguous(), W1.contiguous(), W2.contiguous()
        training = grad and any(ctx.needs_input_grad[:5])
        K = kernels()
        preact = None
        if precision == "e4m3":
            q, scale, s, rstd = K.rmsnorm_fwd_e4m3(x2, g, r2, eps)
            w1q, w1s = K.quantize_e4m3(W1c)
            if training:
                preact, h = K.swiglu_fwd_e4m3(q, scale, w1q, w1s, LAYOUT_STD)
            else:
                h = K.swiglu_fwd_e4m3_h(q, scale, w1q, w1s, LAYOUT_STD)
            del q, w1q
            y = K.matmul_e4m3(*K.quantize_e4m3(h), *K.quantize_e4m3(W2c))
        else:
            n, s, rstd = K.rmsnorm_fwd(x2, g, r2, eps)
            if precision == "mxfp4":
                nq, ns = K.quantize_mxfp4(n)
                del n
                preact, h = _mxfp4_gemm1(K, nq, ns, *K.quantize_mxfp4(W1c), training)
                y = K.matmul_mxfp4(*K.quantize_mxfp4(h), *K.quantize_mxfp4(W2c))
            else:
                if training:
                    preact, h = K.swiglu_fwd(n, W1c, W1_ROWS, LAYOUT_STD, True)
                else:
                    h = K.swiglu_fwd_h(n, W1c, W1_ROWS, LAYOUT_STD, True)
                del n
                y = K.matmul(h, W2c, False, True)
        del h
        if training:
            ctx.save_for_backward(s, g, rstd, W1c, W2c, preact)
        ctx.x_shape, ctx.eps = x.shape, eps
        y = y.reshape(*x.shape[:-1], W2.shape[0])
        return y if residual is None else (y, s.reshape(x.shape))

    @staticmethod
    @_first_derivative_only
    def backward(ctx, grad_y, ds=None):
        s, g, rstd, W1, W2, preact = ctx.saved_tensors
        need_x, need_r, need_g, need_w1, need_w2 = ctx.needs_input_grad[:5]
        if grad_y is None:  # only the stream was used
            return ds, ds, None, None, None, None, None, None
        K = kernels()
        # The norm's output again: the same kernel on the same rows.
        n = K.rmsnorm_fwd(s, g, None, ctx.eps)[0] if need_w1 else None
        need_n = need_x or need_r or need_g
        eager = not torch.compiler.is_compiling()
        mlp = _MLPPart((need_n, need_w1, need_w2), eager and getattr(ctx, "_preact_consumed", False))
        dn, dw1, dw2 = _recompute_backward(mlp, grad_y, n, W1, W2, preact, w_form=W1_ROWS, layout=LAYOUT_STD)
        if eager:
            ctx._preact_consumed = mlp._preact_consumed
        dx = dg = None
        if need_n:
            d2 = None if ds is None else _flatten_rows(ds).to(s.dtype)
            dx, dg = K.rmsnorm_bwd(dn, s, g, rstd, d2)
            dx = dx.reshape(ctx.x_shape)
        return (dx if need_x else None, dx if need_r else None, dg if need_g else None, dw1, dw2, None, None,
                None)


class RMSNormResidual(nn.Module):
    """RMS norm over the last dimension (weight, eps), with the residual's
    addition: forward(x) -> y, forward(x, residual) -> (y, s)."""

    def __init__(self, dim, eps=1e-6, dtype=torch.float32):
        super().__init__()
        self.eps = float(eps)
        self.weight = nn.Parameter(torch.ones(dim, dtype=dtype))

    def forward(self, x, residual=None):
        _same_stream(x, residual)
        return RMSNormResidualFunction.apply(x, self.weight, residual, self.eps)


class SwiGLUPreNormBlock(nn.Module):
    """forward(x, residual=None) -> (y, s): s = x + residual (x without one),
    y = MLP(RMSNorm(s)). precision: "bf16" (the parameters' own type: bf16 or
    f32 kernels), "e4m3" or "mxfp4" (bf16 parameters and a bf16 stream; MXFP4
    wants dim and hidden_dim to be multiples of 32)."""

    def __init__(self, dim, hidden_dim, out_dim=None, eps=1e-6, dtype=torch.bfloat16, precision="bf16"):
        super().__init__()
        if precision not in PRECISIONS:
            raise ValueError(f"precision must be one of {PRECISIONS}, got {precision!r}")
        if precision != "bf16" and dtype != torch.bfloat16:
            raise TypeError(f"{precision} operands go with bf16 parameters")
        self.dim, self.hidden_dim = dim, hidden_dim
        self.out_dim = out_dim if out_dim is not None else dim
        self.eps, self.precision = float(eps), precision
        self.norm_weight = nn.Parameter(torch.ones(dim, dtype=dtype))
        self.w1 = nn.Parameter(torch.empty(2 * hidden_dim, dim, dtype=dtype))
        self.w2 = nn.Parameter(torch.empty(self.out_dim, hidden_dim, dtype=dtype))
        nn.init.xavier_uniform_(self.w1)
        nn.init.xavier_uniform_(self.w2)

    def forward(self, x, residual=None):
        _same_stream(x, residual)
        out = PreNormSwiGLUFunction.apply(x, residual, self.norm_weight, self.w1, self.w2, self.eps, self.precision,
                                          torch.is_grad_enabled())
        return (out, x) if residual is None else out


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm):
    """Scales the gradients of `parameters` (an iterable of tensors, or one) in
    place by min(1, max_norm / (norm + 1e-6)) and returns their global 2-norm,
    on the device. It stands in for torch.nn.utils.clip_grad_norm_(parameters,
    max_norm); norm_type (always 2), error_if_nonfinite and foreach are not taken.
    Gradients are dense, bf16 or f32, on one device; a parameter may be listed once
    only. Parameters without a gradient are skipped, and without any the norm is
    zero."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [p.grad for p in parameters if p.grad is not None]
    if not grads:
        return torch.zeros(())
    return ops.clip_grad_norm_(grads, max_norm)
