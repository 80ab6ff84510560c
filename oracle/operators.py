"""64-bit restatements of the operators around the block. TEST INFRASTRUCTURE
ONLY (see swiglu_oracle.py): the residual RMS norm and its gradient, the MXFP4
format and its product, the global gradient norm."""
from __future__ import annotations

import torch

E4M3_MAX = 448.0
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ------------------------------------------------------------------ RMS norm
def stream(x, residual):
    """The residual stream as it is stored: one f32 addition, one rounding."""
    return x if residual is None else (x.float() + residual.float()).to(x.dtype)


def rmsnorm(x, weight, residual=None, eps=1e-6):
    """(y, s, rstd) in f64 from the stored stream."""
    s = stream(x, residual).double()
    rstd = (s.square().mean(1) + eps).rsqrt()
    return s * rstd[:, None] * weight.double(), s, rstd


def rmsnorm_grad(dy, s, weight, rstd, ds=None):
    """(dx, dweight) in f64, with the rstd that is given."""
    dy, s, w, r = dy.double(), s.double(), weight.double(), rstd.double()[:, None]
    g = dy * w
    dx = r * g - s * r ** 3 * (g * s).mean(1, keepdim=True)
    if ds is not None:
        dx = dx + ds.double()
    return dx, (dy * s * r).sum(0)


# --------------------------------------------------------------------- MXFP4
def mx_quantize(t):
    """(codes [R, K], scale bytes [R, K/32]) element by element from the
    definition, in f64."""
    R, K = t.shape
    v = t.double().view(R, K // 32, 32)
    top = v.abs().amax(-1)
    bad = ~torch.isfinite(v).all(-1)
    exponent = torch.frexp(torch.where(bad, torch.ones_like(top), top))[1].long() - 1
    byte = (exponent - 2 + 127).clamp(min=0)
    byte[top == 0] = 0
    a = v.abs() * torch.pow(torch.tensor(2.0, dtype=torch.float64), (127 - byte).double())[..., None]
    grid = torch.tensor(E2M1, dtype=torch.float64)
    # nearest of the eight values, ties to the even code
    dist = (a.clamp(max=6.0)[..., None] - grid).abs()
    best = dist.min(-1, keepdim=True).values
    tied = dist == best
    even = torch.arange(8) % 2 == 0
    code = torch.where((tied & even).any(-1), (tied & even).to(torch.uint8).argmax(-1), tied.to(torch.uint8).argmax(-1))
    code = code + 8 * torch.signbit(t).view(R, K // 32, 32).long()
    byte[bad] = 255
    return code.view(R, K).to(torch.uint8), byte.to(torch.uint8)


def mx_pack(code):
    return code[:, 0::2] | (code[:, 1::2] << 4)


def mx_tiles(byte):
    """[R, B] scale bytes -> tiles [ceil(R/128), ceil(B/4), 32, 4, 4], one
    element at a time."""
    R, B = byte.shape
    out = torch.zeros((-(-R // 128), -(-B // 4), 32, 4, 4), dtype=torch.uint8)
    r, b = torch.meshgrid(torch.arange(R), torch.arange(B), indexing="ij")
    out[r // 128, b // 4, r % 32, (r % 128) // 32, b % 4] = byte
    return out


def mx_values(code, byte):
    """f64 values of codes and scale bytes (255: NaN)."""
    R, K = code.shape
    grid = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float64)
    scale = torch.pow(torch.tensor(2.0, dtype=torch.float64), byte.double() - 127)
    scale[byte == 255] = float("nan")
    return (grid[code.long()].view(R, K // 32, 32) * scale[..., None]).view(R, K)


# -------------------------------------------------------------- gradient norm
def clip(tensors, max_norm):
    """(norm, [clipped in f64])."""
    norm = sum(t.double().square().sum() for t in tensors).sqrt()
    factor = (max_norm / (norm + 1e-6)).clamp(max=1.0)
    return norm, [t.double() * factor for t in tensors]
