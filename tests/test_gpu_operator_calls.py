"""Calls of the operators around the block that their documentation allows and
that are easily got wrong: the ends of the range, rows and gradients of zeros,
captured joins, ragged ends."""
import pytest
import torch

from oracle import operators as O
from swiglu_b200 import ops

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = 2.0 ** -24
BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("D", [96, 1001, 3584, 65544])   # warp rows, shifted packs, packs, the looping kernel
@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("residual", [True, False])
def test_e4m3_rows_of_tiny_values(D, dt, residual):
    """Rows down to the smallest subnormals reach 448 and read back as y.

    Bounds: half a step of e4m3 (2^-4 of the value, 2^-10 of the scale below the
    normals), the f32 steps of the norm's own tests, and two roundings that are
    absolute among the subnormals, half of 2^-149 each: that of s w, which the
    factor rstd follows, and that of the scale, which a code of up to 448 does."""
    g = torch.Generator().manual_seed(D)
    size = torch.tensor([1e-30, 1e-35, 1.5e-36, 1e-36, 1e-37, 1e-38, 1e-39, 1e-40, 1e-42, 1e-43])[:, None]
    x = (torch.randn(10, D, generator=g) * size).to(dt)
    r = (torch.randn(10, D, generator=g) * size).to(dt) if residual else None
    w = 1 + 0.3 * torch.randn(D, generator=g)
    q, scale, s, _ = ops.rmsnorm_fwd_e4m3(x.to(DEV), w.to(DEV), None if r is None else r.to(DEV))
    y, st, rstd = O.rmsnorm(x, w, r)
    assert torch.equal(s.cpu().double(), st)
    top = y.abs().amax(1)
    code, got = q.cpu().float().double(), scale.cpu().double()
    assert torch.all(code.abs().amax(1)[top > 0] == O.E4M3_MAX)
    assert torch.all(got[top == 0] == 1)
    steps = (D / 32 + 48) * U
    of_product, of_scale = 2.0 ** -150 * rstd[:, None], 448 * 2.0 ** -150
    size = y.abs() + of_product
    bound = (torch.maximum(size * 2 ** -4, got[:, None] * 2 ** -10) * (1 + 2 * steps) + 2 * steps * size
             + of_product + of_scale)
    live = top > 0
    assert torch.all(((code * got[:, None] - y).abs() <= bound)[live])
