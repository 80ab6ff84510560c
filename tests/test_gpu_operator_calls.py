"""Calls of the operators around the block that their documentation allows and
that are easily got wrong: the ends of the range, rows and gradients of zeros,
captured joins, ragged ends."""
import pytest
import torch

import swiglu_block as SB
import swiglu_recompute as SR
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


@pytest.mark.parametrize("dt", [BF, F32])
def test_zeros_and_values_that_f32_squares_lose_side_by_side(dt):
    """Zeros of either sign are told from values whose squares underflow f32 by
    their bits, thread by thread: a lone tiny value among zeros counts, in every
    slot of a chunk and behind its ragged end. Bounds: one square, two at most, is
    exact to 2^-53 in f64; the norm rounds once to f32 (2^-24)."""
    n = 256 * 8 * 8 + 37
    base = torch.zeros(n, dtype=dt)
    base[::3] = -0.0
    assert ops.grad_norm([base.to(DEV)]) == 0
    for at in (0, 1, 255, 2047, 2048 * 3 + 5, 256 * 8 * 4 - 1, 256 * 8 * 8 - 1, n - 1):
        for v in (1e-30, -3e-39, 1e-16, 2e19, -1.5):
            t = base.clone()
            t[at] = v
            got = ops.grad_norm([torch.zeros(5, device=DEV), t.to(DEV)])
            want = t[at].double().abs()
            assert abs(got.cpu().double() - want) <= max(2 * U * want, 2.0 ** -149), (at, v)
    for name, z in (("zeros", torch.zeros(100000, dtype=dt)), ("empty end", torch.zeros(3, dtype=dt))):
        d = [z.to(DEV), torch.ones(4, device=DEV)]
        assert ops.clip_grad_norm_(d, 1.0) == 2 and not d[0].any(), name


@pytest.mark.parametrize("which", ["mlp", "fp8", "fp4", "norm", *SB.PRECISIONS])
@pytest.mark.parametrize("mode", ops.DW2_MODES)
def test_training_without_rows(which, mode):
    """An expert without tokens, an empty last batch: empty outputs, gradients of
    zeros (the weights' gradient used to be refused for its empty sum)."""
    made = {"mlp": SR.SwiGLUMLPCustom, "fp8": SR.SwiGLUMLPFP8Forward, "fp4": SR.SwiGLUMLPFP4Forward}
    if which in made:
        m = made[which](64, 128, 96, dtype=BF)
    else:
        m = SB.RMSNormResidual(64) if which == "norm" else SB.SwiGLUPreNormBlock(64, 128, 96, precision=which)
    m.to(DEV)
    x = torch.empty(0, 5, 64, device=DEV, dtype=BF, requires_grad=True)
    ops.set_dw2_mode(mode)
    try:
        if which in made:
            outs = [m(x)]
        else:
            r = torch.empty_like(x, requires_grad=True)
            outs = list(m(x, r))
        assert outs[0].shape == (0, 5, 64 if which == "norm" else 96)
        torch.autograd.backward(outs, [torch.ones_like(o) for o in outs])
    finally:
        ops.set_dw2_mode("prologue")
    assert x.grad.shape == x.shape
    for p in m.parameters():
        assert p.grad.shape == p.shape and p.grad.dtype == p.dtype and not p.grad.any()
