"""The pre-norm block, the MXFP4 modules and clipping used together.

A block's forward is a chain of this library's operators, each held to its own
64-bit form by its own tests, and must give the chain's bits. (A restatement
of the whole chain in f64 would not do with 4- and 8-bit operands: where f32 and
f64 fall on different sides of a rounding border of an operand, e4m3 moves it by
1/8 of its value and e2m1 by 1/3, and with it a whole row of the result.) The
gradients are held to the f64 formulas from the chain's preact and stream, with
the backward's own rounding points (grad_h, grad_preact and the norm's gradient
are bf16): 1e-2 of the largest value, as the framework's other module tests, for
one rounding of the result (2^-8) and intermediates whose bf16 rounding falls the
other way, which average out over the contractions. f32 results: 1e-5.
"""
import pytest
import torch

import swiglu_block as SB
import swiglu_recompute as SR
from oracle import operators as OP
from oracle import swiglu_oracle as O
from swiglu_b200 import ops

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF = torch.bfloat16


def _bf(t):
    return t.to(BF).double()


def _mx_gemm1(x, w1):
    if w1.shape[0] % 256 == 0:
        return ops.swiglu_fwd_mxfp4(*ops.quantize_mxfp4(x), *ops.quantize_mxfp4(w1), layout=ops.LAYOUT_STD)
    pre = ops.matmul_mxfp4(*ops.quantize_mxfp4(x), *ops.quantize_mxfp4(w1))
    return pre, ops.forward_logic(pre, layout=ops.LAYOUT_STD)


def _chain(x, r, g, w1, w2, precision, eps=1e-6):
    """(y, s, preact) by the operators one after another, on the device."""
    if precision == "e4m3":
        q, scale, s, _ = ops.rmsnorm_fwd_e4m3(x, g, r, eps=eps)
        pre, h = ops.swiglu_fwd_e4m3(q, scale, *ops.quantize_rows_e4m3(w1), layout=ops.LAYOUT_STD, h_from_rounded=True)
        return ops.matmul_e4m3(*ops.quantize_rows_e4m3(h), *ops.quantize_rows_e4m3(w2)), s, pre
    n, s, _ = ops.rmsnorm_fwd(x, g, r, eps=eps)
    if precision == "mxfp4":
        pre, h = _mx_gemm1(n, w1)
        return ops.matmul_mxfp4(*ops.quantize_mxfp4(h), *ops.quantize_mxfp4(w2)), s, pre
    pre, h = ops.swiglu_fwd(n, w1, w_form=ops.W1_ROWS, layout=ops.LAYOUT_STD, h_from_rounded=True)
    return ops.matmul(h, w2, a_t=False, b_t=True), s, pre


def _grads(s, pre, g, w1, w2, gy, gs, eps=1e-6):
    """(dx, dg, dw1, dw2) in f64 from the stream and preact, with the backward's
    bf16 roundings."""
    s, pre, g, w1, w2 = (t.detach().cpu() for t in (s, pre, g, w1, w2))
    n, _, rstd = OP.rmsnorm(s, g, None, eps)
    n = _bf(n)
    left, gate = pre.double().chunk(2, 1)
    sg = torch.sigmoid(gate)
    h = _bf(left * gate * sg)
    gy = gy.detach().double().cpu()
    gh = _bf(gy @ w2.double())
    gp = _bf(torch.cat([gh * gate * sg, gh * left * (sg + gate * sg * (1 - sg))], 1))
    dn = _bf(gp @ w1.double())
    dx, dg = OP.rmsnorm_grad(dn, s, g, rstd, gs)
    return dx, dg, gp.t() @ n, gy.t() @ h


def _make(M, D, H, Dout, seed=0, dtype=BF, precision="bf16"):
    x, w1, w2, gy = O.make_inputs(M, D, H, Dout, seed=seed, dtype=dtype)
    g = torch.Generator().manual_seed(seed + 100)
    r = (torch.randn(M, D, generator=g) * 1.5).to(dtype)
    gs = (torch.randn(M, D, generator=g) * 0.1).to(dtype)
    m = SB.SwiGLUPreNormBlock(D, H, Dout, dtype=dtype, precision=precision).to(DEV)
    with torch.no_grad():
        m.norm_weight.copy_((1 + 0.2 * torch.randn(D, generator=g)).to(dtype))
        m.w1.copy_(w1)
        m.w2.copy_(w2)
    return m, x, r, gy, gs


def _close(got, want, tol=1e-2):
    assert O.rel_max(got.detach().double().cpu(), want) <= tol, O.rel_max(got.detach().double().cpu(), want)


@pytest.mark.parametrize("precision", SB.PRECISIONS)
@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("M,D,H,Dout", [(256, 256, 384, 256), (300, 512, 1024, 136), (1, 256, 256, 256)])
def test_block_forward_backward(precision, residual, M, D, H, Dout):
    m, x, r, gy, gs = _make(M, D, H, Dout, precision=precision)
    xd = x.to(DEV).requires_grad_(True)
    rd = r.to(DEV).requires_grad_(True) if residual else None
    y, s = m(xd, rd)
    with torch.no_grad():
        ry, rs, pre = _chain(x.to(DEV), r.to(DEV) if residual else None, m.norm_weight, m.w1, m.w2, precision)
    assert torch.equal(y, ry) and torch.equal(s, rs)
    leaves = [xd] + ([rd] if residual else []) + [m.norm_weight, m.w1, m.w2]
    got = torch.autograd.grad([y, s], leaves, [gy.to(DEV), gs.to(DEV)])
    ref = _grads(rs, pre, m.norm_weight, m.w1, m.w2, gy, gs)
    for dx in got[:-3]:
        _close(dx, ref[0])
    for k, want in zip(got[-3:], ref[1:]):
        _close(k, want)
    assert ops.device_status(0) == 0


def test_block_f32():
    m, x, r, gy, gs = _make(96, 64, 96, 48, dtype=torch.float32)
    xd, rd = x.to(DEV).requires_grad_(True), r.to(DEV).requires_grad_(True)
    y, s = m(xd, rd)
    got = torch.autograd.grad([y, s], [xd, rd, m.norm_weight, m.w1, m.w2], [gy.to(DEV), gs.to(DEV)])
    leaves = [t.detach().double().cpu().requires_grad_(True) for t in (x, r, m.norm_weight, m.w1, m.w2)]
    a, b, g, w1, w2 = leaves
    st = a + b
    pre = (st * (st.square().mean(1, keepdim=True) + 1e-6).rsqrt() * g) @ w1.t()
    left, gate = pre.chunk(2, 1)
    yr = (left * torch.nn.functional.silu(gate)) @ w2.t()
    want = torch.autograd.grad([yr, st], leaves, [gy.double(), gs.double()])
    _close(y, yr.detach(), 1e-5)
    for u, v in zip(got, want):
        _close(u, v, 1e-5)


def test_leading_dimensions_partial_gradients_and_second_backward():
    m, x, r, gy, gs = _make(60, 64, 128, 64)
    x3, r3 = x.view(3, 4, 5, 64).to(DEV), r.view(3, 4, 5, 64).to(DEV)
    flat, fs = m(x.to(DEV), r.to(DEV))
    xd = x3.clone().requires_grad_(True)
    y, s = m(xd, r3)
    assert y.shape == (3, 4, 5, 64) and torch.equal(y.view(60, 64), flat) and torch.equal(s.view(60, 64), fs)
    (dx,) = torch.autograd.grad(y, [xd], gy.view(3, 4, 5, 64).to(DEV), retain_graph=True)
    assert dx.shape == x3.shape
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, [xd], gy.view(3, 4, 5, 64).to(DEV))
    # only the stream's gradient: it passes through
    y, s = m(xd, r3)
    (ds,) = torch.autograd.grad(s, [xd], gs.view(3, 4, 5, 64).to(DEV))
    assert torch.equal(ds.view(60, 64).cpu(), gs)
    # no second derivative, and it says so
    y, s = m(xd, r3)
    (dx,) = torch.autograd.grad(y, [xd], gy.view(3, 4, 5, 64).to(DEV), create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()
    # weights alone
    y, s = m(x3, r3)
    dg, dw1 = torch.autograd.grad(y, [m.norm_weight, m.w1], gy.view(3, 4, 5, 64).to(DEV))
    assert dg.shape == (64,) and torch.isfinite(dw1).all()
    with torch.no_grad():
        assert torch.equal(m(x3, r3)[0], y.detach())


@pytest.mark.parametrize("precision", SB.PRECISIONS)
def test_no_rows(precision):
    m, x, r, gy, gs = _make(4, 64, 128, 64, precision=precision)
    with torch.no_grad():
        y, s = m(x[:0].to(DEV), r[:0].to(DEV))
    assert y.shape == (0, 64) and s.shape == (0, 64)


def test_norm_module():
    n = SB.RMSNormResidual(96, eps=1e-5, dtype=torch.float32).to(DEV)
    g = torch.Generator().manual_seed(3)
    x, r, dy, ds = ((torch.randn(2, 9, 96, generator=g)).to(BF) for _ in range(4))
    xd, rd = x.to(DEV).requires_grad_(True), r.to(DEV).requires_grad_(True)
    y, s = n(xd, rd)
    got = torch.autograd.grad([y, s], [xd, rd, n.weight], [dy.to(DEV), ds.to(DEV)])
    ry, rs, rstd = OP.rmsnorm(x.view(18, 96), n.weight.detach().cpu(), r.view(18, 96), 1e-5)
    rx, rw = OP.rmsnorm_grad(dy.view(18, 96), rs, n.weight.detach().cpu(), rstd, ds.view(18, 96))
    _close(y.view(18, 96), ry, 2 ** -8)
    _close(got[0].view(18, 96), rx, 2 ** -8)
    assert torch.equal(got[0], got[1])
    _close(got[2], rw, 1e-5)
    z = n(xd)
    z.sum().backward()  # an expanded gradient
    assert xd.grad.shape == x.shape and torch.isfinite(xd.grad).all()
    with pytest.raises(ValueError):
        n(xd, rd[:1])
    with pytest.raises(ValueError):
        n(xd, rd.float())


@pytest.mark.parametrize("M,D,H,Dout", [(1, 256, 512, 256), (5, 512, 256, 128), (384, 256, 384, 264),
                                        (200, 96, 160, 64)])
def test_fp4_modules(M, D, H, Dout):
    x, w1, w2, gy = O.make_inputs(M, D, H, Dout, seed=6, dtype=BF)
    m = SR.SwiGLUMLPFP4Forward(D, H, Dout, dtype=BF).to(DEV)
    with torch.no_grad():
        m.w1.copy_(w1)
        m.w2.copy_(w2)
    xd = x.to(DEV).requires_grad_(True)
    y = m(xd)
    with torch.no_grad():
        pre, h = _mx_gemm1(x.to(DEV), m.w1)
        assert torch.equal(y, ops.matmul_mxfp4(*ops.quantize_mxfp4(h), *ops.quantize_mxfp4(m.w2)))
    gx, gw1, gw2 = torch.autograd.grad(y, [xd, m.w1, m.w2], gy.to(DEV))
    left, gate = pre.double().cpu().chunk(2, 1)
    sg = torch.sigmoid(gate)
    gh = _bf(gy.double() @ w2.double())
    gp = _bf(torch.cat([gh * gate * sg, gh * left * (sg + gate * sg * (1 - sg))], 1))
    for got, want in ((gx, gp @ w1.double()), (gw1, gp.t() @ x.double()),
                      (gw2, gy.double().t() @ _bf(left * gate * sg))):
        _close(got, want)
    served = SR.SwiGLUMLPFP4Inference.from_mlp(m)
    z = served(x.to(DEV))
    assert torch.equal(z, y.detach()) and not z.requires_grad
    assert sum(b.numel() for b in served.buffers()) < 0.6 * (w1.numel() + w2.numel()) + 4 * 512 * 8
    state = served.state_dict()
    assert set(state) == {"w1_q", "w1_scale", "w2_q", "w2_scale"}
    with pytest.raises(TypeError):
        m(x.to(DEV).float())


@pytest.mark.parametrize("precision", SB.PRECISIONS)
def test_a_training_step_of_two_blocks(precision):
    """norm -> MLP -> norm -> MLP -> loss, backward, clip: the gradients before
    clipping against the formulas, the clipped ones against clipping those, and
    a second step from the same state gives the same bits."""
    M, D, H = 192, 128, 256
    blocks, x, r, gy, gs = [], None, None, None, None
    for k in range(2):
        m, xk, rk, gyk, gsk = _make(M, D, H, D, seed=20 + k, precision=precision)
        blocks.append(m)
        x, gy, gs = (xk, gyk, gsk) if k == 0 else (x, gyk, gsk)
    params = [p for m in blocks for p in m.parameters()]

    def step():
        for p in params:
            p.grad = None
        y, s = blocks[0](x.to(DEV))
        y, s = blocks[1](y, s)
        torch.autograd.backward([y, s], [gy.to(DEV), gs.to(DEV)])
        before = [p.grad.clone() for p in params]
        norm = SB.clip_grad_norm_(params, 0.5)
        return before, norm, [p.grad.clone() for p in params]

    before, norm, after = step()
    # Block 1's gradients from the chain, then its dx into block 0 as the gradient of
    # both its y and its stream. Block 0's see one more bf16 gradient: 2e-2.
    with torch.no_grad():
        y0, s0, pre0 = _chain(x.to(DEV), None, *blocks[0].parameters(), precision)
        y1, s1, pre1 = _chain(y0, s0, *blocks[1].parameters(), precision)
    r1 = _grads(s1, pre1, *blocks[1].parameters(), gy, gs)
    r0 = _grads(s0, pre0, *blocks[0].parameters(), r1[0].to(BF), r1[0].to(BF))
    for got, want, tol in zip(before, r0[1:] + r1[1:], [2e-2] * 3 + [1e-2] * 3):
        _close(got, want, tol)
    rn, clipped = OP.clip([t.cpu() for t in before], 0.5)
    assert abs(norm.cpu().double() - rn) <= 34 * 2.0 ** -24 * rn
    for got, want in zip(after, clipped):
        assert torch.all((got.cpu().double() - want).abs() <= (2 ** -8 + 2.0 ** -18) * want.abs())
    again = step()
    assert torch.equal(again[1], norm) and all(torch.equal(a, b) for a, b in zip(again[0], before))
    assert ops.device_status(0) == 0


@pytest.mark.parametrize("precision", SB.PRECISIONS)
def test_a_step_captured_in_a_graph(precision):
    """Forward, gradients and clipping of a block in one CUDA graph, replayed on
    other inputs: the eager call's bits (at this size no GEMM splits its tail)."""
    m, x, r, gy, gs = _make(160, 128, 256, 128, precision=precision)
    params = list(m.parameters())
    xs, rs, gys = x.to(DEV), r.to(DEV), gy.to(DEV)

    def step(a, b, g):
        a, b = a.detach().requires_grad_(True), b.detach().requires_grad_(True)
        y, s = m(a, b)
        grads = torch.autograd.grad([y, s], [a, b] + params, [g, g])
        return (y, s, ops.clip_grad_norm_(grads[2:], 0.1), *grads)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(xs, rs, gys)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(xs, rs, gys)
    for seed in (1, 2):
        g = torch.Generator().manual_seed(seed)
        new = [torch.randn(t.shape, generator=g).to(BF).to(DEV) for t in (xs, rs, gys)]
        want = [t.detach().clone() for t in step(*new)]
        for a, b in zip((xs, rs, gys), new):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert ops.device_status(0) == 0


def test_clip_like_torch():
    m, x, r, gy, gs = _make(64, 64, 64, 64)
    y, s = m(x.to(DEV), r.to(DEV))
    y.backward(gy.to(DEV))
    want = [p.grad.clone() for p in m.parameters()]
    for p, g in zip(m.parameters(), want):
        p.grad = g.clone()
    norm = SB.clip_grad_norm_(m.parameters(), 1.0)
    twin = [torch.nn.Parameter(torch.zeros_like(g)) for g in want]
    for t, g in zip(twin, want):
        t.grad = g
    ref = torch.nn.utils.clip_grad_norm_(twin, 1.0)
    assert abs(norm.item() - ref.item()) <= 1e-2 * ref.item()      # torch sums bf16 norms
    for p, t in zip(m.parameters(), twin):
        assert torch.allclose(p.grad.float(), t.grad.float(), rtol=2e-2, atol=1e-6)
    assert SB.clip_grad_norm_([torch.nn.Parameter(torch.ones(3, device=DEV))], 1.0) == 0
    p = torch.nn.Parameter(torch.ones(4, device=DEV))
    p.grad = torch.full((4,), 3.0, device=DEV)
    assert SB.clip_grad_norm_(p, 3.0).item() == 6.0
    assert torch.allclose(p.grad, torch.full((4,), 1.5, device=DEV))


@pytest.mark.parametrize("precision", SB.PRECISIONS)
def test_block_compiles(precision):
    m, x, r, gy, gs = _make(128, 128, 256, 128, precision=precision)
    eager = m(x.to(DEV), r.to(DEV))
    ge = torch.autograd.grad(eager[0], list(m.parameters()), gy.to(DEV))
    c = torch.compile(m, fullgraph=True)
    y, s = c(x.to(DEV), r.to(DEV))
    gc = torch.autograd.grad(y, list(m.parameters()), gy.to(DEV))
    assert torch.equal(y, eager[0]) and torch.equal(s, eager[1])
    for a, b in zip(ge, gc):
        assert torch.equal(a, b)
