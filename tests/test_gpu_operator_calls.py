"""Calls of the operators around the block that their documentation allows and
that are easily got wrong: the ends of the range, rows and gradients of zeros,
captured joins, ragged ends."""
import ctypes

import pytest
import torch

import swiglu_block as SB
import swiglu_recompute as SR
from oracle import operators as O
from swiglu_b200 import _lib, ops

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


# Rows of odd widths through the shared-memory ring (at least three rows a block),
# with every number of elements that a matrix can leave in its last pack.
RAGGED = ([(3000 + k, 2051, F32) for k in (1, 2, 3)] + [(445, 4095, F32), (446, 4095, F32)]
          + [(3000 + k, 1029, BF) for k in range(1, 8)] + [(445, 8191, BF), (450, 8190, BF)])


@pytest.mark.parametrize("M,D,dt", RAGGED)
@pytest.mark.parametrize("with_ds", [True, False])
def test_norm_gradient_of_a_matrix_that_ends_inside_a_pack(M, D, dt, with_ds):
    """dx and dweight to the bounds of the norm's own tests, and nothing written
    behind or before dx."""
    assert M * D % (128 // torch.finfo(dt).bits) != 0
    g = torch.Generator().manual_seed(M + D)
    s, dy = torch.randn(M, D, generator=g).to(dt), torch.randn(M, D, generator=g).to(dt)
    ds = (torch.randn(M, D, generator=g) * 0.25).to(dt) if with_ds else None
    w = (1 + 0.3 * torch.randn(D, generator=g)).to(dt)
    rstd = O.rmsnorm(s, w)[2].float()
    es, guard = s.element_size(), 256
    raw = torch.full((M * D * es + 2 * guard,), 0xA5, dtype=torch.uint8, device=DEV)
    dx = raw[guard:guard + M * D * es].view(dt).view(M, D)
    dw = torch.empty(D, device=DEV, dtype=dt)
    n = ctypes.c_int64(0)
    _lib.call("swiglu_b200_rmsnorm_bwd_workspace", M, D, ops._num_sms(0), ctypes.byref(n))
    ws = torch.empty(n.value, device=DEV)
    code = _lib.F32 if dt == F32 else _lib.BF16
    a = [None if t is None else t.to(DEV) for t in (dy, s, w, rstd, ds)]
    _lib.call("swiglu_b200_rmsnorm_bwd", *(None if t is None else t.data_ptr() for t in a), dx.data_ptr(), dw.data_ptr(),
              ws.data_ptr(), n.value, M, D, code, code, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert bool((raw[:guard] == 0xA5).all()) and bool((raw[guard + M * D * es:] == 0xA5).all())
    rx, rw = O.rmsnorm_grad(dy, s, w, rstd, ds)
    half, r = torch.finfo(dt).eps / 2, rstd.double()[:, None]
    gw, S = (dy.double() * w.double()).abs(), s.double().abs()
    along = S * r ** 3 * (gw * S).mean(1, keepdim=True)
    size = r * gw + along + (0 if ds is None else ds.double().abs())
    assert torch.all((dx.cpu().double() - rx).abs() <= half * rx.abs() + (D / 32 + 48) * U * along + 8 * U * size)
    mass = (dy.double().abs() * S * r).sum(0)
    assert torch.all((dw.cpu().double() - rw).abs() <= half * rw.abs() + (M + 48) * U * mass)
    assert ops.device_status(0) == 0


def test_captured_behind_a_join_of_two_streams():
    """Kernels that are placed early (programmatic dependent launch) behind a fork and
    a join in a captured graph: the eager call's bits, replayed on other inputs."""
    g = torch.Generator().manual_seed(4)
    new = lambda: [torch.randn(700, 512, generator=g).to(BF).to(DEV) for _ in range(2)]  # noqa: E731
    x, r = new()
    w = torch.ones(512, device=DEV, dtype=BF)
    side = torch.cuda.Stream()

    def step():
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        q, scale = ops.quantize_mxfp4(x)
        with torch.cuda.stream(side):
            y, s, rstd = ops.rmsnorm_fwd(r, w, x)
        main.wait_stream(side)
        dx, dw = ops.rmsnorm_bwd(y, s, w, rstd, x)       # directly behind the join
        back = ops.dequantize_mxfp4(q, scale)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            c = ops.matmul_mxfp4(q, scale, q[:64], scale[:1])
        norm = ops.clip_grad_norm_([dx, dw, back], 1.0)
        main.wait_stream(side)
        return y, s, dx, dw, back, c, norm

    for _ in range(2):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        for a, b in zip((x, r), new()):
            a.copy_(b)
        want = [t.clone() for t in step()]
        for t in out:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert ops.device_status(0) == 0


@pytest.mark.parametrize("which", ["fp4", "served", "norm", *SB.PRECISIONS])
def test_modules_compile_with_and_without_gradients(which):
    """torch.compile gives the eager bits, in training and under torch.no_grad."""
    torch.manual_seed(3)
    x, r = (torch.randn(96, 128, device=DEV).to(BF) for _ in range(2))
    if which in ("fp4", "served"):
        m = SR.SwiGLUMLPFP4Forward(128, 256, dtype=BF).to(DEV)
        m = SR.SwiGLUMLPFP4Inference.from_mlp(m) if which == "served" else m
        args = (x,)
    else:
        m = SB.RMSNormResidual(128).to(DEV) if which == "norm" else SB.SwiGLUPreNormBlock(128, 256, precision=which).to(DEV)
        args = (x, r)
    torch._dynamo.reset()
    c = torch.compile(m, fullgraph=True)
    outs = lambda f: [f(*args)] if len(args) == 1 else list(f(*args))  # noqa: E731
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(outs(c), outs(m)))
    params = list(m.parameters())
    if params:
        a, b = outs(m), outs(c)
        assert all(torch.equal(u, v) for u, v in zip(a, b))
        ga, gb = (torch.autograd.grad(o[0].float().square().sum(), params) for o in (a, b))
        assert all(torch.equal(u, v) for u, v in zip(ga, gb))
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(outs(c), outs(m)))


@pytest.mark.parametrize("M,D", [(5, 96), (700, 1001), (300, 3584), (3, 40000)])
@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("e4m3", [True, False])
def test_stream_written_over_either_of_its_terms(M, D, dt, e4m3):
    """The C entry points take s = x or s = residual: the same bits."""
    g = torch.Generator().manual_seed(D)
    x, r = (torch.randn(M, D, generator=g).to(dt).to(DEV) for _ in range(2))
    w = torch.ones(D, device=DEV, dtype=dt)
    code = _lib.F32 if dt == F32 else _lib.BF16
    eps = ctypes.byref(ctypes.c_float(1e-6))
    st = torch.cuda.current_stream().cuda_stream

    def run(over):
        a, b = x.clone(), r.clone()
        s = {"none": torch.empty_like(x), "x": a, "residual": b}[over]
        y = torch.empty(M, D, device=DEV, dtype=torch.uint8 if e4m3 else dt)
        scale, rstd = torch.zeros(M, device=DEV), torch.empty(M, device=DEV)
        p = [t.data_ptr() for t in (a, b, w, y)] + ([scale.data_ptr()] if e4m3 else []) + [s.data_ptr(), rstd.data_ptr()]
        _lib.call("swiglu_b200_rmsnorm_fwd_e4m3" if e4m3 else "swiglu_b200_rmsnorm_fwd", *p, M, D, eps, code, code, st)
        torch.cuda.synchronize()
        return y, s, rstd, scale

    want = run("none")
    for over in ("x", "residual"):
        assert all(torch.equal(a, b) for a, b in zip(run(over), want)), over


@pytest.mark.parametrize("M,D", [(3, 128), (640, 1024), (6000, 2048)])
def test_a_chain_without_a_pause_gives_the_bits_of_one_with_pauses(M, D):
    """Each kernel is placed while the previous one drains: a chain in which each
    reads, or writes over, what the one before it wrote or read."""
    g = torch.Generator().manual_seed(M)
    x0, r0 = (torch.randn(M, D, generator=g).to(BF).to(DEV) for _ in range(2))
    w = torch.ones(D, device=DEV, dtype=BF)
    weight = ops.quantize_mxfp4((torch.randn(D, D, generator=g) * D ** -0.5).to(BF).to(DEV))

    def chain(pause):
        x, r, norms = x0.clone(), r0.clone(), []
        wait = torch.cuda.synchronize if pause else lambda: None
        for _ in range(12):
            y, s, rstd = ops.rmsnorm_fwd(x, w, r)
            wait()
            q = ops.quantize_mxfp4(y)
            wait()
            c = ops.matmul_mxfp4(*q, *weight)
            wait()
            dx, dw = ops.rmsnorm_bwd(c, s, w, rstd, x)
            wait()
            norms.append(ops.clip_grad_norm_([dx, dw], 30.0))      # in place
            wait()
            norms.append(ops.clip_grad_norm_([dx, s], 40.0, out=[r, x]))  # over what the norm reads next
            wait()
        return x, r, *norms

    want = chain(True)
    for _ in range(8):
        assert all(torch.equal(a, b) for a, b in zip(chain(False), want))
    assert ops.device_status(0) == 0
