"""Residual RMS norm (forward, e4m3 output, gradient) against its 64-bit form.

Tolerances. A rounding to type t is off by at most eps(t)/2 of the value. f32
sums over a row run at most cols/32 additions in sequence in one thread (a
warp is the smallest group that shares a row), then a tree: (cols/32 + 40)
steps of 2^-24 of the sum of magnitudes bound them; over the rows of dweight,
rows + 40 steps. A product chain adds less than 8 such steps.
"""
import pytest
import torch

from oracle import operators as O
from swiglu_b200 import ops

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = 2.0 ** -24
BF, F32 = torch.bfloat16, torch.float32

SHAPES = [(1, 1), (1, 8), (3, 7), (5, 64), (1, 3584), (257, 1000), (333, 1001), (64, 1024), (19, 2816), (130, 3584),
          (40, 4099), (33, 8192), (9, 16384), (3, 20001), (2, 65544), (700, 96)]


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _inputs(M, D, dt, wdt, seed=0, residual=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, D, generator=g)
    x[:, :: max(1, D // 5)] *= 20
    r = torch.randn(M, D, generator=g) * 2 if residual else None
    w = 1 + 0.3 * torch.randn(D, generator=g)
    return x.to(dt), w.to(wdt), None if r is None else r.to(dt)


def _dev(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


@pytest.mark.parametrize("M,D", SHAPES)
@pytest.mark.parametrize("dt,wdt", [(BF, BF), (BF, F32), (F32, F32), (F32, BF)])
@pytest.mark.parametrize("residual", [True, False])
def test_forward(M, D, dt, wdt, residual):
    x, w, r = _inputs(M, D, dt, wdt, residual=residual)
    y, s, rstd = ops.rmsnorm_fwd(*_dev(x, w, r), eps=1e-5)
    ry, rs, rr = O.rmsnorm(x, w, r, 1e-5)
    assert torch.equal(s.cpu(), O.stream(x, r))
    steps = (D / 32 + 48) * U
    assert torch.all((rstd.cpu().double() - rr).abs() <= steps * rr)
    assert torch.all((y.cpu().double() - ry).abs() <= (_half(dt) + steps) * ry.abs() + 1e-30)


@pytest.mark.parametrize("M,D", SHAPES)
@pytest.mark.parametrize("dt,wdt", [(BF, BF), (F32, F32), (BF, F32)])
@pytest.mark.parametrize("residual", [True, False])
def test_forward_e4m3(M, D, dt, wdt, residual):
    x, w, r = _inputs(M, D, dt, wdt, seed=1, residual=residual)
    if M > 2:
        x[2] = 0
        if r is not None:
            r[2] = 0
    q, scale, s, rstd = ops.rmsnorm_fwd_e4m3(*_dev(x, w, r))
    ry, rs, rr = O.rmsnorm(x, w, r)
    assert torch.equal(s.cpu(), O.stream(x, r))
    steps = (D / 32 + 48) * U
    top = ry.abs().amax(1)
    want = torch.where(top > 0, top / O.E4M3_MAX, torch.ones_like(top))
    got = scale.cpu().double()
    assert torch.all((got - want).abs() <= steps * want)
    # half a step of e4m3: 2^-4 of a normal value, 2^-10 of the scale below the normals
    value = q.cpu().float().double() * got[:, None]
    bound = torch.maximum(ry.abs() * 2 ** -4, got[:, None] * 2 ** -10) * (1 + 2 * steps) + 2 * steps * ry.abs()
    assert torch.all((value - ry).abs() <= bound)
    nz = top > 0
    assert torch.all(q.cpu().float().abs().amax(1)[nz] == O.E4M3_MAX)


@pytest.mark.parametrize("M,D", SHAPES + [(1500, 520), (2000, 3584), (1201, 1029), (3000, 2051),
                                            (1000, 8190), (701, 16381), (1777, 1556)])
@pytest.mark.parametrize("dt,wdt", [(BF, BF), (BF, F32), (F32, F32), (F32, BF)])
@pytest.mark.parametrize("with_ds", [True, False])
def test_backward(M, D, dt, wdt, with_ds):
    s, w, dy = _inputs(M, D, dt, wdt, seed=2)
    ds = _inputs(M, D, dt, wdt, seed=3)[0] * 0.25 if with_ds else None
    rstd = O.rmsnorm(s, w)[2].float()
    dx, dw = ops.rmsnorm_bwd(*_dev(dy, s, w, rstd, ds))
    rx, rw = O.rmsnorm_grad(dy, s, w, rstd, ds)
    r, g, S = rstd.double()[:, None], (dy.double() * w.double()).abs(), s.double().abs()
    along = S * r ** 3 * (g * S).mean(1, keepdim=True)
    size = r * g + along + (0 if ds is None else ds.double().abs())
    bound = _half(dt) * rx.abs() + (D / 32 + 48) * U * along + 8 * U * size
    assert torch.all((dx.cpu().double() - rx).abs() <= bound)
    mass = (dy.double().abs() * S * r).sum(0)
    assert dw.dtype == wdt
    assert torch.all((dw.cpu().double() - rw).abs() <= _half(wdt) * rw.abs() + (M + 48) * U * mass)


def test_gradient_against_differences():
    """The gradient formula itself, in f64 on the CPU, against central
    differences; the kernel is held to that formula above."""
    g = torch.Generator().manual_seed(5)
    x, w, dy = (torch.randn(3, 11, generator=g, dtype=torch.float64), torch.randn(11, generator=g, dtype=torch.float64),
                torch.randn(3, 11, generator=g, dtype=torch.float64))
    y, s, rstd = O.rmsnorm(x, w)
    dx, dw = O.rmsnorm_grad(dy, x, w, rstd)
    h = 1e-6
    for i in range(3):
        for j in range(11):
            d = torch.zeros_like(x)
            d[i, j] = h
            num = ((O.rmsnorm(x + d, w)[0] - O.rmsnorm(x - d, w)[0]) * dy).sum() / (2 * h)
            assert abs(num - dx[i, j]) < 1e-7
    for j in range(11):
        d = torch.zeros_like(w)
        d[j] = h
        num = ((O.rmsnorm(x, w + d)[0] - O.rmsnorm(x, w - d)[0]) * dy).sum() / (2 * h)
        assert abs(num - dw[j]) < 1e-7


@pytest.mark.parametrize("D", [96, 1001, 3584])
def test_rows_that_hold_no_number_stay_alone(D):
    """A NaN or an infinity makes its own row NaN (an infinity: NaN where it
    stands) and leaves the other rows as they are."""
    x, w, r = _inputs(6, D, BF, BF, seed=7)
    clean = [t.cpu() for t in ops.rmsnorm_fwd(*_dev(x, w, r))]
    q0, sc0, *_ = ops.rmsnorm_fwd_e4m3(*_dev(x, w, r))
    x[1, D // 2] = float("nan")
    x[4, 3] = float("inf")
    y, s, rstd = [t.cpu() for t in ops.rmsnorm_fwd(*_dev(x, w, r))]
    q, sc, *_ = ops.rmsnorm_fwd_e4m3(*_dev(x, w, r))
    assert y[1].isnan().all() and rstd[1].isnan()
    assert y[4, 3].isnan() and rstd[4] == 0
    assert sc.cpu()[1].isnan() and sc.cpu()[4].isnan()
    for k in (0, 2, 3, 5):
        assert torch.equal(y[k], clean[0][k]) and rstd[k] == clean[2][k]
        assert torch.equal(q[k].view(torch.uint8), q0[k].view(torch.uint8)) and sc[k] == sc0[k]


def test_tiny_rows():
    """Rows far below eps^(1/2): finite, and e4m3 rows still reach 448."""
    x, w, _ = _inputs(4, 256, F32, F32, seed=8, residual=False)
    x[0] *= 1e-20
    x[1] *= 1e-37
    x[2, 1:] = 0
    q, scale, _, rstd = ops.rmsnorm_fwd_e4m3(*_dev(x, w), eps=0.0)
    assert torch.isfinite(q.float()).all()
    q, scale, _, rstd = ops.rmsnorm_fwd_e4m3(*_dev(x, w))
    assert torch.isfinite(q.float()).all() and torch.isfinite(scale).all()
    assert q.float().abs().amax(1)[0] == 448 and q.float().abs().amax(1)[2] == 448


def test_no_rows():
    x, w = torch.empty(0, 64, device=DEV, dtype=BF), torch.ones(64, device=DEV, dtype=F32)
    y, s, rstd = ops.rmsnorm_fwd(x, w)
    assert y.shape == (0, 64) and rstd.shape == (0,)
    q, scale, _, _ = ops.rmsnorm_fwd_e4m3(x, w, x)
    assert q.shape == (0, 64) and scale.shape == (0,)
    dx, dw = ops.rmsnorm_bwd(x, x, w, rstd)
    assert dx.shape == (0, 64) and torch.equal(dw, torch.zeros_like(w))


@pytest.mark.parametrize("D", [64, 3584, 1001])
@pytest.mark.parametrize("off", [1, 3, 8])
def test_pointers_off_the_16_byte_grid(D, off):
    """Contiguous tensors that start anywhere in their storage."""
    x, w, r = _inputs(5, D, BF, BF, seed=9)
    def shift(t):
        buf = torch.zeros(t.numel() + off, dtype=t.dtype, device=DEV)
        buf[off:] = t.flatten().to(DEV)
        return buf[off:].view(t.shape)
    a = ops.rmsnorm_fwd(*_dev(x, w, r))
    b = ops.rmsnorm_fwd(shift(x), shift(w), shift(r))
    ry = O.rmsnorm(x, w, r)[0]
    for y in (a[0], b[0]):
        assert torch.all((y.cpu().double() - ry).abs() <= (_half(BF) + (D / 32 + 48) * U) * ry.abs())
    rstd = O.rmsnorm(x, w)[2].float().to(DEV)
    dx, dw = ops.rmsnorm_bwd(*_dev(r, x, w), rstd)
    ex, ew = ops.rmsnorm_bwd(shift(r), shift(x), shift(w), rstd)
    assert torch.allclose(dx.float(), ex.float(), rtol=2 ** -7, atol=1e-5)
    assert torch.allclose(dw.float(), ew.float(), rtol=2 ** -7, atol=1e-4)


def test_run_to_run_and_other_streams_and_graph():
    x, w, r = _dev(*_inputs(777, 1368, BF, F32, seed=10))
    first = ops.rmsnorm_fwd_e4m3(x, w, r) + ops.rmsnorm_bwd(r, x, w, ops.rmsnorm_fwd(x, w)[2])
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        second = ops.rmsnorm_fwd_e4m3(x, w, r) + ops.rmsnorm_bwd(r, x, w, ops.rmsnorm_fwd(x, w)[2])
        st.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            third = ops.rmsnorm_fwd_e4m3(x, w, r) + ops.rmsnorm_bwd(r, x, w, ops.rmsnorm_fwd(x, w)[2])
    torch.cuda.current_stream().wait_stream(st)
    for t in third:
        t.view(torch.uint8).zero_() if t.dtype == torch.float8_e4m3fn else t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(first, second, third):
        for t in (b, c):
            assert torch.equal(a.view(torch.uint8), t.view(torch.uint8))


def test_refusals():
    x, w = torch.ones(4, 8, device=DEV, dtype=BF), torch.ones(8, device=DEV, dtype=BF)
    with pytest.raises(ValueError):
        ops.rmsnorm_fwd(x, w[:4])
    with pytest.raises(ValueError):
        ops.rmsnorm_fwd(x[0], w)
    with pytest.raises(ValueError):
        ops.rmsnorm_fwd(x.t(), w[:4])
    with pytest.raises(ValueError):
        ops.rmsnorm_fwd(x, w, x[:2])
    with pytest.raises(TypeError):
        ops.rmsnorm_fwd(x, w, x.float())
    with pytest.raises(TypeError):
        ops.rmsnorm_fwd(x.half(), w)
    with pytest.raises(ValueError):
        ops.rmsnorm_fwd(x.cpu(), w)
    with pytest.raises(Exception, match="eps"):
        ops.rmsnorm_fwd(x, w, eps=-1.0)
    with pytest.raises(ValueError):
        ops.rmsnorm_bwd(x, x, w, torch.ones(3, device=DEV))
