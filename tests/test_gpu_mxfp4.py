"""MXFP4 operands: quantisation bit for bit, its inverse exactly, and the
product against the f64 product of the same values.

Product tolerance: eps/2 of the output type for its rounding, plus the f32
accumulation: one addition per 64 products, each off by at most 2^-22 (the
tensor core may cut instead of round) of the sum of magnitudes, with 8 more
for the sums inside an instruction."""
import pytest
import torch

from oracle import operators as O
from oracle import swiglu_oracle as SO
from swiglu_b200 import _lib, ops

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def _matrix(R, K, dt, seed=0):
    g = torch.Generator().manual_seed(seed)
    t = torch.randn(R, K, generator=g) * torch.logspace(-3, 3, R)[:, None]
    t[:, ::17] *= 9
    return t.to(dt)


@pytest.mark.parametrize("R,K", [(1, 32), (1, 3584), (5, 64), (37, 1056), (128, 128), (129, 160), (300, 512), (257, 2080)])
@pytest.mark.parametrize("dt", [BF, F32])
def test_quantize_bit_for_bit_and_back(R, K, dt):
    t = _matrix(R, K, dt)
    if R > 4:
        t[1] = 0
        t[2, 0:32] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 4).to(dt)     # ties
        t[2, 32:64] = -t[2, 0:32] * 2.0 ** -20
        t[3, 0:32] = torch.tensor([7.9, -0.2, 0.0, -0.0] * 8).to(dt)                           # saturation, signs
    q, scale = ops.quantize_mxfp4(t.to(DEV))
    code, byte = O.mx_quantize(t)
    assert torch.equal(scale.cpu(), O.mx_tiles(byte))
    assert torch.equal(q.cpu(), O.mx_pack(code))
    for out in (BF, F32):
        back = ops.dequantize_mxfp4(q, scale, dtype=out)
        assert back.dtype == out and torch.equal(back.cpu().double(), O.mx_values(code, byte))


def test_quantize_range_ends():
    """The largest and smallest exponents, subnormals, infinities and NaN."""
    t = torch.zeros(8, 64)
    t[0, :32] = torch.finfo(F32).max
    t[1, 3] = 2.0 ** -126
    t[2, 5] = 2.0 ** -149
    t[3, 7] = -(2.0 ** -124) * 1.5
    t[4, :32] = torch.linspace(-1, 1, 32) * 2.0 ** -125
    t[5, 9] = float("inf")
    t[6, 40] = float("nan")
    t[7] = torch.linspace(-3e38, 3e38, 64)
    q, scale = ops.quantize_mxfp4(t.to(DEV))
    code, byte = O.mx_quantize(t)
    assert torch.equal(scale.cpu(), O.mx_tiles(byte))
    live = (byte != 255).repeat_interleave(32, 1)
    got = torch.stack((q.cpu() & 15, q.cpu() >> 4), -1).view(8, 64)
    assert torch.equal(got[live], code[live])
    back = ops.dequantize_mxfp4(q, scale, dtype=F32).cpu()
    assert back[5, :32].isnan().all() and back[6, 32:].isnan().all()
    assert torch.equal(back[live].double(), O.mx_values(code, byte)[live])


def _product(M, N, K, out, seed=0, special=None):
    a, b = _matrix(M, K, BF, seed), _matrix(N, K, BF, seed + 1) * K ** -0.5
    b = b.to(BF)
    if special:
        special(a, b)
    aq, asc = ops.quantize_mxfp4(a.to(DEV))
    bq, bsc = ops.quantize_mxfp4(b.to(DEV))
    c = ops.matmul_mxfp4(aq, asc, bq, bsc, out_dtype=out)
    av, bv = O.mx_values(*O.mx_quantize(a)), O.mx_values(*O.mx_quantize(b))
    return c, av, bv


def _check(c, av, bv, out):
    K = av.shape[1]
    want, mass = av @ bv.t(), av.abs() @ bv.abs().t()
    bound = torch.finfo(out).eps / 2 * want.abs() + (K / 64 + 8) * 2.0 ** -22 * mass
    err = (c.cpu().double() - want).abs()
    assert torch.all(err <= bound), (err - bound).max()
    assert ops.device_status(0) == 0


@pytest.mark.parametrize("M,N,K", [(1, 8, 32), (1, 3584, 3584), (2, 128, 64), (3, 136, 96), (7, 256, 14336), (16, 1000, 1056),
                                   (17, 520, 2048), (33, 3584, 544), (64, 264, 3616), (65, 128, 256), (100, 2816, 1024),
                                   (128, 512, 512), (129, 776, 288), (256, 256, 256), (333, 1000, 1440), (512, 3584, 1024),
                                   (700, 1032, 736), (1025, 520, 320), (2048, 2816, 1024), (4096, 1024, 2816), (3000, 8, 64),
                                   (300, 16, 32), (9, 16392, 96), (130, 40, 8192), (20000, 72, 32)])
@pytest.mark.parametrize("out", [BF, F32])
def test_product(M, N, K, out):
    _check(*_product(M, N, K, out), out)


@pytest.mark.parametrize("layout", [SO.STD, SO.PACKED])
@pytest.mark.parametrize("M,K,H", [(1, 256, 128), (17, 1056, 384), (100, 512, 256), (257, 64, 128), (300, 1440, 640),
                                   (1500, 512, 1408), (4100, 96, 256)])
def test_swiglu_forward(layout, M, K, H):
    """preact as the product gives it (its own tests hold that to f64), h within
    one bf16 rounding of left * silu(gate) of that preact, and the same bits
    whichever outputs are asked for."""
    lay = ops.LAYOUT_STD if layout == SO.STD else ops.LAYOUT_PACKED128
    x, w1 = _matrix(M, K, BF), (_matrix(2 * H, K, BF, 1) * K ** -0.5).to(BF)
    li, gi = SO.col_index(H, layout)
    w = torch.empty_like(w1)
    w[li], w[gi] = w1[:H], w1[H:]
    xq, xs = ops.quantize_mxfp4(x.to(DEV))
    wq, ws = ops.quantize_mxfp4(w.to(DEV))
    preact, h = ops.swiglu_fwd_mxfp4(xq, xs, wq, ws, layout=lay)
    assert torch.equal(preact, ops.matmul_mxfp4(xq, xs, wq, ws))
    p = preact.double().cpu()
    left, gate = p[:, li], p[:, gi]
    ref = left * gate * torch.sigmoid(gate)
    # Half a bf16 step, and the f32 sigmoid 1 / (1 + e^-g) of the fused form. By the
    # CUDA programming guide's table __expf(x) is off by at most 2 + 1.173 |x| ulp and
    # __fdividef by 2, and __fdividef gives 0 for a divisor above 2^126: with the three
    # other roundings (1 + e, g s, l silu) at most 7 + 1.173 |g| ulp of 2^-23, and below
    # g = -87 an absolute |l g| 2^-126. (The pointwise kernel's expf and division are
    # within 2 ulp each.) The gates here reach hundreds.
    bound = (2 ** -8 + (7 + 1.173 * gate.abs()) * 2.0 ** -23) * ref.abs() + (left * gate).abs() * 2.0 ** -126 + 1e-37
    assert torch.all((h.double().cpu() - ref).abs() <= bound)
    assert torch.equal(ops.swiglu_fwd_mxfp4(xq, xs, wq, ws, layout=lay, want_preact=False)[1], h)
    assert torch.equal(ops.swiglu_fwd_mxfp4(xq, xs, wq, ws, layout=lay, want_h=False)[0], preact)
    assert ops.device_status(0) == 0


@pytest.mark.parametrize("M", [1, 5, 40, 130, 600])
def test_rows_are_independent(M):
    """A row whose block holds a NaN is NaN in the product; no other row is."""
    def spoil(a, b):
        a[M // 2, 100] = float("nan")
    c, av, bv = _product(M, 264, 256, F32, special=spoil)
    c = c.cpu()
    assert c[M // 2].isnan().all()
    keep = torch.arange(M) != M // 2
    assert torch.isfinite(c[keep]).all()


def test_product_is_run_to_run_identical_and_runs_elsewhere():
    for M, N, K in [(1, 3584, 3584), (48, 1024, 7168), (333, 1000, 14336), (2048, 1024, 1024)]:
        a, b = _matrix(M, K, BF).to(DEV), _matrix(N, K, BF, 1).to(DEV)
        aq, asc = ops.quantize_mxfp4(a)
        bq, bsc = ops.quantize_mxfp4(b)
        first = ops.matmul_mxfp4(aq, asc, bq, bsc)
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            second = ops.matmul_mxfp4(aq, asc, bq, bsc)
        torch.cuda.current_stream().wait_stream(st)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            third = ops.matmul_mxfp4(aq, asc, bq, bsc)
        graph.replay()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(first, second) and torch.equal(first, third)
    assert ops.device_status(0) == 0


def test_two_streams_at_once_and_a_reserve():
    mats = []
    for k, (M, N, K) in enumerate([(40, 1024, 4096), (700, 1032, 1056)]):
        a, b = _matrix(M, K, BF, k).to(DEV), _matrix(N, K, BF, 9 + k).to(DEV)
        mats.append((*ops.quantize_mxfp4(a), *ops.quantize_mxfp4(b)))
    want = [ops.matmul_mxfp4(*m) for m in mats]
    streams = [torch.cuda.Stream() for _ in mats]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for st, m in zip(streams, mats):
            with torch.cuda.stream(st):
                got.append(ops.matmul_mxfp4(*m))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    _lib.set_sm_reserve(40)
    try:
        for m, w in zip(mats, want):
            assert torch.allclose(ops.matmul_mxfp4(*m).float(), w.float(), rtol=2 ** -6,
                                  atol=2 ** -6 * w.float().abs().max().item())
    finally:
        _lib.set_sm_reserve(0)
    assert ops.device_status(0) == 0


def test_scale_bytes_of_rows_beyond_the_matrix_do_not_matter():
    for M, N, K in [(5, 24, 128), (300, 520, 256)]:
        a, b = _matrix(M, K, BF).to(DEV), _matrix(N, K, BF, 1).to(DEV)
        aq, asc = ops.quantize_mxfp4(a)
        bq, bsc = ops.quantize_mxfp4(b)
        want = ops.matmul_mxfp4(aq, asc, bq, bsc)
        for sc, rows in ((asc, M), (bsc, N)):
            r = torch.arange(sc.shape[0] * 128, device=DEV)
            r = r[r >= rows]
            sc[r // 128, :, r % 32, (r % 128) // 32, :] = 255
        assert torch.equal(ops.matmul_mxfp4(aq, asc, bq, bsc), want)


def test_empty_and_refusals():
    q, s = ops.quantize_mxfp4(torch.empty(0, 64, device=DEV))
    assert q.shape == (0, 32) and s.shape == (0, 1, 32, 4, 4)
    assert ops.dequantize_mxfp4(q, s).shape == (0, 64)
    bq, bs = ops.quantize_mxfp4(torch.ones(16, 64, device=DEV))
    assert ops.matmul_mxfp4(q, s, bq, bs).shape == (0, 16)
    with pytest.raises(ValueError):
        ops.quantize_mxfp4(torch.ones(4, 40, device=DEV))
    with pytest.raises(ValueError):
        ops.quantize_mxfp4(torch.ones(4, 64))
    with pytest.raises(TypeError):
        ops.quantize_mxfp4(torch.ones(4, 64, device=DEV).half())
    with pytest.raises(ValueError):
        ops.quantize_mxfp4(torch.ones(64, 4, device=DEV).t())
    with pytest.raises(Exception, match="16-byte"):
        ops.quantize_mxfp4(torch.ones(65, device=DEV)[1:].view(1, 64))
    with pytest.raises(ValueError):
        ops.dequantize_mxfp4(bq, bs[:, :0])
    with pytest.raises(TypeError):
        ops.dequantize_mxfp4(bq.float(), bs)
    cq, cs = ops.quantize_mxfp4(torch.ones(16, 96, device=DEV))
    with pytest.raises(ValueError):
        ops.matmul_mxfp4(bq, bs, cq, cs)
    dq, ds = ops.quantize_mxfp4(torch.ones(12, 64, device=DEV))
    with pytest.raises(Exception, match="multiple of 8"):
        ops.matmul_mxfp4(bq, bs, dq, ds)
