"""Global gradient norm and clipping against their 64-bit forms.

Tolerances: at most 64 squares are summed in f32 before f64 takes over, so the
squared norm is off by at most 64 * 2^-24 and the norm by half of that, plus
its rounding to f32; a clipped value by eps/2 of its type on top."""
import pytest
import torch

from oracle import operators as O
from swiglu_b200 import ops

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = 2.0 ** -24
BF, F32 = torch.bfloat16, torch.float32
NORM_TOL = 34 * U


def _list(shapes, dtypes, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(*s, generator=g) * scale).to(dtypes[i % len(dtypes)]) for i, s in enumerate(shapes)]


LISTS = {
    "one": [(1,)],
    "block": [(200,), (528, 200), (200, 264)],
    "ragged": [(1,), (0,), (7,), (15,), (17, 3), (0, 4), (4097,), (33, 129)],
    "chunks": [(256 * 8 * 8,), (256 * 8 * 8 + 1,), (256 * 8 * 8 - 1,), (100001,)],
    "many": [(k % 37,) for k in range(400)],
    "large": [(3001, 2003), (64,), (1500, 999)],
}


@pytest.mark.parametrize("name", LISTS)
@pytest.mark.parametrize("dtypes", [(BF,), (F32,), (F32, BF)])
@pytest.mark.parametrize("ratio", [0.3, 1.7])
@pytest.mark.parametrize("inplace", [True, False])
def test_clip(name, dtypes, ratio, inplace):
    ts = _list(LISTS[name], dtypes)
    norm = O.clip(ts, 1.0)[0]
    max_norm = float(norm) * ratio
    rn, rts = O.clip(ts, max_norm)
    dev = [t.to(DEV) for t in ts]
    out = None if inplace else [torch.full_like(t, 7.0) for t in dev]
    n0 = ops.grad_norm(dev)
    n = ops.clip_grad_norm_(dev, max_norm, out=out)
    assert n.shape == () and n.dtype == F32
    for v in (n0, n):
        assert abs(v.cpu().double() - rn) <= NORM_TOL * rn
    for t, d, o, r in zip(ts, dev, dev if inplace else out, rts):
        assert torch.all((o.cpu().double() - r).abs() <= (torch.finfo(t.dtype).eps / 2 + NORM_TOL + 2 * U) * r.abs() + 1e-38)
        if not inplace:
            assert torch.equal(d.cpu(), t)
        if ratio > 1:
            assert torch.equal(o.cpu(), t)


def test_known_norm_scales_alone():
    ts = [t.to(DEV) for t in _list(LISTS["block"], (BF, F32))]
    norm = ops.grad_norm(ts)
    a = [t.clone() for t in ts]
    ops.clip_grads_by_norm_(a, norm, 2.0)
    b = [torch.empty_like(t) for t in ts]
    ops.clip_grad_norm_(ts, 2.0, out=b)
    for u, v in zip(a, b):
        assert torch.allclose(u.float(), v.float(), rtol=2 ** -7, atol=0)


@pytest.mark.parametrize("scale", [1e-30, 1e-22, 1e18, 1e25, 1e36])
def test_values_whose_squares_leave_f32(scale):
    ts = _list([(5000,), (300, 7)], (F32, BF), scale=scale)
    rn, rts = O.clip(ts, scale)
    dev = [t.to(DEV) for t in ts]
    n = ops.clip_grad_norm_(dev, scale)
    assert abs(n.cpu().double() - rn) <= NORM_TOL * rn
    for o, r in zip(dev, rts):
        assert torch.all((o.cpu().double() - r).abs() <= (torch.finfo(o.dtype).eps / 2 + NORM_TOL + 2 * U) * r.abs() + 1e-38)


def test_zeros_nan_and_infinity():
    z = [torch.zeros(100, device=DEV), torch.zeros(3, 5, device=DEV, dtype=BF)]
    assert ops.clip_grad_norm_(z, 1.0) == 0 and not z[0].any()
    z[0][7] = float("inf")
    assert ops.clip_grad_norm_(z, 1.0) == float("inf")
    assert z[0][7].isnan() and z[0][8] == 0
    assert ops.clip_grad_norm_(z, 1.0).isnan()
    assert z[0].isnan().all() and z[1].isnan().all()
    e = [torch.empty(0, device=DEV)]
    assert ops.grad_norm(e) == 0 and ops.clip_grad_norm_(e, 1.0) == 0


@pytest.mark.parametrize("off_in,off_out", [(1, 1), (3, 3), (1, 2), (0, 5)])
def test_tensors_off_the_16_byte_grid(off_in, off_out):
    src = torch.randn(20000).to(BF)
    buf, obuf = torch.zeros(20000 + off_in, dtype=BF, device=DEV), torch.zeros(20010 + off_out, dtype=BF, device=DEV)
    t, o = buf[off_in:], obuf[off_out:off_out + 20000]
    t.copy_(src)
    rn, (r,) = O.clip([src], 3.0)
    n = ops.clip_grad_norm_([t], 3.0, out=[o])
    assert abs(n.cpu().double() - rn) <= NORM_TOL * rn
    assert torch.all((o.cpu().double() - r).abs() <= (2 ** -8 + NORM_TOL + 2 * U) * r.abs())
    assert not obuf[:off_out].any() and not obuf[off_out + 20000:].any()


def test_in_place_bumps_the_version_and_runs_in_a_graph():
    ts = [torch.randn(5000, device=DEV), torch.randn(70, 9, device=DEV).to(BF)]
    v = ts[0]._version
    keep = [t.clone() for t in ts]
    first = ops.clip_grad_norm_(ts, 1.0)
    assert ts[0]._version > v
    clipped = [t.clone() for t in ts]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        n = ops.clip_grad_norm_(ts, 1.0)
    for t, k in zip(ts, keep):
        t.copy_(k)
    graph.replay()
    torch.cuda.synchronize()
    assert n == first and all(torch.equal(a, b) for a, b in zip(ts, clipped))


def test_dense_tensors_of_any_dimension_order():
    src = torch.randn(40, 30, 7)
    t = src.to(DEV).permute(2, 0, 1)
    u = src.to(BF).to(DEV).transpose(0, 1)
    rn, (r, ru) = O.clip([src, src.to(BF)], 2.0)
    n = ops.clip_grad_norm_([t, u], 2.0)
    assert abs(n.cpu().double() - rn) <= NORM_TOL * rn
    assert torch.all((t.permute(1, 2, 0).cpu().double() - r).abs() <= (NORM_TOL + 4 * U) * r.abs())
    assert torch.all((u.transpose(0, 1).cpu().double() - ru).abs() <= (2 ** -8 + NORM_TOL + 2 * U) * ru.abs())
    with pytest.raises(ValueError):
        ops.clip_grad_norm_([t], 1.0, out=[torch.empty(7, 40, 30, device=DEV)])     # other strides
    for bad in (t[:, ::2], torch.ones(1, device=DEV).expand(5)):
        with pytest.raises(ValueError):
            ops.grad_norm([bad])


def test_two_streams_at_once():
    lists = [[torch.randn(300000, device=DEV), torch.randn(1000, 77, device=DEV).to(BF)] for _ in range(2)]
    want = [ops.grad_norm(ts) for ts in lists]
    outs = [[torch.empty_like(t) for t in ts] for ts in lists]
    ref = [[torch.empty_like(t) for t in ts] for ts in lists]
    for ts, o in zip(lists, ref):
        ops.clip_grad_norm_(ts, 1.0, out=o)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for st, ts, o in zip(streams, lists, outs):
            with torch.cuda.stream(st):
                got.append(ops.clip_grad_norm_(ts, 1.0, out=o))
        torch.cuda.synchronize()
        for k in range(2):
            assert got[k] == want[k] and all(torch.equal(a, b) for a, b in zip(outs[k], ref[k]))


def test_refusals():
    t = torch.ones(64, device=DEV)
    with pytest.raises(ValueError):
        ops.grad_norm([])
    with pytest.raises(ValueError):
        ops.clip_grad_norm_([t, t[:4].cpu()], 1.0)
    with pytest.raises(ValueError):
        ops.clip_grad_norm_([t[::2]], 1.0)
    with pytest.raises(TypeError):
        ops.grad_norm([t.half()])
    with pytest.raises(Exception, match="overlaps"):
        ops.clip_grad_norm_([t, t], 1.0)
    with pytest.raises(Exception, match="overlaps"):
        ops.clip_grad_norm_([t[:40], t[32:]], 1.0)
    with pytest.raises(Exception, match="overlaps"):
        ops.clip_grad_norm_([t[:8]], 1.0, out=[t[4:12]])
    for bad in (-1.0, float("nan")):
        with pytest.raises(Exception, match="max_norm"):
            ops.clip_grad_norm_([t], bad)
    with pytest.raises(ValueError):
        ops.clip_grad_norm_([t], 1.0, out=[t.to(BF)])
    with pytest.raises(ValueError):
        ops.clip_grads_by_norm_([t], torch.ones(2, device=DEV), 1.0)
    assert torch.equal(t, torch.ones_like(t))
    # the same tensor twice is fine where nothing is written
    assert abs(ops.grad_norm([t, t]).item() - 128 ** 0.5) < 1e-4
