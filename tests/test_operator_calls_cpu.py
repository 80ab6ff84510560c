"""Refusals and host-side behaviour of the operators around the block that need
no GPU."""
import ctypes
import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from torch._subclasses.fake_tensor import FakeTensorMode

import swiglu_block as SB
import swiglu_recompute as SR
from swiglu_b200 import _lib, library, tp

P = 256
TOP = 2 ** 31 - 1


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


@pytest.fixture
def calls(monkeypatch):
    """Names of the kernels that the Functions call; they run as the registered
    ops' fake forms, on fake tensors."""
    names = []

    class Recorded:
        def __getattr__(self, name):
            names.append(name)
            return getattr(library._Traced, name)

    for mod in (SR, SB):
        monkeypatch.setattr(mod, "kernels", lambda: Recorded())
    with FakeTensorMode():
        yield names


def _refused(lib, rc, text):
    assert rc == 1 and text in lib.swiglu_b200_last_error_message(), (rc, lib.swiglu_b200_last_error_message())


@pytest.mark.parametrize("cols", [TOP, TOP - 1023])
def test_norm_rows_whose_column_numbers_would_overflow(lib, cols):
    """The looping kernels add up to 1024 to an int column number: past
    2^31 - 1025 columns it would turn negative inside the row."""
    eps = ctypes.byref(ctypes.c_float(1e-6))
    n = ctypes.c_int64(0)
    _refused(lib, lib.swiglu_b200_rmsnorm_fwd(P, P, P, P, P, P, 1, cols, eps, 1, 1, None), b"at most 2147482623 columns")
    _refused(lib, lib.swiglu_b200_rmsnorm_fwd_e4m3(P, P, P, P, P, P, P, 1, cols, eps, 1, 1, None), b"at most")
    _refused(lib, lib.swiglu_b200_rmsnorm_bwd(P, P, P, P, P, P, P, P, 1 << 40, 1, cols, 1, 1, None), b"at most")
    _refused(lib, lib.swiglu_b200_rmsnorm_bwd_workspace(1, cols, 148, ctypes.byref(n)), b"at most")
    assert lib.swiglu_b200_rmsnorm_bwd_workspace(1, TOP - 1024, 148, ctypes.byref(n)) == 0


def test_mxfp4_matrices_whose_tiles_would_overflow(lib):
    """Rows and columns are rounded up to tiles of up to 256 in ints."""
    wide, tall = 2 ** 31 - 32, 2 ** 31 - 8
    q, d, m = lib.swiglu_b200_quantize_mxfp4, lib.swiglu_b200_dequantize_mxfp4, lib.swiglu_b200_matmul_mxfp4
    for f in (q, d):
        _refused(lib, f(P, P, P, 1, wide, 1, None), b"at most 2147483392 rows and columns")
        _refused(lib, f(P, P, P, tall, 32, 1, None), b"at most 2147483392 rows and columns")
    _refused(lib, m(P, P, P, P, P, 1, 8, wide, 1, None), b"at most")
    _refused(lib, m(P, P, P, P, P, 1, tall, 32, 1, None), b"at most")
    _refused(lib, m(P, P, P, P, P, tall, 8, 32, 1, None), b"at most")
    f = lib.swiglu_b200_fused_matmul_swiglu_mxfp4
    _refused(lib, f(P, P, P, P, P, P, tall, 32, 128, 0, None), b"at most")
    # an empty matrix of the largest size that is left is no error
    assert q(None, None, None, 0, 2 ** 31 - 256, 1, None) == 0


@pytest.mark.parametrize("precision", ["e4m3", "mxfp4"])
def test_few_bit_block_wants_a_bf16_stream_and_parameters(precision):
    """Refused before any kernel runs: an f32 stream or weight used to pass the
    forward and to fail in the backward, after preact had been overwritten."""
    b = SB.SwiGLUPreNormBlock(64, 64, precision=precision)
    x = torch.zeros(4, 64)
    for grad in (True, False):
        with torch.set_grad_enabled(grad):
            with pytest.raises(TypeError, match="bf16 stream"):
                b(x, x)
            with pytest.raises(TypeError, match="bf16 stream"):
                b(x)
    b.w2.data = b.w2.data.float()
    with pytest.raises(TypeError, match="bf16 parameters"):
        b(x.bfloat16(), x.bfloat16())


@pytest.mark.parametrize("which", ["fp4", *SB.PRECISIONS])
def test_evaluation_without_gradients_writes_no_preact(calls, which):
    """Under torch.no_grad, with parameters that require gradients, the modules take
    the forms that write h alone; with gradients, those that write preact too."""
    bf = torch.bfloat16
    m = SR.SwiGLUMLPFP4Forward(128, 256, dtype=bf) if which == "fp4" else SB.SwiGLUPreNormBlock(128, 256, precision=which)
    gemm1 = {"fp4": "swiglu_fwd_mxfp4", "mxfp4": "swiglu_fwd_mxfp4", "e4m3": "swiglu_fwd_e4m3", "bf16": "swiglu_fwd"}[which]
    x = torch.empty(64, 128, dtype=bf)
    with torch.no_grad():
        m(x)
    assert f"{gemm1}_h" in calls and gemm1 not in calls
    calls.clear()
    m(x)
    assert gemm1 in calls and f"{gemm1}_h" not in calls


def test_fp4_training_wants_bf16_parameters():
    """As the block: f32 weights passed the forward and failed in the backward."""
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    m = SR.SwiGLUMLPFP4Forward(64, 64)
    half = SR.SwiGLUMLPFP4Forward(64, 64, dtype=torch.bfloat16)
    half.w2.data = half.w2.data.float()
    for mlp in (m, half):
        with pytest.raises(TypeError, match="bf16 activations and parameters"):
            mlp(x)
        with pytest.raises(ValueError, match="CUDA"), torch.no_grad():  # allowed as far as the device
            mlp(x)


@pytest.mark.parametrize("which", ["fp4", "norm", *SB.PRECISIONS])
@pytest.mark.parametrize("leaf", ["x", "all"])
def test_second_derivatives_are_refused(calls, which, leaf):
    """A penalty on a gradient used to drop out of a loss in silence."""
    bf = torch.bfloat16
    if which == "fp4":
        m = SR.SwiGLUMLPFP4Forward(64, 64, dtype=bf)
    else:
        m = SB.RMSNormResidual(64) if which == "norm" else SB.SwiGLUPreNormBlock(64, 64, precision=which)
    x = torch.empty(32, 64, dtype=bf, requires_grad=True)
    params = list(m.parameters())
    y = m(x) if which in ("fp4", "norm") else m(x)[0]
    leaves = [x] if leaf == "x" else [x, *params]
    grads = torch.autograd.grad(y.sum(), leaves, create_graph=True)
    assert all(g.shape == t.shape and g.dtype == t.dtype for g, t in zip(grads, leaves))
    for g in grads:
        with pytest.raises(RuntimeError, match="no second derivative"):
            (params[0].square().sum() + g.square().sum()).backward()
    y = m(x) if which in ("fp4", "norm") else m(x)[0]   # and a plain backward is as before
    assert not any(g.requires_grad for g in torch.autograd.grad(y.sum(), leaves))


def test_sharded_clipping_takes_any_iterable(monkeypatch):
    """A generator was used up by the norm, and the scaling found nothing; an empty
    one counted as some gradients."""
    scaled = []
    monkeypatch.setattr(tp.dist, "all_reduce", lambda t, group=None: None)
    monkeypatch.setattr(tp.ops, "grad_norm", lambda ts: torch.cat([t.flatten() for t in list(ts)]).norm())
    monkeypatch.setattr(tp.ops, "clip_grads_by_norm_", lambda ts, norm, max_norm: scaled.extend(ts))
    grads = [torch.full((4,), 3.0), torch.full((5,), 4.0)]
    norm = tp.clip_sharded_grad_norm_((g for g in grads), 1.0, torch.device("cpu"))
    assert abs(norm.item() - (36 + 80) ** 0.5) < 1e-5 and all(a is b for a, b in zip(scaled, grads)) and len(scaled) == 2
    assert tp.clip_sharded_grad_norm_(iter(()), 1.0, torch.device("cpu")) == 0


def _replicated_worker(rank, world, port, q):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        # the local parts on the CPU; the joining of the ranks is what is tested
        tp.ops.grad_norm = lambda ts: torch.cat([t.flatten() for t in ts]).double().norm().float()

        def scale(ts, norm, max_norm, out=None):
            for t in ts:
                t.mul_(min(1.0, max_norm / (float(norm) + 1e-6)))

        tp.ops.clip_grads_by_norm_ = scale
        g = torch.Generator().manual_seed(rank)
        shards = [torch.randn(5, 3, generator=g)] if rank < 2 else []
        both = [torch.arange(7.0)]
        keep = [t.clone() for t in shards]
        norm = tp.clip_sharded_grad_norm_(shards, 0.5, torch.device("cpu"), replicated=both)
        # by value: a tensor would travel by a handle to memory that the rank takes with it
        q.put((rank, norm.item(), *([t.tolist() for t in ts] for ts in (keep, shards, both))))
    finally:
        dist.destroy_process_group()


def test_sharded_clipping_counts_replicated_gradients_once():
    world = 3
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    procs = [ctx.Process(target=_replicated_worker, args=(r, world, port, q)) for r in range(world)]
    for p in procs:
        p.start()
    res = [q.get(timeout=120) for _ in range(world)]
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    every = torch.cat([torch.tensor(t).flatten() for r in res for t in r[2]] + [torch.arange(7.0)]).double()
    want = every.norm().item()
    for _, norm, before, after, both in res:
        assert abs(norm - want) <= 1e-6 * want
        for a, b in zip([*before, torch.arange(7.0)], [*after, both[0]]):
            assert torch.allclose(torch.tensor(b), torch.as_tensor(a) * (0.5 / want), rtol=1e-5)
