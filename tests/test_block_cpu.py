"""The pre-norm block and sharded clipping without a GPU: the registered ops
trace, shapes come from their fake forms, bad arguments are refused, and the
ranks' norms are joined (gloo)."""
import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp
from torch.fx.experimental.proxy_tensor import make_fx

import swiglu_block as SB
import swiglu_recompute as SR
from swiglu_b200 import library

M, D, H, Dout = 64, 128, 256, 96


@pytest.fixture
def traced(monkeypatch):
    for mod in (library, SR, SB):
        monkeypatch.setattr(mod, "kernels", lambda: library._Traced)


def _targets(g):
    return [str(n.target) for n in g.graph.nodes if n.op == "call_function"]


@pytest.mark.parametrize("precision", SB.PRECISIONS)
@pytest.mark.parametrize("residual", [True, False])
def test_block_traces_through_registered_ops(traced, precision, residual):
    bf = dict(dtype=torch.bfloat16, requires_grad=True)
    args = [torch.randn(M, D, **bf), torch.randn(M, D, **bf), torch.randn(D, **bf), torch.randn(2 * H, D, **bf),
            torch.randn(Dout, H, **bf), torch.randn(M, Dout, dtype=torch.bfloat16)]

    def f(x, r, g, w1, w2, gy):
        out = SB.PreNormSwiGLUFunction.apply(x, r if residual else None, g, w1, w2, 1e-6, precision)
        y = out[0] if residual else out
        return (y,) + torch.autograd.grad(y, [x, g, w1, w2], gy)

    g = make_fx(f, tracing_mode="fake")(*args)
    t = _targets(g)
    ours = [x for x in t if x.startswith("swiglu_b200.")]
    foreign = [x for x in t if not x.startswith(("swiglu_b200.", "aten.view", "aten.empty", "aten._unsafe_view",
                                                 "aten.detach"))
               and x != "<built-in function getitem>"]
    assert not foreign, foreign
    assert "swiglu_b200.rmsnorm_bwd.default" in ours
    # the norm's output is formed again in the backward
    norms = [x for x in ours if "rmsnorm_fwd" in x]
    assert len(norms) == 2 and ("swiglu_b200.rmsnorm_fwd_e4m3.default" in norms) == (precision == "e4m3")
    assert ("swiglu_b200.matmul_mxfp4.default" in ours) == (precision == "mxfp4")
    outs = [n for n in g.graph.nodes if n.op == "output"][0].args[0]
    assert [tuple(o.meta["val"].shape) for o in outs] == [(M, Dout), (M, D), (D,), (2 * H, D), (Dout, H)]


def test_fp4_forward_traces(traced):
    args = [torch.randn(M, D, dtype=torch.bfloat16, requires_grad=True),
            torch.randn(2 * H, D, dtype=torch.bfloat16, requires_grad=True),
            torch.randn(Dout, H, dtype=torch.bfloat16, requires_grad=True), torch.randn(M, Dout, dtype=torch.bfloat16)]

    def f(x, w1, w2, gy):
        y = SR.SwiGLUFP4ForwardFunction.apply(x, w1, w2)
        return (y,) + torch.autograd.grad(y, [x, w1, w2], gy)

    t = _targets(make_fx(f, tracing_mode="fake")(*args))
    assert sum(x == "swiglu_b200.quantize_mxfp4.default" for x in t) == 4
    assert sum(x == "swiglu_b200.matmul_mxfp4.default" for x in t) == 1
    assert sum(x == "swiglu_b200.swiglu_fwd_mxfp4.default" for x in t) == 1


def test_refusals():
    with pytest.raises(ValueError):
        SB.SwiGLUPreNormBlock(64, 64, precision="fp6")
    with pytest.raises(TypeError):
        SB.SwiGLUPreNormBlock(64, 64, dtype=torch.float32, precision="mxfp4")
    b = SB.SwiGLUPreNormBlock(64, 64)
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        b(x, x[:2])
    with pytest.raises(ValueError):
        b(x, x.float())
    with pytest.raises(ValueError, match="CUDA"):   # no CPU path
        b(x, x)
    assert SB.clip_grad_norm_(b.parameters(), 1.0) == 0   # no gradients yet
    for name in ("forward_logic", "quantize_mxfp4", "matmul_mxfp4", "rmsnorm_fwd", "rmsnorm_fwd_e4m3", "rmsnorm_bwd",
                 "swiglu_fwd_mxfp4", "swiglu_fwd_mxfp4_h"):
        s = getattr(torch.ops.swiglu_b200, name).default._schema
        assert not any(a.alias_info is not None and a.alias_info.is_write for a in s.arguments), name


def _free_port():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


def _clip_worker(rank, world, port, q):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        from oracle import operators as OP
        from swiglu_b200 import ops, tp

        # the local parts on the CPU; the joining of the ranks is what is tested
        ops.grad_norm = lambda ts: OP.clip(ts, 1.0)[0].float()

        def scale(ts, norm, max_norm, out=None):
            for t in ts:
                t.mul_(min(1.0, max_norm / (float(norm) + 1e-6)))

        ops.clip_grads_by_norm_ = scale
        g = torch.Generator().manual_seed(rank)
        # rank 1 has gradients of another size, rank 2 none at all
        shapes = [[(8, 4), (3,)], [(5,)], []][rank]
        grads = [torch.randn(*s, generator=g) for s in shapes]
        keep = [t.clone() for t in grads]
        norm = tp.clip_sharded_grad_norm_(grads, 0.7, torch.device("cpu"))
        q.put((rank, norm, keep, grads))
    finally:
        dist.destroy_process_group()


def test_sharded_clipping_joins_the_ranks():
    world = 3
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    port = _free_port()
    procs = [ctx.Process(target=_clip_worker, args=(r, world, port, q)) for r in range(world)]
    for p in procs:
        p.start()
    res = sorted([q.get(timeout=120) for _ in range(world)], key=lambda t: t[0])
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    every = torch.cat([t.flatten() for r in res for t in r[2]]).double()
    norm = every.norm()
    for r in res:
        assert abs(r[1].double() - norm) <= 1e-6 * norm
        for before, after in zip(r[2], r[3]):
            assert torch.allclose(after, before * (0.7 / float(norm)), rtol=1e-5)
