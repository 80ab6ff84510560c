"""Cases of the operators around the SwiGLU block: the residual RMS norm that
feeds it (bf16 or row-scaled e4m3 out, and its gradient), the MXFP4 operand
path (quantisation with its inverse, and the product), and the global
gradient norm with clipping.

`run` computes a case in elementary torch operations, or, where `own` is
true, through this package's entry points; both take what `prepare` gives.
"""
import math
import os
import sys

import torch

own = False

EPS = 1e-6
BF16, F32 = "bf16", "f32"
TYPES = {BF16: torch.bfloat16, F32: torch.float32}


def _ops():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "swiglu-recompute_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from swiglu_b200 import ops
    return ops


# ------------------------------------------------------------------- the cases
def listed():
    return [
        # One token of a served model: the norm in front of an e4m3 block, residual added. Latency.
        {"name": "norm_e4m3_token", "op": "norm_e4m3", "rows": 1, "cols": 3584, "type": BF16, "weight": BF16, "residual": True},
        # The same in a training or prefill step of 11136 tokens (the benchmark's second configuration).
        {"name": "norm_e4m3_step", "op": "norm_e4m3", "rows": 11136, "cols": 3584, "type": BF16, "weight": BF16, "residual": True},
        # A long batch at the widest model dimension (the benchmark's fifth configuration), bf16 output.
        {"name": "norm_wide", "op": "norm", "rows": 65536, "cols": 8192, "type": BF16, "weight": F32, "residual": True},
        # The norm's gradient in a training step, with the gradient that arrives on the residual stream.
        {"name": "norm_bwd_step", "op": "norm_bwd", "rows": 11136, "cols": 3584, "type": BF16, "weight": BF16, "residual": True},
        # The gradient on an odd small shape in f32: a test or a small model without a residual.
        {"name": "norm_bwd_odd_f32", "op": "norm_bwd", "rows": 333, "cols": 1001, "type": F32, "weight": F32, "residual": False},
        # A first-layer weight taken to MXFP4 and read back (checking a checkpoint, quantisation-aware steps).
        {"name": "mxfp4_weight", "op": "mxfp4", "rows": 28672, "cols": 3584, "type": BF16},
        # The activations of a small decode batch, a ragged number of rows and of scale tiles.
        {"name": "mxfp4_small", "op": "mxfp4", "rows": 37, "cols": 1056, "type": F32},
        # One token through a first-layer weight in MXFP4: the weight's bytes are the work.
        {"name": "product_token", "op": "product", "rows": 1, "out": 28672, "inner": 3584, "type": BF16},
        # A middling ragged batch over a long contraction, f32 partial results (a tensor-parallel shard's).
        {"name": "product_ragged", "op": "product", "rows": 333, "out": 1000, "inner": 14336, "type": F32},
        # The first-layer product of a training or prefill step.
        {"name": "product_step", "op": "product", "rows": 11136, "out": 28672, "inner": 3584, "type": BF16},
        # Gradients of eight stacked blocks (norm weight, W1, W2), as the stacked benchmark trains.
        {"name": "clip_blocks", "op": "clip", "layers": 8, "dim": 3584, "hidden": 14336, "type": BF16, "ragged": False, "ratio": 0.5},
        # A small model's gradients with ragged extra tensors, in f32.
        {"name": "clip_small", "op": "clip", "layers": 3, "dim": 200, "hidden": 264, "type": F32, "ragged": True, "ratio": 0.25},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm_e4m3", "norm_bwd", "mxfp4", "product", "clip"])
    if op in ("norm", "norm_e4m3", "norm_bwd"):
        cols = _log(rng, 64, 16384)
        cols = rng.choice([cols, -(-cols // 8) * 8, -(-cols // 64) * 64])  # odd ones, and whole vectors
        rows = _log(rng, 1, min(65536, 65536 * 4096 // cols))
        return {"op": op, "rows": rows, "cols": cols, "type": rng.choice([BF16, BF16, F32]), "weight": rng.choice([BF16, F32]),
                "residual": rng.random() < 0.7}
    if op == "mxfp4":
        cols = 32 * _log(rng, 2, 512)
        return {"op": op, "rows": _log(rng, 1, min(65536, 28672 * 3584 // cols)), "cols": cols, "type": rng.choice([BF16, BF16, F32])}
    if op == "product":
        inner, out = 32 * _log(rng, 2, 448), 8 * _log(rng, 8, 3584)
        return {"op": op, "rows": min(_log(rng, 1, 16384), 11136 * 28672 * 3584 // (inner * out)), "out": out, "inner": inner,
                "type": rng.choice([BF16, BF16, F32])}
    return {"op": op, "layers": _log(rng, 1, 12), "dim": 8 * _log(rng, 8, 256), "hidden": 8 * _log(rng, 8, 512), "type": rng.choice([BF16, F32]),
            "ragged": rng.random() < 0.5, "ratio": rng.choice([0.1, 0.5, 0.9, 2.0])}


# ------------------------------------------------------------------ the inputs
def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _activations(g, rows, cols, dtype):
    """Residual-stream values: normal, with a few columns an order larger."""
    t = _randn(g, rows, cols)
    big = torch.randint(0, cols, (max(1, cols // 256),), generator=g, device="cuda")
    t[:, big] *= 12.0
    return t.to(dtype)


def _tiles(byte):
    """[R, K/32] scale bytes as [ceil(R/128), ceil(K/128), 32, 4, 4]: element
    (r, b) at [r / 128, b / 4, r % 32, (r % 128) / 32, b % 4], zeros beyond."""
    R, B = byte.shape
    rt, kt = -(-R // 128), -(-B // 4)
    full = torch.zeros((rt * 128, kt * 4), dtype=torch.uint8, device=byte.device)
    full[:R, :B] = byte
    return full.view(rt, 4, 32, kt, 4).permute(0, 3, 2, 1, 4).contiguous()


def _untile(tiled, rows, blocks):
    rt, kt = tiled.shape[:2]
    return tiled.permute(0, 3, 2, 1, 4).reshape(rt * 128, kt * 4)[:rows, :blocks]


def _powers(device, lowest):
    """2^lowest and the 254 powers above it, exactly."""
    return torch.tensor([2.0 ** (lowest + i) for i in range(255)], dtype=torch.float32, device=device)


def _tables(device):
    """What the plain MXFP4 forms look values up in."""
    levels = [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    return {"powers": _powers(device, -127), "levels": torch.tensor(levels + [-v for v in levels], dtype=torch.float32, device=device)}


def _mx_quantize(t, powers):
    """(codes [R, K] uint8, scale bytes [R, K/32]): a block of 32 values
    shares 2^(floor(log2 amax) - 2), each value is the nearest of
    0 0.5 1 1.5 2 3 4 6 (ties to the even code, larger ones to 6) with its sign."""
    R, K = t.shape
    v = t.float().view(R, K // 32, 32)
    top = torch.frexp(v.abs().amax(-1))[1] - 1                       # floor(log2 amax)
    byte = (top + 125).clamp(0, 254)
    byte = torch.where(v.abs().amax(-1) > 0, byte, torch.zeros_like(byte))
    a = v.abs() * powers[(254 - byte).long()][..., None]
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)).to(torch.uint8)
    code = code + 8 * torch.signbit(v).to(torch.uint8)
    return code.view(R, K), byte.to(torch.uint8)


def _pack(code):
    return code[:, 0::2] | (code[:, 1::2] << 4)


def _mx_values(q, tiled, tables):
    """The values [R, K] that packed codes and tiled scales stand for."""
    R, K = q.shape[0], 2 * q.shape[1]
    code = torch.stack((q & 15, q >> 4), dim=-1).view(R, K)
    scale = tables["powers"][_untile(tiled, R, K // 32).long()]
    return (tables["levels"][code.int()].view(R, K // 32, 32) * scale[..., None]).view(R, K)


def _mx_operand(g, rows, cols, std, powers):
    """A quantised operand as a program holds it, made 4096 rows at a time."""
    q = torch.empty((rows, cols // 2), dtype=torch.uint8, device="cuda")
    byte = torch.empty((rows, cols // 32), dtype=torch.uint8, device="cuda")
    for r in range(0, rows, 4096):
        code, b = _mx_quantize((_randn(g, min(4096, rows - r), cols) * std).to(torch.bfloat16), powers)
        q[r:r + 4096], byte[r:r + 4096] = _pack(code), b
    return q, _tiles(byte)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    s = {"case": case}
    if op in ("norm", "norm_e4m3", "norm_bwd"):
        M, D, dt = case["rows"], case["cols"], TYPES[case["type"]]
        s["weight"] = (1.0 + 0.2 * _randn(g, D)).to(TYPES[case["weight"]])
        s["x"] = _activations(g, M, D, dt)
        if op == "norm_bwd":
            s["rstd"] = torch.rsqrt(s["x"].double().square().mean(-1) + EPS).float()
            s["dy"] = (_randn(g, M, D) * 0.01).to(dt)
            s["ds"] = (_randn(g, M, D) * 0.02).to(dt) if case["residual"] else None
        else:
            s["residual"] = (2.0 * _randn(g, M, D)).to(dt) if case["residual"] else None
    elif op == "mxfp4":
        s["x"] = _activations(g, case["rows"], case["cols"], TYPES[case["type"]])
        s["tables"] = _tables("cuda")
    elif op == "product":
        K = case["inner"]
        s["tables"] = _tables("cuda")
        s["a"], s["a_scale"] = _mx_operand(g, case["rows"], K, 1.0, s["tables"]["powers"])
        s["b"], s["b_scale"] = _mx_operand(g, case["out"], K, K ** -0.5, s["tables"]["powers"])
    else:
        dt = TYPES[case["type"]]
        grads = []
        for layer in range(case["layers"]):
            D, H = case["dim"], case["hidden"]
            shapes = [(D,), (2 * H, D), (D, H)] + ([(7 * layer + 1,), (D + 1, 3)] if case["ragged"] else [])
            for k, shape in enumerate(shapes):
                grads.append((_randn(g, *shape) * 1e-3 * (1 + k)).to(torch.float32 if k == 0 else dt))
        s["grads"] = grads
        s["out"] = [torch.empty_like(t) for t in grads]
        total = math.sqrt(sum(float(t.double().square().sum()) for t in grads))
        s["max_norm"] = case["ratio"] * total
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    ops = _ops()
    case = s["case"]
    op = case["op"]
    if op == "norm":
        return ops.rmsnorm_fwd(s["x"], s["weight"], s["residual"], eps=EPS)
    if op == "norm_e4m3":
        return ops.rmsnorm_fwd_e4m3(s["x"], s["weight"], s["residual"], eps=EPS)
    if op == "norm_bwd":
        return ops.rmsnorm_bwd(s["dy"], s["x"], s["weight"], s["rstd"], s["ds"])
    if op == "mxfp4":
        q, scale = ops.quantize_mxfp4(s["x"])
        return ops.dequantize_mxfp4(q, scale, dtype=TYPES[case["type"]])
    if op == "product":
        return ops.matmul_mxfp4(s["a"], s["a_scale"], s["b"], s["b_scale"], out_dtype=TYPES[case["type"]])
    norm = ops.clip_grad_norm_(s["grads"], s["max_norm"], out=s["out"])
    return [norm] + s["out"]


def _run_plain(s):
    case = s["case"]
    op = case["op"]
    if op in ("norm", "norm_e4m3"):
        x, w, r = s["x"], s["weight"].float(), s["residual"]
        total = x if r is None else (x.float() + r.float()).to(x.dtype)   # the stream as it is stored
        v = total.float()
        rstd = torch.rsqrt(v.square().mean(-1) + EPS)
        y = v * rstd[:, None] * w
        if op == "norm":
            return y.to(x.dtype), total, rstd
        amax = y.abs().amax(-1)
        live = amax > 0
        scale = torch.where(live, amax / 448.0, torch.ones_like(amax))
        q = y * torch.where(live, 448.0 / amax, torch.ones_like(amax))[:, None]
        return q.clamp(-448.0, 448.0).to(torch.float8_e4m3fn), scale, total, rstd
    if op == "norm_bwd":
        v, w, rstd = s["x"].float(), s["weight"].float(), s["rstd"][:, None]
        dy = s["dy"].float()
        xhat = v * rstd
        g = dy * w
        dx = rstd * (g - xhat * (g * xhat).mean(-1, keepdim=True))
        if s["ds"] is not None:
            dx = dx + s["ds"].float()
        return dx.to(s["x"].dtype), (dy * xhat).sum(0).to(s["weight"].dtype)
    if op == "mxfp4":
        code, byte = _mx_quantize(s["x"], s["tables"]["powers"])
        return _mx_values(_pack(code), _tiles(byte), s["tables"]).to(s["x"].dtype)
    if op == "product":
        a, b = _mx_values(s["a"], s["a_scale"], s["tables"]), _mx_values(s["b"], s["b_scale"], s["tables"])
        return (a @ b.t()).to(TYPES[case["type"]])
    squares = torch.stack([t.double().square().sum() for t in s["grads"]])
    norm = squares.sum().sqrt()
    factor = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    for t, o in zip(s["grads"], s["out"]):
        o.copy_(t.float() * factor)
    return [norm.float()] + s["out"]


# ------------------------------------------------------------------ its work
def work(case):
    op = case["op"]
    size = {BF16: 2, F32: 4}
    if op in ("norm", "norm_e4m3", "norm_bwd"):
        M, D, e, w = case["rows"], case["cols"], size[case["type"]], size[case["weight"]]
        n = M * D
        if op == "norm_bwd":  # dy, x, rstd, weight in (the residual's gradient too); dx, dweight out
            return {"bytes": n * e * (3 + case["residual"]) + 4 * M + 2 * D * w, "flops": 9 * n}
        streams = 3 if case["residual"] else 1          # x; residual in and the new stream out
        out = n * e if op == "norm" else n + 4 * M
        return {"bytes": n * e * streams + out + 4 * M + D * w, "flops": 5 * n}
    if op == "mxfp4":  # values in, codes and scales made and read back, values out
        n = case["rows"] * case["cols"]
        return {"bytes": 2 * n * size[case["type"]] + n + n // 16, "flops": 4 * n}
    if op == "product":
        M, N, K = case["rows"], case["out"], case["inner"]
        return {"bytes": (M + N) * K * 17 // 32 + M * N * size[case["type"]], "flops": 2 * M * N * K}
    D, H, L, e = case["dim"], case["hidden"], case["layers"], size[case["type"]]
    n = L * 3 * H * D + (sum(7 * i + 1 + 3 * (D + 1) for i in range(L)) if case["ragged"] else 0)
    return {"bytes": 2 * (n * e + 4 * L * D) + 4, "flops": 3 * (n + L * D)}


# ------------------------------------------------- the definition in 64 bits
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exact_mx(q, tiled):
    """Decoded block by block from the layout's definition."""
    R, half = q.shape
    r = torch.arange(R, device=q.device)[:, None]
    b = torch.arange(half // 16, device=q.device)[None, :]
    byte = tiled[r // 128, b // 4, r % 32, (r % 128) // 32, b % 4].long()
    table = torch.tensor(_E2M1, dtype=torch.float64, device=q.device)
    out = torch.empty((R, 2 * half), dtype=torch.float64, device=q.device)
    for part, nibble in ((0, q.int() % 16), (1, q.int() // 16)):
        out[:, part::2] = torch.where(nibble >= 8, -1.0, 1.0) * table[(nibble % 8).long()]
    return out * ((byte + (1023 - 127)) << 52).view(torch.float64).repeat_interleave(32, dim=1)  # 2^(byte - 127) by its bits


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("norm", "norm_e4m3"):
        total = s["x"] if s["residual"] is None else (s["x"].double() + s["residual"].double()).to(s["x"].dtype)
        v = total.double()
        rms = (v.pow(2).sum(1) / case["cols"] + EPS).sqrt()
        y = (v / rms[:, None]) * s["weight"].double()
        if op == "norm":
            return y, total.double(), 1.0 / rms
        top = y.abs().max(1).values
        scale = torch.where(top == 0, 1.0, top / 448.0)
        return y / scale[:, None], scale, total.double(), 1.0 / rms
    if op == "norm_bwd":
        # d/dx of x_j w_j / sqrt(mean x^2 + eps), with the inverse root that the call is given.
        x, w, dy, r = s["x"].double(), s["weight"].double(), s["dy"].double(), s["rstd"].double()
        along = (dy * w * x).sum(1) * r.pow(3) / case["cols"]
        dx = dy * w * r[:, None] - x * along[:, None]
        dx = dx if s["ds"] is None else dx + s["ds"].double()
        return dx, torch.einsum("md,md,m->d", dy, x, r)
    if op == "mxfp4":
        v = s["x"].double().view(case["rows"], -1, 32)
        top = v.abs().max(-1, keepdim=True).values
        field = (top.view(torch.int64) >> 52) - 2                    # 1023 + floor(log2 amax) - 2
        unit = (field.clamp(min=1023 - 127) << 52).view(torch.float64)
        step = v.abs() / unit
        # Spacing 0.5 below 2, 1 below 4, 2 above; torch.round takes ties to even.
        near = torch.where(step < 2, torch.round(step * 2) / 2, torch.where(step < 4, torch.round(step), torch.round(step / 2) * 2))
        return (torch.sign(v) * near.clamp(max=6.0) * unit).view(case["rows"], case["cols"])
    if op == "product":
        return _exact_mx(s["a"], s["a_scale"]) @ _exact_mx(s["b"], s["b_scale"]).t()
    squared = 0.0
    for t in s["grads"]:
        squared = squared + torch.linalg.vector_norm(t.double()) ** 2
    norm = torch.sqrt(squared)
    factor = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0)
    return [norm] + [t.double() * factor for t in s["grads"]]
