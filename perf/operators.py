"""The 8-bit operators: what is measured, and their plain forms.

matmul_i8      C = a_scale * w_scale * (A @ W.T) + bias, A [M, K] and W [N, K] int8, one scale a token and a channel
rmsnorm_i8     root-mean-square norm of x (or of x + residual), quantised to int8 with one scale a row
silu_mul_i8    silu(gate) * up, quantised the same way
mlp_i8         the path that runs them in a row: add + norm, product, silu * up, product

Quantised outputs are returned as the values they stand for (code * scale, in 32 bits).
"""
import math
import os
import sys

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # One token through a 4096-wide projection: the smallest product of a decode step, latency.
        {"name": "matmul_decode_1x4096x4096", "op": "matmul", "M": 1, "N": 4096, "K": 4096, "out": "bf16", "bias": 0, "pad": 0},
        # A decode batch of 16 through the wide projection: a stream of weights.
        {"name": "matmul_decode_16x14336x4096", "op": "matmul", "M": 16, "N": 14336, "K": 4096, "out": "f16", "bias": 0, "pad": 0},
        # A short ragged prompt and sizes that no alignment holds for; logits in 32 bits, with a bias.
        {"name": "matmul_ragged_77x1000x777", "op": "matmul", "M": 77, "N": 1000, "K": 777, "out": "f32", "bias": 1, "pad": 0},
        # A prefill-sized square product, the largest: tensor rate.
        {"name": "matmul_prefill_8192x8192x8192", "op": "matmul", "M": 8192, "N": 8192, "K": 8192, "out": "bf16", "bias": 0, "pad": 0},
        # The norm before a block for one token: the smallest call of all.
        {"name": "norm_decode_1x4096", "op": "norm", "rows": 1, "cols": 4096, "dtype": "bf16", "residual": 1, "pad": 0},
        # Odd rows with padding between them, no residual (the first block of a model).
        {"name": "norm_ragged_333x1001", "op": "norm", "rows": 333, "cols": 1001, "dtype": "f16", "residual": 0, "pad": 7},
        # The norm of a prefill: memory bandwidth.
        {"name": "norm_prefill_8192x4096", "op": "norm", "rows": 8192, "cols": 4096, "dtype": "bf16", "residual": 1, "pad": 0},
        # The activation of a decode batch, gate and up being halves of one product's rows.
        {"name": "silu_decode_16x14336", "op": "silu", "rows": 16, "cols": 14336, "dtype": "bf16"},
        # The activation of a prefill: memory bandwidth.
        {"name": "silu_prefill_4096x14336", "op": "silu", "rows": 4096, "cols": 14336, "dtype": "f16"},
        # A whole block for one token: the latency of a chain of four kernels over 176 MB of weights.
        {"name": "mlp_decode_1x4096x14336", "op": "mlp", "M": 1, "K": 4096, "F": 14336, "dtype": "bf16"},
        # A small model's block for a few tokens, odd count.
        {"name": "mlp_batch_7x896x4864", "op": "mlp", "M": 7, "K": 896, "F": 4864, "dtype": "f16"},
        # A block of a prefill.
        {"name": "mlp_prefill_2048x4096x14336", "op": "mlp", "M": 2048, "K": 4096, "F": 14336, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size of [lo, hi], log-uniform: a multiple of 64 half of the time, any number otherwise."""
    n = _log(rng, lo, hi)
    return max(64, (n + 32) // 64 * 64) if rng.random() < 0.5 else n


def draw(rng):
    op = rng.choice(["matmul", "norm", "silu", "mlp"])
    while True:
        if op == "matmul":
            c = {"op": op, "M": _log(rng, 1, 8192), "N": _size(rng, 64, 28672), "K": _size(rng, 64, 16384),
                 "out": rng.choice(["bf16", "f16", "f32"]), "bias": rng.randrange(2), "pad": 0}
            if rng.random() < 0.5:  # rows padded to whole 16-byte pieces, as an allocator of weights would
                c["pad"] = -c["K"] % 16
            if 2 * c["M"] * c["N"] * c["K"] <= 2 * 8192**3 and c["M"] * c["N"] <= 1 << 26:
                return c
        elif op in ("norm", "silu"):
            c = {"op": op, "rows": _log(rng, 1, 8192), "cols": _size(rng, 64, 28672), "dtype": rng.choice(["bf16", "f16"])}
            if op == "norm":
                c["residual"], c["pad"] = rng.randrange(2), rng.choice([0, 0, 8, 3])
            if c["rows"] * c["cols"] <= 4096 * 14336:
                return c
        else:
            c = {"op": op, "M": _log(rng, 1, 2048), "K": _size(rng, 128, 8192), "F": _size(rng, 256, 14336),
                 "dtype": rng.choice(["bf16", "f16"])}
            if c["M"] * c["F"] * c["K"] <= 2048 * 4096 * 14336:
                return c


def _codes(g, rows, cols, pad=0):
    """int8 codes as a quantiser leaves them: normal, clipped to [-127, 127], rows `pad` bytes apart."""
    x = torch.randn(rows, cols, device="cuda", generator=g, dtype=torch.float16).mul_(34.0).round_().clamp_(-127, 127)
    q = torch.zeros(rows, cols + pad, device="cuda", dtype=torch.int8)
    q[:, :cols] = x
    return q[:, :cols]


def _stream(g, rows, cols, dtype, pad=0):
    """A residual stream: normal, with a few channels much larger than the rest."""
    x = torch.randn(rows, cols + pad, device="cuda", generator=g, dtype=torch.float32)
    x *= torch.where(torch.rand(cols + pad, device="cuda", generator=g) < 0.01, 12.0, 1.0)
    return x.to(dtype)[:, :cols]


def _weights(g, n, k):
    w = _codes(g, n, k)
    s = (torch.rand(n, device="cuda", generator=g) + 0.5) / (34.0 * math.sqrt(k))
    return w, s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    s = {"case": case}
    if op == "matmul":
        M, N, K = case["M"], case["N"], case["K"]
        s["a"] = _codes(g, M, K, case["pad"])
        s["w"] = _codes(g, N, K, case["pad"])
        s["a_scale"] = torch.rand(M, device="cuda", generator=g) * 0.05 + 0.01
        s["w_scale"] = (torch.rand(N, device="cuda", generator=g) + 0.5) / (34.0 * math.sqrt(K))
        s["bias"] = torch.randn(N, device="cuda", generator=g).to(_DT[case["out"]]) if case["bias"] else None
    elif op == "norm":
        rows, cols, dt = case["rows"], case["cols"], _DT[case["dtype"]]
        s["x"] = _stream(g, rows, cols, dt, case["pad"])
        s["residual"] = _stream(g, rows, cols, dt, case["pad"]) if case["residual"] else None
        if not case["residual"] and rows > 8:
            s["x"][rows // 2] = 0  # a padding token
        s["g"] = (torch.randn(cols, device="cuda", generator=g) * 0.2 + 1.0).to(dt)
        s["eps"] = 1e-5
    elif op == "silu":
        rows, cols, dt = case["rows"], case["cols"], _DT[case["dtype"]]
        gu = torch.randn(rows, 2 * cols, device="cuda", generator=g, dtype=torch.float32).mul_(1.5).to(dt)
        s["gate"], s["up"] = gu[:, :cols], gu[:, cols:]
    else:
        M, K, F, dt = case["M"], case["K"], case["F"], _DT[case["dtype"]]
        s["x"], s["residual"] = _stream(g, M, K, dt), _stream(g, M, K, dt)
        s["g"] = (torch.randn(K, device="cuda", generator=g) * 0.2 + 1.0).to(dt)
        s["eps"] = 1e-5
        s["w_gate_up"], s["s_gate_up"] = _weights(g, 2 * F, K)
        s["w_down"], s["s_down"] = _weights(g, K, F)
    return s


# ------------------------------------------------------------- plain forms
def _matmul(a, w, a_scale, w_scale, bias, dt):
    acc = a.float() @ w.float().t()
    acc = acc * a_scale[:, None] * w_scale[None, :]
    if bias is not None:
        acc = acc + bias.float()
    return acc.to(dt)


def _quantise(t):
    """Codes of the rows of t (64 bits: the quotient is rounded to whole numbers), and each row's largest magnitude."""
    m = t.abs().amax(dim=1, keepdim=True)
    q = torch.where(m > 0, torch.round(127.0 * t / m), torch.zeros_like(t))
    return q.to(torch.int8), m[:, 0]


def _norm(x, residual, g, eps):
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    hd = h.double()
    q, m = _quantise(hd * g.double())
    scale = (m / torch.sqrt(hd.square().mean(dim=1) + eps) / 127.0).float()
    return q, scale, h


def _silu_mul(gate, up):
    gd = gate.double()
    q, m = _quantise(gd / (1.0 + torch.exp(-gd)) * up.double())
    return q, (m / 127.0).float()


def _ops():
    """torch.ops.aegis with the operators registered."""
    if "aegis_torch" not in sys.modules:
        sys.path.insert(0, os.path.join(os.getcwd(), "aegis-core_b200"))
        import aegis_torch  # noqa: F401
    return torch.ops.aegis


def run(state):
    case = state["case"]
    op = case["op"]
    if op == "matmul":
        a, w, sa, sw, bias, dt = state["a"], state["w"], state["a_scale"], state["w_scale"], state["bias"], _DT[case["out"]]
        if own:
            return _ops().matmul_i8(a, w, sa, sw, bias, out_dtype=dt)
        return _matmul(a, w, sa, sw, bias, dt)
    if op == "norm":
        x, r, g, eps = state["x"], state["residual"], state["g"], state["eps"]
        if own:
            if r is None:
                q, scale = _ops().rmsnorm_i8(x, g, eps)
                h = x
            else:
                q, scale, h = _ops().add_rmsnorm_i8(x, r, g, eps)
        else:
            q, scale, h = _norm(x, r, g, eps)
        out = {"values": q * scale[:, None], "scale": scale}
        if r is not None:
            out["h"] = h
        return out
    if op == "silu":
        q, scale = _ops().silu_mul_i8(state["gate"], state["up"]) if own else _silu_mul(state["gate"], state["up"])
        return {"values": q * scale[:, None], "scale": scale}
    x, r, g, eps = state["x"], state["residual"], state["g"], state["eps"]
    if own:
        y, h = _ops().mlp_i8(x, r, g, eps, state["w_gate_up"], state["s_gate_up"], state["w_down"], state["s_down"])
        return {"y": y, "h": h}
    F = case["F"]
    q, scale, h = _norm(x, r, g, eps)
    gu = _matmul(q, state["w_gate_up"], scale, state["s_gate_up"], None, x.dtype)
    q, scale = _silu_mul(gu[:, :F], gu[:, F:])
    return {"y": _matmul(q, state["w_down"], scale, state["s_down"], None, x.dtype), "h": h}


def work(case):
    op = case["op"]
    if op == "matmul":
        M, N, K = case["M"], case["N"], case["K"]
        o = 4 if case["out"] == "f32" else 2
        return {"bytes": M * K + N * K + 4 * (M + N) + o * N * (M + case["bias"]), "flops": 2 * M * N * K}
    if op == "norm":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (3 + 4 * case["residual"]) + 2 * case["cols"] + 4 * case["rows"], "flops": 8 * n}
    if op == "silu":
        n = case["rows"] * case["cols"]
        return {"bytes": 5 * n + 4 * case["rows"], "flops": 8 * n}
    M, K, F = case["M"], case["K"], case["F"]
    return {"bytes": 3 * F * K + 8 * M * K + 2 * K + 4 * (2 * F + K), "flops": 6 * M * F * K}


# ------------------------------------------------------------- 64 bits, from the definitions
def _product64(q, w, s_row, s_col, bias=None):
    y = torch.einsum("mk,nk->mn", q.to(torch.float64), w.to(torch.float64))  # whole numbers below 2^53: exact
    y.mul_(s_row.to(torch.float64).unsqueeze(1)).mul_(s_col.to(torch.float64).unsqueeze(0))
    return y if bias is None else y.add_(bias.to(torch.float64))


def _codes64(v):
    """(codes, largest magnitude of each row) of 64-bit rows: the nearest whole number to 127 v / max|v|, ties to even."""
    top = torch.linalg.vector_norm(v, ord=math.inf, dim=-1)
    r = v * 127.0 / torch.where(top == 0, 1.0, top).unsqueeze(-1)
    return r.round(), top


def _norm64(x, residual, g, eps):
    h = x.to(torch.float64)
    if residual is not None:
        h = h.add(residual.to(torch.float64)).to(x.dtype).to(torch.float64)  # the stream is kept in its own type
    codes, top = _codes64(h * g.to(torch.float64).unsqueeze(0))
    rms = (torch.einsum("rc,rc->r", h, h) / h.shape[1] + eps).sqrt()
    return codes, top / (127.0 * rms), h


def _silu_mul64(gate, up):
    codes, top = _codes64(torch.sigmoid(gate.to(torch.float64)) * gate.to(torch.float64) * up.to(torch.float64))
    return codes, top / 127.0


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "matmul":
        return _product64(s["a"], s["w"], s["a_scale"], s["w_scale"], s["bias"])
    if op == "norm":
        codes, scale, h = _norm64(s["x"], s["residual"], s["g"], s["eps"])
        out = {"values": codes * scale.unsqueeze(1), "scale": scale}
        if s["residual"] is not None:
            out["h"] = h
        return out
    if op == "silu":
        codes, scale = _silu_mul64(s["gate"], s["up"])
        return {"values": codes * scale.unsqueeze(1), "scale": scale}
    codes, scale, h = _norm64(s["x"], s["residual"], s["g"], s["eps"])
    gu = _product64(codes, s["w_gate_up"], scale, s["s_gate_up"]).to(s["x"].dtype)  # the product's own output type
    codes, scale = _silu_mul64(gu[:, :case["F"]], gu[:, case["F"]:])
    return {"y": _product64(codes, s["w_down"], scale, s["s_down"]), "h": h}
