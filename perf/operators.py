"""Workloads of the 8-bit operators: the quantising row operators and the int8 product that
reads what they write, in the order in which a quantised linear layer or gated MLP uses them.

Each case is one pass through one operator as a program calls it. `run` has two forms on the
same inputs: the plain one, elementary torch operations in 32 bits rounded once at the end,
and (with `own` set) the calls of ridge_b200. What an operator holds in 8 bits is returned as
the values it stands for, in a 16-bit type, beside its scales.
"""

import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}
EPS = 1e-6


def listed():
    return [
        # the norm in front of a layer while one sequence decodes: latency only
        {"name": "norm_1x4096", "op": "norm", "rows": 1, "cols": 4096, "type": "f16",
         "residual": True},
        # the same norm over a long prompt, or a large batch of them
        {"name": "norm_8192x8192", "op": "norm", "rows": 8192, "cols": 8192, "type": "bf16",
         "residual": True},
        # a first norm (nothing to add yet) of a 32-bit stream, rows of an odd length
        {"name": "norm_333x5003", "op": "norm", "rows": 333, "cols": 5003, "type": "f32",
         "residual": False},
        # the gated activation of a small decode batch
        {"name": "silu_16x11008", "op": "silu", "rows": 16, "cols": 11008, "type": "bf16"},
        # the gated activation of a prompt
        {"name": "silu_4096x14336", "op": "silu", "rows": 4096, "cols": 14336, "type": "f16"},
        # a weight matrix quantised by output channel when a model is loaded
        {"name": "quantize_14336x4096", "op": "quantize", "rows": 14336, "cols": 4096,
         "type": "bf16"},
        # activations of a short ragged batch, quantised by token
        {"name": "quantize_77x1000", "op": "quantize", "rows": 77, "cols": 1000, "type": "f32"},
        # one token through a linear layer: the weights are read once, nothing else counts
        {"name": "gemm_1x8192x8192", "op": "gemm", "m": 1, "n": 8192, "k": 8192, "type": "f16",
         "bias": False},
        # a decode batch through the same layer
        {"name": "gemm_128x8192x8192", "op": "gemm", "m": 128, "n": 8192, "k": 8192,
         "type": "bf16", "bias": False},
        # a short prompt into an odd number of classes, 32-bit scores with a bias
        {"name": "gemm_517x1003x2600", "op": "gemm", "m": 517, "n": 1003, "k": 2600,
         "type": "f32", "bias": True},
        # a prompt through the wide layer of an MLP
        {"name": "gemm_2048x14336x4096", "op": "gemm", "m": 2048, "n": 14336, "k": 4096,
         "type": "bf16", "bias": False},
        # a large prefill batch, or calibration of a whole layer
        {"name": "gemm_8192x8192x8192", "op": "gemm", "m": 8192, "n": 8192, "k": 8192,
         "type": "f16", "bias": True},
    ]


def _size(rng, low, high):
    """A size spread over the logarithm of its range; two of three are whole multiples of 8."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.67 and n >= 8:
        n = n // 8 * 8
    return max(low, min(high, n))


def draw(rng):
    op = rng.choice(["norm", "silu", "quantize", "gemm", "gemm"])
    kind = rng.choice(["f16", "bf16", "bf16", "f32"])
    if op == "gemm":
        while True:
            m, n, k = _size(rng, 1, 8192), _size(rng, 16, 16384), _size(rng, 16, 16384)
            if m * n * k <= 8192 ** 3:
                return {"op": op, "m": m, "n": n, "k": k, "type": kind,
                        "bias": rng.random() < 0.5}
    while True:
        rows, cols = _size(rng, 1, 16384), _size(rng, 16, 16384)
        if rows * cols <= 1 << 26:
            break
    case = {"op": op, "rows": rows, "cols": cols, "type": kind}
    if op == "norm":
        case["residual"] = rng.random() < 0.7
    return case


def _activations(rows, cols, g):
    """Hidden states: normal values, a few channels several times larger, and rows of different
    size; in a batch of some rows the last one is padding (zeros)."""
    x = torch.randn(rows, cols, device="cuda", generator=g)
    x *= torch.exp(0.3 * torch.randn(rows, 1, device="cuda", generator=g))
    loud = torch.rand(cols, device="cuda", generator=g) < 0.01
    x *= torch.where(loud, 4.0, 1.0)
    if rows > 8:
        x[-1] = 0
    return x


def _int8(x):
    """Rows in 8 bits with their scales; the rows' pitch is a multiple of 16 bytes, as a product
    with any row length wants it."""
    rows, cols = x.shape
    scale = x.abs().amax(1) / 127
    q = torch.zeros(rows, (cols + 15) // 16 * 16, dtype=torch.int8, device="cuda")[:, :cols]
    q.copy_(torch.round(x / scale.clamp_min(1e-30)[:, None]))
    return q, scale


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    kind = TYPES[case["type"]]
    if case["op"] == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        a, a_scale = _int8(_activations(m, k, g))
        b, b_scale = _int8(torch.randn(n, k, device="cuda", generator=g) / math.sqrt(k))
        bias = torch.randn(n, device="cuda", generator=g).to(kind) if case["bias"] else None
        return {"op": "gemm", "a": a, "a_scale": a_scale, "b": b, "b_scale": b_scale,
                "bias": bias, "kind": kind}
    rows, cols = case["rows"], case["cols"]
    s = {"op": case["op"], "x": _activations(rows, cols, g).to(kind),
         "value": torch.float16 if kind == torch.float32 else kind}
    if case["op"] == "norm":
        s["weight"] = (1 + 0.2 * torch.randn(cols, device="cuda", generator=g)).to(kind)
        s["residual"] = (2 * _activations(rows, cols, g)).to(kind) if case["residual"] else None
    if case["op"] == "silu":
        s["up"] = _activations(rows, cols, g).to(kind)
    return s


def _rows_to_int8(y):
    """The rows of y on a grid of 255 steps: (whole steps, step). A row of zeros has step 0."""
    scale = y.abs().amax(1, keepdim=True) / 127
    q = torch.round(y / scale.masked_fill(scale == 0, 1)).clamp(-127, 127)
    return q, scale


def _plain(s):
    op = s["op"]
    if op == "gemm":
        c = s["a"].float() @ s["b"].float().t()
        c = c * s["b_scale"] * s["a_scale"][:, None]
        if s["bias"] is not None:
            c = c + s["bias"].float()
        return {"out": c.to(s["kind"])}
    total = None
    if op == "norm":
        h = s["x"].float()
        if s["residual"] is not None:
            h = h + s["residual"].float()
            total = h.to(s["x"].dtype)
        y = h * torch.rsqrt(h.square().mean(1, keepdim=True) + EPS) * s["weight"].float()
    elif op == "silu":
        gate = s["x"].float()
        y = gate / (1 + torch.exp(-gate)) * s["up"].float()
    else:
        y = s["x"].float()
    q, scale = _rows_to_int8(y)
    out = {"values": (q * scale).to(s["value"]), "scale": scale[:, 0]}
    if total is not None:
        out["sum"] = total
    return out


def _own(s):
    import ridge_b200 as rb
    op = s["op"]
    if op == "gemm":
        return {"out": rb.gemm_i8(s["a"], s["a_scale"], s["b"], s["b_scale"], bias=s["bias"],
                                  dtype=s["kind"])}
    total = None
    if op == "norm":
        q, scale, total = rb.rms_norm_i8(s["x"], s["weight"], residual=s["residual"], eps=EPS)
    elif op == "silu":
        q, scale = rb.silu_mul_i8(s["x"], s["up"])
    else:
        q, scale = rb.quantize_i8(s["x"])
    out = {"values": rb.dequantize_i8(q, scale, dtype=s["value"]), "scale": scale}
    if total is not None:
        out["sum"] = total
    return out


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    size = SIZE[case["type"]]
    if case["op"] == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + n * k + 4 * (m + n) + size * m * n
                + (size * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    rows, cols = case["rows"], case["cols"]
    read = {"norm": 1, "silu": 2, "quantize": 1}[case["op"]]
    wrote = 0
    extra = 4 * rows
    if case["op"] == "norm":
        extra += size * cols
        if case["residual"]:
            read, wrote = 2, 1
    per = {"norm": 8, "silu": 10, "quantize": 4}[case["op"]]
    return {"bytes": rows * cols * (size * (read + wrote) + 2) + extra,
            "flops": per * rows * cols}


def exact(case, seed):
    """The operators' definitions in 64 bits.

    product:   out[i, j] = a_scale[i] b_scale[j] sum_k a[i, k] b[j, k] + bias[j]
    norm:      y = w (x + r) / sqrt(mean((x + r)^2) + eps)
    gate:      y = up gate / (1 + e^-gate)
    8 bits:    scale = max |y| / 127 over a row; value = scale * (y / scale to the nearest whole
               number, ties to even)
    """
    s = prepare(case, seed)
    d = torch.float64
    if case["op"] == "gemm":
        out = torch.matmul(s["a"].to(d), s["b"].to(d).mT)
        out.mul_(torch.outer(s["a_scale"].to(d), s["b_scale"].to(d)))
        if s["bias"] is not None:
            out += s["bias"].to(d)
        return {"out": out}
    x = s["x"].to(d)
    more = {}
    if case["op"] == "norm":
        if s["residual"] is not None:
            x = x + s["residual"].to(d)
            more["sum"] = x
        x = x / torch.sqrt((x * x).mean(dim=1) + EPS).unsqueeze(1) * s["weight"].to(d)
    elif case["op"] == "silu":
        x = x * torch.sigmoid(x) * s["up"].to(d)
    top = torch.amax(torch.abs(x), dim=1)
    step = (top / 127).unsqueeze(1)
    values = torch.where(step > 0, torch.round(x / step), torch.zeros_like(x)) * step
    return {"values": values, "scale": step.squeeze(1), **more}
