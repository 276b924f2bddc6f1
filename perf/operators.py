"""Performance cases of the 8-bit layer operators: what runs around the quantized attention in a W8A8 model.

Four operators, each through its public entry point:

  rows    ``quantize_rows``: a tensor's rows as int8 codes with one scale each (a projection's input, a weight)
  norm    ``rms_norm_quant``: the residual's addition, the RMS norm and the quantization of its rows
  silu    ``silu_mul_quant``: the SwiGLU product and the quantization of its rows
  linear  ``int8_linear``: int8 matrix product with a scale for each token and each output channel

Codes are returned as the values they stand for (code times scale, bf16).  Sizes are those of the models this
repository ships maps for (hidden 3584 / intermediate 18944, hidden 4096 / intermediate 14336), token counts from
one generated token to a long prompt, and odd ones.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6
TINY = 2.0 ** -118     # rows of smaller values are quantized on this one's scale
MOST_FLOPS = 2.0 * 8192 * 37888 * 3584
MOST_BYTES = 5.0 * 8192 * 18944


def listed():
    return [
        # a generated token's fused Q/K/V projection, Qwen2-7B width
        dict(name="linear_1_qkv", op="linear", m=1, n=4608, k=3584, bias=True, residual=False, dtype="bf16"),
        # a small batch's down projection with the residual's addition: the longest sums
        dict(name="linear_8_down", op="linear", m=8, n=3584, k=18944, bias=False, residual=True, dtype="bf16"),
        # one token's logits in fp32 over a large vocabulary: a stream of weights
        dict(name="linear_1_vocab", op="linear", m=1, n=152064, k=3584, bias=False, residual=False, dtype="f32"),
        # a short question at odd sizes, fp16
        dict(name="linear_77_odd", op="linear", m=77, n=5001, k=2049, bias=True, residual=False, dtype="f16"),
        # a chunk of prompt through an output projection with the residual's addition, hidden 4096
        dict(name="linear_500_out", op="linear", m=500, n=4096, k=4096, bias=False, residual=True, dtype="bf16"),
        # a long prompt's fused gate and up projections, Qwen2-7B width
        dict(name="linear_8k_gate_up", op="linear", m=8192, n=37888, k=3584, bias=False, residual=False, dtype="bf16"),
        # a generated token's norm: latency alone
        dict(name="norm_1", op="norm", m=1, k=3584, residual=True, dtype="bf16"),
        # a long prompt's norm, odd token count, hidden 4096
        dict(name="norm_8191", op="norm", m=8191, k=4096, residual=True, dtype="bf16"),
        # a small batch's SwiGLU
        dict(name="silu_8", op="silu", m=8, k=18944, dtype="bf16"),
        # a long prompt's SwiGLU
        dict(name="silu_8k", op="silu", m=8192, k=18944, dtype="bf16"),
        # a small batch's attention output before the output projection, fp16
        dict(name="rows_33", op="rows", m=33, k=3584, dtype="f16"),
        # a layer's gate weight on its way to int8
        dict(name="rows_weight", op="rows", m=18944, k=3584, dtype="bf16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("linear", "linear", "linear", "norm", "silu", "rows"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    while True:
        m = _log(rng, 1, 8192)
        if op == "linear":
            case = dict(op=op, m=m, n=_log(rng, 16, 40000), k=_log(rng, 64, 19000), bias=rng.random() < 0.5,
                        residual=rng.random() < 0.5, dtype=dtype)
            if rng.random() < 0.5:  # (widths are mostly multiples of 128)
                case["n"], case["k"] = -(-case["n"] // 128) * 128, -(-case["k"] // 128) * 128
        else:
            case = dict(op=op, m=m, k=_log(rng, 64, 19000), dtype=dtype)
            if rng.random() < 0.5:
                case["k"] = -(-case["k"] // 128) * 128
            if op == "norm":
                case["residual"] = rng.random() < 0.7
        w = work(case)
        if w["flops"] <= MOST_FLOPS and w["bytes"] <= MOST_BYTES:
            return case


def work(case):
    m, k = case["m"], case["k"]
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "linear":
        n = case["n"]
        outs = 2 if case["residual"] else 1
        return {"bytes": m * k + n * k + 4 * m + 4 * n + outs * m * n * size + (n * size if case["bias"] else 0),
                "flops": 2 * m * n * k}
    reads = {"rows": 1, "silu": 2, "norm": 2 if case.get("residual") else 1}[case["op"]]
    hidden = m * k * size if case.get("residual") else 0
    weight = k * size if case["op"] == "norm" else 0
    ops = {"rows": 3, "silu": 8, "norm": 6}[case["op"]]
    return {"bytes": reads * m * k * size + weight + hidden + m * k + 4 * m, "flops": ops * m * k}


def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _activations(g, m, k, dtype):
    """Hidden states: tokens of different magnitudes, a few channels far above the rest."""
    x = torch.randn(m, k, generator=g, device=DEV)
    x *= torch.exp(0.5 * torch.randn(m, 1, generator=g, device=DEV))
    loud = torch.rand(k, generator=g, device=DEV) < 4 / k
    x *= 1 + 19 * loud
    return x.to(dtype)


def _codes(g, rows, k):
    """int8 codes as a symmetric quantizer leaves them, rows at a stride of a multiple of 16 bytes."""
    x = torch.empty(rows, -(-k // 16) * 16, dtype=torch.int8, device=DEV)[:, :k]
    x.copy_((torch.randn(rows, k, generator=g, device=DEV) * 32).round_().clamp_(-127, 127))
    return x


def prepare(case, seed):
    g = _generator(seed)
    m, k, dtype = case["m"], case["k"], TYPES[case["dtype"]]
    state = dict(op=case["op"], dtype=dtype)
    if case["op"] == "linear":
        n = case["n"]
        state["x"], state["w"] = _codes(g, m, k), _codes(g, n, k)
        state["xs"] = 0.02 * torch.exp(0.5 * torch.randn(m, generator=g, device=DEV))
        state["ws"] = (0.5 + torch.rand(n, generator=g, device=DEV)) * (0.02 / math.sqrt(k))
        state["bias"] = torch.randn(n, generator=g, device=DEV).to(dtype) if case["bias"] else None
        state["residual"] = _activations(g, m, n, dtype) if case["residual"] else None
    elif case["op"] == "silu":
        both = _activations(g, m, 2 * k, dtype)  # (the fused gate and up projections' output)
        state["gate"], state["up"] = both[:, :k], both[:, k:]
    else:
        state["x"] = _activations(g, m, k, dtype)
        if case["op"] == "norm":
            state["w"] = (1 + 0.3 * torch.randn(k, generator=g, device=DEV)).to(dtype)
            state["residual"] = _activations(g, m, k, dtype) if case["residual"] else None
    return state


def _values(codes, scales):
    out = torch.empty(codes.shape, dtype=torch.bfloat16, device=codes.device)
    return torch.mul(codes, scales.unsqueeze(-1), out=out)


def _quantize(y):
    top = y.abs().amax(-1).clamp(min=TINY)
    return (y * (127 / top).unsqueeze(-1)).round(), top / 127


def _plain(s):
    if s["op"] == "linear":
        y = (s["x"].float() @ s["w"].float().t()) * (s["xs"].unsqueeze(-1) * s["ws"])
        if s["bias"] is not None:
            y = y + s["bias"].float()
        if s["residual"] is not None:
            y = y + s["residual"].float()
        return y.to(s["dtype"])
    if s["op"] == "silu":
        g = s["gate"].float()
        codes, scales = _quantize(g / (1 + torch.exp(-g)) * s["up"].float())
        return _values(codes, scales), scales
    if s["op"] == "rows":
        codes, scales = _quantize(s["x"].float())
        return _values(codes, scales), scales
    h = s["x"]
    if s["residual"] is not None:
        h = (h.float() + s["residual"].float()).to(s["dtype"])
    y = h.float()
    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * s["w"].float()
    codes, scales = _quantize(y)
    out = (_values(codes, scales), scales)
    return out if s["residual"] is None else out + (h,)


def run(state):
    if not own:
        return _plain(state)
    from triattention_amd.kernels import linear

    s = state
    if s["op"] == "linear":
        return linear.int8_linear(s["x"], s["xs"], s["w"], s["ws"], bias=s["bias"], residual=s["residual"],
                                  out_dtype=s["dtype"])
    if s["op"] == "silu":
        codes, scales = linear.silu_mul_quant(s["gate"], s["up"])
        return _values(codes, scales), scales
    if s["op"] == "rows":
        codes, scales = linear.quantize_rows(s["x"])
        return _values(codes, scales), scales
    codes, scales, h = linear.rms_norm_quant(s["x"], s["w"], EPS, residual=s["residual"])
    out = (_values(codes, scales), scales)
    return out if s["residual"] is None else out + (h,)


def _exact_codes(y):
    top = torch.linalg.vector_norm(y, ord=math.inf, dim=-1, keepdim=True).clamp(min=TINY)
    scale = top / 127
    return torch.round(127 * y / top) * scale, scale.squeeze(-1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        y = torch.einsum("mk,nk->mn", s["x"].double() * s["xs"].double()[:, None],
                         s["w"].double() * s["ws"].double()[:, None])
        for extra in (s["bias"], s["residual"]):
            if extra is not None:
                y += extra.double()
        return y
    if case["op"] == "silu":
        g, u = s["gate"].double(), s["up"].double()
        return _exact_codes(g * torch.sigmoid(g) * u)
    if case["op"] == "rows":
        return _exact_codes(s["x"].double())
    h = s["x"].double()
    if s["residual"] is not None:
        h = (h + s["residual"].double()).to(s["dtype"]).double()  # (the norm reads the rounded hidden state)
    y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + EPS) * s["w"].double()
    return _exact_codes(y) if s["residual"] is None else _exact_codes(y) + (h,)
