"""Cases and plain forms of the 8-bit operators (``triton_client_amd.ops.int8``).

Four operators, each in the range a language-model server meets, from one token to a long prefill:

``norm``      root-mean-square norm with the residual's addition, output in 8 bits with a scale per token
``quantize``  rows to 8 bits and back
``gate``      SiLU-gated product of an MLP's two halves, output in 8 bits with a scale per token
``product``   matrix product in 8-bit integers with a scale per token and per output channel

8-bit outputs are returned as the values they stand for (scale times integer), in the type of the activations.
"""

import math

import torch

own = False

_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # one token of a decode step enters a block: latency of one small launch
        {"name": "norm token", "op": "norm", "rows": 1, "width": 4096, "dtype": "fp16", "residual": True},
        # a ragged batch of prompts at a width that is no power of two
        {"name": "norm ragged", "op": "norm", "rows": 777, "width": 5000, "dtype": "bf16", "residual": True},
        # a long prefill: memory bandwidth
        {"name": "norm prefill", "op": "norm", "rows": 16384, "width": 8192, "dtype": "bf16", "residual": True},
        # fp32 master weights of an odd layer, quantised when a model is loaded
        {"name": "quantize odd", "op": "quantize", "rows": 1021, "width": 4095, "dtype": "fp32"},
        # activations of a large batch
        {"name": "quantize large", "op": "quantize", "rows": 8192, "width": 16384, "dtype": "bf16"},
        # MLP activation of a few decoded tokens
        {"name": "gate few", "op": "gate", "rows": 8, "width": 8192, "dtype": "fp16"},
        # MLP activation of a prefill
        {"name": "gate prefill", "op": "gate", "rows": 4096, "width": 16384, "dtype": "bf16"},
        # one decoded token through a square projection: the weights' bytes count
        {"name": "product token", "op": "product", "m": 1, "n": 4096, "k": 4096, "dtype": "fp16", "bias": False,
         "residual": False},
        # sixteen concurrent requests through an MLP's widening projection
        {"name": "product few", "op": "product", "m": 16, "n": 16384, "k": 4096, "dtype": "bf16", "bias": False,
         "residual": False},
        # a classifier's head (2048 features, 1000 classes) over an odd number of rows, logits in fp32
        {"name": "product head", "op": "product", "m": 300, "n": 1000, "k": 2048, "dtype": "fp32", "bias": True,
         "residual": False},
        # no dimension a multiple of anything: a ragged prefill of a pruned layer
        {"name": "product odd", "op": "product", "m": 1999, "n": 2999, "k": 4001, "dtype": "fp16", "bias": True,
         "residual": False},
        # a large prefill: arithmetic counts
        {"name": "product prefill", "op": "product", "m": 8192, "n": 8192, "k": 8192, "dtype": "bf16", "bias": False,
         "residual": True},
    ]


def _log_between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _size(rng, low, high):
    """A size of [low, high]: half of them multiples of 64, where the range has them."""
    n = _log_between(rng, low, high)
    return min(high, max(64, n // 64 * 64)) if rng.random() < 0.5 and high >= 64 else n


def draw(rng):
    op = rng.choice(["norm", "quantize", "gate", "product", "product"])
    if op == "product":
        while True:
            m, n, k = _log_between(rng, 1, 8192), _size(rng, 16, 16384), _size(rng, 16, 16384)
            if m * n * k <= 8192 ** 3:
                break
        return {"op": op, "m": m, "n": n, "k": k, "dtype": rng.choice(["fp16", "bf16", "fp32"]),
                "bias": rng.random() < 0.5, "residual": rng.random() < 0.5}
    while True:
        rows, width = _log_between(rng, 1, 16384), _size(rng, 64, 16384)
        if rows * width <= (1 << 26):
            break
    case = {"op": op, "rows": rows, "width": width,
            "dtype": rng.choice(["fp16", "bf16", "fp32"] if op == "quantize" else ["fp16", "bf16"])}
    if op == "norm":
        case["residual"] = rng.random() < 0.75
    return case


def _activations(g, rows, width, dtype, spread=1.0):
    """What a network's residual stream looks like: normal values, tokens of different size, a few loud channels."""
    dev = "cuda"
    x = torch.randn(rows, width, generator=g, device=dev)
    token = torch.exp(0.5 * torch.randn(rows, 1, generator=g, device=dev))
    channel = torch.where(torch.rand(width, generator=g, device=dev) < 0.004, 8.0, 1.0)
    return (x * token * channel * spread).to(dtype)


def _int8(g, rows, width):
    return torch.randn(rows, width, generator=g, device="cuda").mul_(32).round_().clamp_(-127, 127).to(torch.int8)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = _TYPES[case["dtype"]]
    state = {"op": case["op"], "dtype": dtype}
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        state["x"], state["w"] = _int8(g, m, k), _int8(g, n, k)
        state["x_scale"] = torch.exp(0.5 * torch.randn(m, generator=g, device="cuda")) * 0.03
        state["w_scale"] = torch.exp(0.3 * torch.randn(n, generator=g, device="cuda")) * 0.001
        state["bias"] = torch.randn(n, generator=g, device="cuda").to(dtype) if case["bias"] else None
        state["residual"] = _activations(g, m, n, dtype) if case["residual"] else None
        return state
    rows, width = case["rows"], case["width"]
    if case["op"] == "norm":
        state["x"] = _activations(g, rows, width, dtype)
        state["residual"] = _activations(g, rows, width, dtype, 3.0) if case["residual"] else None
        state["weight"] = (1 + 0.2 * torch.randn(width, generator=g, device="cuda")).to(dtype)
        state["eps"] = 1e-6
    elif case["op"] == "quantize":
        state["x"] = _activations(g, rows, width, dtype)
    else:
        state["x"] = _activations(g, rows, 2 * width, dtype)
    return state


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    from triton_client_amd.ops import int8

    if s["op"] == "product":
        return int8.linear_int8(s["x"], s["x_scale"], s["w"], s["w_scale"], bias=s["bias"], residual=s["residual"],
                                dtype=s["dtype"])
    if s["op"] == "norm" and s["residual"] is not None:
        q, scale, summed = int8.rms_norm_int8(s["x"], s["weight"], residual=s["residual"], eps=s["eps"])
        return int8.dequantize_int8(q, scale, dtype=s["dtype"]), scale, summed
    if s["op"] == "norm":
        q, scale = int8.rms_norm_int8(s["x"], s["weight"], eps=s["eps"])
    elif s["op"] == "quantize":
        q, scale = int8.quantize_int8(s["x"])
    else:
        q, scale = int8.silu_mul_int8(s["x"])
    return int8.dequantize_int8(q, scale, dtype=s["dtype"]), scale


def _to_8_bits(p, factor=None):
    """Integers nearest to 127 p / max|p| of each row (the quotient in 64 bits: it decides borders), and the scales."""
    top = p.abs().amax(dim=-1, keepdim=True)
    q = torch.round(p.double() * 127 / top.double()).float()
    scale = (top if factor is None else top * factor) / 127
    return torch.where(top > 0, q, 0.0), scale


def _run_plain(s):
    dtype = s["dtype"]
    if s["op"] == "product":
        y = s["x"].float() @ s["w"].float().t()
        y = y * (s["x_scale"][:, None] * s["w_scale"])
        if s["bias"] is not None:
            y = y + s["bias"].float()
        if s["residual"] is not None:
            y = y + s["residual"].float()
        return y.to(dtype)
    if s["op"] == "norm":
        h = s["x"]
        if s["residual"] is not None:
            h = (h.float() + s["residual"].float()).to(dtype)
        f = h.float()
        q, scale = _to_8_bits(f * s["weight"].float(), torch.rsqrt(f.square().mean(dim=-1, keepdim=True) + s["eps"]))
        values = (q * scale).to(dtype)
        return (values, scale[:, 0]) if s["residual"] is None else (values, scale[:, 0], h)
    if s["op"] == "quantize":
        p = s["x"].float()
    else:
        gate, up = s["x"].float().chunk(2, dim=-1)
        p = gate / (1 + torch.exp(-gate)) * up
    q, scale = _to_8_bits(p)
    return (q * scale).to(dtype), scale[:, 0]


def work(case):
    e = {"fp16": 2, "bf16": 2, "fp32": 4}[case["dtype"]]
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        more = n * e * case["bias"] + m * n * e * case["residual"]
        return {"bytes": m * k + n * k + 4 * (m + n) + more + m * n * e, "flops": 2 * m * n * k}
    # inputs read once, outputs (the values, the scales, the sum) written once; the integers in between are not counted
    rows, width = case["rows"], case["width"]
    n = rows * width
    if case["op"] == "norm":
        return {"bytes": n * e * (3 if case["residual"] else 1) + width * e + n * e + 4 * rows, "flops": 8 * n}
    if case["op"] == "quantize":
        return {"bytes": 2 * n * e + 4 * rows, "flops": 4 * n}
    return {"bytes": 3 * n * e + 4 * rows, "flops": 10 * n}


def exact(case, seed):
    """From the definitions, in 64 bits: each row's largest magnitude stands for 127, every value is the nearest of
    the 255 levels.  The sum with the residual is held in the activations' type, which is part of the definition."""
    s = prepare(case, seed)
    dtype = s["dtype"]
    if case["op"] == "product":
        x, w = s["x"].to(torch.float64), s["w"].to(torch.float64)
        out = torch.matmul(x, w.transpose(0, 1))
        out *= s["x_scale"].to(torch.float64).unsqueeze(1)
        out *= s["w_scale"].to(torch.float64).unsqueeze(0)
        for more in (s["bias"], s["residual"]):
            if more is not None:
                out += more.to(torch.float64)
        return out
    x = s["x"].to(torch.float64)
    summed = None
    if case["op"] == "norm":
        if s["residual"] is not None:
            summed = (x + s["residual"].to(torch.float64)).to(dtype).to(torch.float64)
            x = summed
        y = x / torch.sqrt(torch.sum(x * x, dim=1, keepdim=True) / case["width"] + s["eps"])
        y = y * s["weight"].to(torch.float64)
    elif case["op"] == "quantize":
        y = x
    else:
        width = case["width"]
        y = x[:, :width] * torch.sigmoid(x[:, :width]) * x[:, width:]
    step = torch.max(torch.abs(y), dim=1)[0] / 127
    levels = torch.round(y / torch.where(step > 0, step, 1.0).unsqueeze(1))
    values = levels * step.unsqueeze(1)
    return (values, step) if summed is None else (values, step, summed)
