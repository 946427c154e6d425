"""The 8-bit products of a transformer block, as cases to measure: tokens and weights in 8-bit
integers with a scale for each row, the operators that bring tokens into that form (the residual's
addition with the root-mean-square norm, SiLU(gate) * up, and rows as they are), and the matrix product
of the two with the scales applied.

A row v is held as codes and a scale:

    a     = max |v|
    scale = a / 127                        (fp32; 0 where a < 2**-100)
    code  = round(v * 127 / a)             (to even, -127 .. 127)

and stands for ``scale * code``.  The product of tokens x [rows, k] and weights w [channels, k] is

    y[t][r] = x_scale[t] * w_scale[r] * sum_k x_code[t][k] * w_code[r][k] + bias[r]
"""

import math

import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}
LEAST = 2.0 ** -100


# --------------------------------------------------------------------------------------------
# Cases
# --------------------------------------------------------------------------------------------
def listed():
    return [
        # One sequence's next token between two projections: the whole call is latency.
        {"name": "norm_one", "op": "norm", "rows": 1, "n": 4096, "type": "fp32", "added": "fp16", "weight": "fp16"},
        # A step of a busy server on a wide model, the residual stream in 16 bits.
        {"name": "norm_96", "op": "norm", "rows": 96, "n": 8192, "type": "bf16", "added": "bf16", "weight": "bf16"},
        # Prompts of odd lengths together, the residual stream in 32 bits: memory bound.
        {"name": "norm_prompts", "op": "norm", "rows": 8191, "n": 4096, "type": "fp32", "added": "fp16",
         "weight": "fp16"},
        # A step's gated activations before the down projection.
        {"name": "silu_64", "op": "silu", "rows": 64, "n": 14336, "type": "bf16"},
        # The same for whole prompts.
        {"name": "silu_prompts", "op": "silu", "rows": 4097, "n": 14336, "type": "fp16"},
        # What attention gives for a chunk of a prompt, before the output projection.
        {"name": "quant_chunk", "op": "quant", "rows": 512, "n": 4096, "type": "fp16"},
        # A layer's weights brought into 8 bits while a model loads.
        {"name": "quant_weights", "op": "quant", "rows": 28672, "n": 4096, "type": "fp16"},
        # One token through the gate and up projections: as fast as the weights can be read.
        {"name": "linear_one", "op": "linear", "rows": 1, "k": 4096, "channels": 28672, "type": "fp16", "bias": False},
        # A step of a few sequences through the down projection.
        {"name": "linear_24", "op": "linear", "rows": 24, "k": 14336, "channels": 4096, "type": "bf16", "bias": False},
        # One chunk of a prompt through the q, k and v projections.
        {"name": "linear_chunk", "op": "linear", "rows": 512, "k": 4096, "channels": 6144, "type": "fp16",
         "bias": True},
        # Odd sizes all around, results in 32 bits.
        {"name": "linear_odd", "op": "linear", "rows": 333, "k": 1000, "channels": 1011, "type": "fp32", "bias": True},
        # Whole prompts through the gate and up projections: compute bound.
        {"name": "linear_prompts", "op": "linear", "rows": 8191, "k": 4096, "channels": 28672, "type": "fp16",
         "bias": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["norm", "silu", "quant", "linear", "linear", "linear"])
    if op == "linear":
        k, channels = _log_int(rng, 64, 16384), _log_int(rng, 64, 32768)
        if rng.random() < 0.6:  # most layers are whole multiples of something
            k, channels = max(64, k // 64 * 64), max(64, channels // 128 * 128)
        rows = _log_int(rng, 1, min(8191, max(1, 8191 * 4096 * 28672 // (k * channels))))
        return {"op": op, "rows": rows, "k": k, "channels": channels, "type": rng.choice(["fp16", "bf16", "fp16", "fp32"]),
                "bias": rng.random() < 0.4}
    n = _log_int(rng, 64, 28672 if op == "silu" else 16384)
    if rng.random() < 0.6:
        n = max(64, n // 64 * 64)
    c = {"op": op, "rows": _log_int(rng, 1, min(8191, (1 << 25) // n)), "n": n, "type": rng.choice(["fp16", "bf16", "fp32"])}
    if op == "norm":
        # what is added has the residual's type, or 16 bits beside a residual of 32; or there is nothing to add
        c["added"] = rng.choice(["fp16", "bf16", "fp32"]) if c["type"] == "fp32" else c["type"]
        c["added"] = rng.choice([c["added"], c["added"], "none"])
        c["weight"] = rng.choice(["fp16", "bf16", "fp32", "none"])
    return c


def _held(case):
    """The 16-bit type in which a pass gives what the codes stand for."""
    return "fp16" if case["type"] == "fp32" else case["type"]


def work(case):
    rows, size = case["rows"], BYTES[case["type"]]
    if case["op"] == "linear":
        k, m = case["k"], case["channels"]
        return {"bytes": rows * k + m * k + 4 * (rows + m) + (2 if case["bias"] else 0) * m + rows * m * size,
                "flops": 2 * rows * k * m}
    n = case["n"]
    out = rows * n * (1 + BYTES[_held(case)]) + 4 * rows  # codes, the values they stand for, scales
    if case["op"] == "quant":
        return {"bytes": rows * n * size + out, "flops": 4 * rows * n}
    if case["op"] == "silu":
        return {"bytes": 2 * rows * n * size + out, "flops": 9 * rows * n}
    added = case["added"]
    move = size if added == "none" else 2 * size + BYTES[added]
    return {"bytes": rows * n * move + (0 if case["weight"] == "none" else n * BYTES[case["weight"]]) + out,
            "flops": 8 * rows * n}


# --------------------------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------------------------
def _tokens(rows, n, g, device):
    """Activations: a normal bulk, and a few channels of every row several times as large."""
    x = torch.randn(rows, n, generator=g, device=device)
    large = torch.randint(0, n, (max(1, n // 512),), generator=g, device=device)
    x[:, large] *= 6.0
    return x


def _codes(rows, k, g, device):
    """Codes of a quantized normal matrix in rows that start on 16 bytes, as the quantizing operators write them."""
    held = torch.zeros(rows, -(-k // 16) * 16, dtype=torch.int8, device=device)
    step = max(1, (1 << 26) // k)
    for a in range(0, rows, step):
        v = torch.randn(min(step, rows - a), k, generator=g, device=device)
        held[a:a + step, :k] = (v * (127.0 / v.abs().amax(-1, keepdim=True))).round().to(torch.int8)
    return held[:, :k]


def prepare(case, seed):
    device = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=device)
    g.manual_seed(int(seed))
    kind = TYPES[case["type"]]
    s = {"case": case, "eps": 1e-5}
    rows = case["rows"]
    if case["op"] == "linear":
        k, m = case["k"], case["channels"]
        s["x"], s["w"] = _codes(rows, k, g, device), _codes(m, k, g, device)
        s["x_scale"] = 0.03 * (0.5 + torch.rand(rows, generator=g, device=device))
        s["w_scale"] = 6e-4 * (0.5 + torch.rand(m, generator=g, device=device))
        s["bias"] = torch.randn(m, generator=g, device=device).half() if case["bias"] else None
        if own:
            from opac1ty_b200 import int8

            s["weight"] = int8.Int8Weight(s["w"], s["w_scale"])
            s["tokens"] = int8.Int8Rows(s["x"], s["x_scale"])
        return s
    n = case["n"]
    if case["op"] == "quant":
        s["x"] = _tokens(rows, n, g, device).to(kind)
    elif case["op"] == "silu":
        s["gate_up"] = (1.5 * torch.randn(rows, 2 * n, generator=g, device=device)).to(kind)
    else:
        s["h"] = _tokens(rows, n, g, device).mul_(3.0).to(kind)
        s["y"] = None if case["added"] == "none" else torch.randn(rows, n, generator=g, device=device).to(TYPES[case["added"]])
        s["weight"] = None if case["weight"] == "none" else \
            (1.0 + 0.2 * torch.randn(n, generator=g, device=device)).to(TYPES[case["weight"]])
    return s


# --------------------------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------------------------
def run(s):
    case = s["case"]
    op, held = case["op"], TYPES[_held(case)]
    if own:
        from opac1ty_b200 import int8

        if op == "linear":
            return {"y": int8.linear(s["tokens"], s["weight"], bias=s["bias"], dtype=TYPES[case["type"]])}
        if op == "quant":
            r = int8.quantize(s["x"], values=held)
            return {"values": r.values, "scales": r.scales}
        if op == "silu":
            r = int8.silu_mul(s["gate_up"], values=held)
            return {"values": r.values, "scales": r.scales}
        h, r = int8.add_rmsnorm(s["h"], s["y"], s["weight"], eps=s["eps"], values=held)
        return {"h": h, "values": r.values, "scales": r.scales}
    if op == "linear":
        y = torch.matmul(s["x"].float(), s["w"].float().T) * s["x_scale"][:, None] * s["w_scale"][None, :]
        if s["bias"] is not None:
            y = y + s["bias"].float()[None, :]
        return {"y": y.to(TYPES[case["type"]])}
    if op == "quant":
        codes, scale = _rows8(s["x"].float())
    elif op == "silu":
        gate, up = s["gate_up"].float().chunk(2, -1)
        codes, scale = _rows8(gate / (1.0 + (-gate).exp()) * up)
    else:
        t = s["h"].float() if s["y"] is None else s["h"].float() + s["y"].float()
        rms = ((t * t).mean(-1, keepdim=True) + s["eps"]).sqrt()
        codes, scale = _rows8(t if s["weight"] is None else t.double() * s["weight"].double())
        scale = scale / rms
    out = {"values": (codes * scale).to(held), "scales": scale.squeeze(-1)}
    if op == "norm":
        out["h"] = t.to(s["h"].dtype)
    return out


def _rows8(v):
    """Codes (whole numbers in fp32) and scales of the rows of v; formed in 64 bits, since values lie next to a border."""
    v = v.double()
    big = v.abs().amax(-1, keepdim=True)
    live = big >= LEAST
    codes = (v * torch.where(live, 127.0 / big, torch.zeros_like(big))).round()
    return codes.float(), torch.where(live, big / 127.0, torch.zeros_like(big)).float()


# --------------------------------------------------------------------------------------------
# The same from the definitions, in 64 bits
# --------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        x = s["x"].to(torch.float64).mul_(s["x_scale"].double().unsqueeze(1))
        w = s["w"].to(torch.float64).mul_(s["w_scale"].double().unsqueeze(1))
        y = torch.mm(x, w.t())
        return {"y": y if s["bias"] is None else y.add_(s["bias"].double())}
    if case["op"] == "quant":
        return _stands_for(s["x"].double())
    if case["op"] == "silu":
        n = case["n"]
        g, u = s["gate_up"][:, :n].double(), s["gate_up"][:, n:].double()
        return _stands_for(g * torch.reciprocal(1 + torch.exp(-g)) * u)
    t = s["h"].double()
    if s["y"] is not None:
        t = t + s["y"].double()
    z = t / torch.sqrt(t.square().sum(-1, keepdim=True) / case["n"] + s["eps"])
    return {"h": t, **_stands_for(z if s["weight"] is None else z * s["weight"].double())}


def _stands_for(z):
    scale = torch.linalg.vector_norm(z, ord=math.inf, dim=-1, keepdim=True) / 127
    codes = torch.round(torch.where(scale > 0, z / scale, torch.zeros_like(z)))
    return {"values": codes * scale, "scales": scale[:, 0]}
