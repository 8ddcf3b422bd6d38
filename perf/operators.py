"""The 8-bit inference operators as cases that can be timed: in their plain form, and by the framework's calls.

Five kinds:

* ``linear``   - the product of 8-bit rows with an 8-bit weight, a scale per token and per output channel, plus a bias;
* ``quantize`` - rows to 8-bit integers with a scale per row, behind nothing, GELU or SiLU (the inputs of a product);
* ``rms``      - residual addition and RMS norm, the result in 8 bits;
* ``adaln``    - gated residual addition, LayerNorm and modulation, the result in 8 bits;
* ``mlp``      - a run of them: the second half of a transformer block up to its last product.

A row y in 8 bits: a = max|y|, scale = a / 127, q = y * (127 / a) rounded to the nearest integer, ties to even.  What is held in 8
bits is returned as q * scale.

Widths are those of the model configurations (hidden 384 / 768 / 1024 / 1152, 4 times that in the MLP, 6 times that in the
modulation), tokens those of the 256- and 512-pixel settings (256 and 1024 an image), of single conditioning vectors and odd ones.
"""

from __future__ import annotations

import torch

own = False

DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
TINY = 2.0 ** -120      # a row whose values are all below this counts as zeros


def listed():
    return [
        # the modulation of one image: one conditioning vector times the widest weight of the largest model (latency, and the weight's bytes)
        _linear("linear_modulation_1_image", 1, 1152, 6912),
        # the MLP's second product on one 256-pixel image of the largest model: few rows, a long sum
        _linear("linear_256_tokens", 256, 4608, 1152),
        # sizes that fit no tile: a cropped image's tokens in fp16
        _linear("linear_odd_fp16", 333, 1001, 777, dtype="fp16"),
        # the qkv projection of 8 guided 512-pixel images (16 in the batch) of the largest model
        _linear("linear_qkv_512px", 16384, 1152, 3456),
        # the conditioning vectors of a batch of 8 behind SiLU, in front of the modulation
        {"name": "quantize_silu_8_vectors", "kind": "quantize", "M": 8, "C": 1152, "act": "silu", "dtype": "bf16"},
        # the MLP's hidden activations behind GELU, 8 guided 512-pixel images
        {"name": "quantize_gelu_512px", "kind": "quantize", "M": 16384, "C": 4608, "act": "gelu", "dtype": "bf16"},
        # residual + RMS norm of one token, the residual stream in fp32
        {"name": "rms_1_token", "kind": "rms", "M": 1, "C": 1152, "dtype": "bf16", "stream": "fp32", "residual": True},
        # residual + RMS norm over the tokens of 32 512-pixel images
        {"name": "rms_512px", "kind": "rms", "M": 32768, "C": 1152, "dtype": "bf16", "stream": "bf16", "residual": True},
        # adaLN in front of the MLP, one 256-pixel image of the smallest model
        {"name": "adaln_1_image", "kind": "adaln", "B": 1, "L": 256, "C": 384, "dtype": "bf16", "gated": True},
        # the same, 8 guided 512-pixel images of the largest model
        {"name": "adaln_512px", "kind": "adaln", "B": 16, "L": 1024, "C": 1152, "dtype": "bf16", "gated": True},
        # adaLN, first product, GELU, second product: one 256-pixel image of the smallest model
        {"name": "mlp_1_image", "kind": "mlp", "B": 1, "L": 256, "C": 384},
        # the same, 8 guided 512-pixel images of the largest model
        {"name": "mlp_512px", "kind": "mlp", "B": 16, "L": 1024, "C": 1152},
    ]


def _linear(name, M, K, N, dtype="bf16", bias=True):
    return {"name": name, "kind": "linear", "M": M, "K": K, "N": N, "dtype": dtype, "bias": bias}


def _spread(rng, lo, hi):
    """A whole number, spread over the logarithm."""
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def _width(rng, lo, hi):
    """Half of them widths of the models, half anything."""
    if rng.random() < 0.5:
        return rng.choice([c for c in (384, 768, 1024, 1152, 1536, 3456, 4096, 4608, 6912) if lo <= c <= hi])
    return _spread(rng, lo, hi)


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "quantize", "rms", "adaln", "mlp"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "linear":
        M, K, N = _spread(rng, 1, 16384), _width(rng, 64, 4608), _width(rng, 64, 6912)
        most = 16384 * 1152 * 3456
        return {"kind": kind, "M": max(1, min(M, most // (K * N))), "K": K, "N": N, "dtype": rng.choice([dtype, dtype, "fp32"]),
                "bias": rng.random() < 0.7}
    if kind == "quantize":
        C = _width(rng, 64, 4608)
        return {"kind": kind, "M": _spread(rng, 1, min(32768, 16384 * 4608 // C)), "C": C, "act": rng.choice(["none", "gelu", "silu"]),
                "dtype": dtype}
    if kind == "rms":
        C = _width(rng, 64, 4608)
        return {"kind": kind, "M": _spread(rng, 1, min(32768, 32768 * 1152 // C)), "C": C, "dtype": dtype,
                "stream": rng.choice([dtype, "fp32"]), "residual": rng.random() < 0.8}
    if kind == "adaln":
        C = _width(rng, 64, 4608)
        B = _spread(rng, 1, 32)
        return {"kind": kind, "B": B, "L": _spread(rng, 1, max(1, min(1024, 16 * 1024 * 1152 // (C * B)))), "C": C, "dtype": dtype,
                "gated": rng.random() < 0.7}
    return {"kind": kind, "B": _spread(rng, 1, 16), "L": rng.choice([256, 1024, _spread(rng, 1, 1024)]), "C": rng.choice([384, 768, 1024, 1152])}


# ---- what a program has in hand before the call ---------------------------------------------------------------------

def _randn(gen, *shape, dtype=torch.bfloat16, std=1.0):
    return (torch.randn(*shape, device=DEV, generator=gen) * std).to(dtype)


def _activations(gen, *shape, dtype=torch.bfloat16):
    """Normal values whose channels differ in size, a few of them much larger, as a network's activations do."""
    x = torch.randn(*shape, device=DEV, generator=gen)
    size = torch.exp(0.3 * torch.randn(shape[-1], device=DEV, generator=gen))
    size *= torch.where(torch.rand(shape[-1], device=DEV, generator=gen) < 0.005, 6.0, 1.0)
    return (x * size).to(dtype)


def _held(y):
    """(q, scale) of the rows of y, rows of q at a pitch of whole 16-byte units."""
    q, scale = _quantize(y.float())
    K = q.shape[-1]
    rows = torch.zeros(*q.shape[:-1], -(-K // 16) * 16, dtype=torch.int8, device=y.device)[..., :K]
    rows.copy_(q)
    return rows, scale


def _weight(gen, N, K):
    bound = (6.0 / (N + K)) ** 0.5
    return _held((torch.rand(N, K, device=DEV, generator=gen) * 2 - 1) * bound)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    kind, s = case["kind"], {"case": case}
    if kind == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        s["x"], s["w"] = _held(_activations(gen, M, K)), _weight(gen, N, K)
        s["bias"] = _randn(gen, N, dtype=torch.float32, std=0.1) if case["bias"] else None
    elif kind == "quantize":
        s["x"] = _activations(gen, case["M"], case["C"], dtype=DTYPES[case["dtype"]])
    elif kind == "rms":
        M, C = case["M"], case["C"]
        s["x"] = _activations(gen, M, C, dtype=DTYPES[case["dtype"]])
        s["residual"] = _activations(gen, M, C, dtype=DTYPES[case["stream"]]) if case["residual"] else None
        s["weight"] = 1 + _randn(gen, C, dtype=torch.float32, std=0.1)
    else:
        B, L, C, dt = case["B"], case["L"], case["C"], DTYPES[case.get("dtype", "bf16")]
        s["x"], s["h"] = _activations(gen, B, L, C, dtype=dt), _activations(gen, B, L, C, dtype=dt)
        # six modulation vectors a sample, as one product gives them: three of them are slices of it here
        s["mod"] = _randn(gen, B, 1, 6 * C, dtype=dt, std=0.3)
        if kind == "mlp":
            s["w1"], s["w2"] = _weight(gen, 4 * C, C), _weight(gen, C, 4 * C)
            s["b1"], s["b2"] = _randn(gen, 4 * C, dtype=torch.float32, std=0.1), _randn(gen, C, dtype=torch.float32, std=0.1)
    return s


# ---- the operators in their plain form --------------------------------------------------------------------------------

def _quantize(y):
    """Rows of fp32 values -> whole numbers from -127 to 127 (held in fp32) and a scale per row."""
    a = y.abs().amax(-1)
    some = a >= TINY
    inverse = torch.where(some, 127.0 / a, torch.zeros_like(a))
    return torch.round(y * inverse[..., None]), torch.where(some, a / 127.0, torch.zeros_like(a))


def _values(q, scale, dtype):
    return (q * scale[..., None]).to(dtype)


def _act(x, act):
    if act == "gelu":
        return 0.5 * x * (1 + torch.tanh(0.7978845608028654 * (x + 0.044715 * x * x * x)))
    return x / (1 + torch.exp(-x)) if act == "silu" else x


def _product(q, scale, w, bias):
    """fp32 sums of products of whole numbers; not rounded yet."""
    wq, wscale = w
    out = (q.float() @ wq.float().t()) * scale[..., None] * wscale
    return out if bias is None else out + bias


def _rms(z, weight):
    return z * torch.rsqrt((z * z).mean(-1, keepdim=True) + 1e-6) * weight


def _modulated(z, shift, scale):
    c = z - z.mean(-1, keepdim=True)
    return c * torch.rsqrt((c * c).mean(-1, keepdim=True) + 1e-6) * (1 + scale) + shift


def _mods(s):
    return s["mod"].chunk(6, dim=-1)[2:5]       # the attention's gate, the MLP's shift and scale


def _narrow(case):
    return torch.float16 if case["dtype"] == "fp16" else torch.bfloat16


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "linear":
        return _product(*s["x"], s["w"], s["bias"]).to(DTYPES[case["dtype"]])
    if kind == "quantize":
        return _values(*_quantize(_act(s["x"].float(), case["act"])), _narrow(case))
    if kind == "rms":
        z = s["x"].float()
        if s["residual"] is not None:
            z = s["residual"].float() + z
        values = _values(*_quantize(_rms(z, s["weight"])), _narrow(case))
        return values if s["residual"] is None else (values, z.to(s["residual"].dtype))
    gate, shift, scale = (m.float() for m in _mods(s))
    z = s["x"].float()
    if case.get("gated", True):
        z = z + gate * s["h"].float()
    q, row_scale = _quantize(_modulated(z, shift, scale))
    if kind == "adaln":
        values = _values(q, row_scale, _narrow(case))
        return (values, z.to(s["x"].dtype)) if case["gated"] else values
    u = _product(q, row_scale, s["w1"], s["b1"]).to(s["x"].dtype)       # held in 16 bits between the products
    out = _product(*_quantize(_act(u.float(), "gelu")), s["w2"], s["b2"])
    return out.to(s["x"].dtype), z.to(s["x"].dtype)


# ---- the framework's calls --------------------------------------------------------------------------------------------

def _run_own(s):
    from dmf_b200.int8 import Int8Rows, int8_linear, ln_modulate_int8, quantize_int8, rms_norm_int8
    case = s["case"]
    kind = case["kind"]
    if kind == "linear":
        return int8_linear(Int8Rows(*s["x"]), Int8Rows(*s["w"]), s["bias"], out_dtype=DTYPES[case["dtype"]])
    if kind == "quantize":
        return quantize_int8(s["x"], None if case["act"] == "none" else case["act"]).dequantize(_narrow(case))
    if kind == "rms":
        if s["residual"] is None:
            return rms_norm_int8(s["x"], s["weight"], 1e-6).dequantize(_narrow(case))
        rows, z = rms_norm_int8(s["x"], s["weight"], 1e-6, residual=s["residual"])
        return rows.dequantize(_narrow(case)), z
    gate, shift, scale = _mods(s)
    if not case.get("gated", True):
        return ln_modulate_int8(s["x"], shift, scale, 1e-6).dequantize(_narrow(case))
    rows, z = ln_modulate_int8(s["x"], shift, scale, 1e-6, gate=gate, h=s["h"])
    if kind == "adaln":
        return rows.dequantize(_narrow(case)), z
    u = int8_linear(rows, Int8Rows(*s["w1"]), s["b1"], out_dtype=s["x"].dtype)
    return int8_linear(quantize_int8(u, "gelu"), Int8Rows(*s["w2"]), s["b2"], out_dtype=s["x"].dtype), z


# ---- what a pass cannot do without ------------------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    if kind == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        return {"bytes": M * K + N * K + 4 * (M + N) + 4 * N * case["bias"] + M * N * size[case["dtype"]], "flops": 2 * M * N * K}
    if kind == "quantize":
        n = case["M"] * case["C"]
        return {"bytes": 4 * n, "flops": {"none": 3, "gelu": 11, "silu": 7}[case["act"]] * n}
    if kind == "rms":
        n = case["M"] * case["C"]
        return {"bytes": n * (4 + 2 * size[case["stream"]] * case["residual"]) + 4 * case["C"], "flops": (7 + case["residual"]) * n}
    B, L, C = case["B"], case["L"], case["C"]
    n = B * L * C
    gated = case.get("gated", True)
    if kind == "adaln":
        return {"bytes": n * (8 if gated else 4) + 2 * B * C * (3 if gated else 2), "flops": (10 + 2 * gated) * n}
    return {"bytes": 8 * n + 6 * B * C + 8 * C * C + 4 * (4 * C + C) * 2, "flops": 16 * n * C}


# ---- from the definition, in 64 bits ----------------------------------------------------------------------------------

def _exact_rows(y):
    most = y.abs().max(dim=-1, keepdim=True).values
    step = most / 127
    whole = torch.where(most >= TINY, (127 * y / most.clamp_min(TINY)).round(), 0.0)
    return whole, torch.where(most >= TINY, step, 0.0)


def _exact_gelu(x):
    u = (2 / torch.pi) ** 0.5 * (x + 0.044715 * x ** 3)
    return x * torch.sigmoid(2 * u)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]

    def linear(whole, step, w, bias):
        out = torch.mm(whole, w[0].double().t()) * step * w[1].double().unsqueeze(0)
        return out + (0 if bias is None else bias.double())

    if kind == "linear":
        q, scale = s["x"]
        return linear(q.double(), scale.double().unsqueeze(1), s["w"], s["bias"])
    if kind == "quantize":
        x = s["x"].double()
        x = {"none": lambda v: v, "gelu": _exact_gelu, "silu": lambda v: v * torch.sigmoid(v)}[case["act"]](x)
        whole, step = _exact_rows(x)
        return whole * step
    if kind == "rms":
        z = s["x"].double() + (0 if s["residual"] is None else s["residual"].double())
        whole, step = _exact_rows(z / (z.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * s["weight"].double())
        return whole * step if s["residual"] is None else (whole * step, z)
    gate, shift, scale = (m.double() for m in _mods(s))
    gated = case.get("gated", True)
    z = s["x"].double() + (gate * s["h"].double() if gated else 0)
    normal = (z - z.mean(-1, keepdim=True)) / (z.var(-1, unbiased=False, keepdim=True) + 1e-6).sqrt()
    whole, step = _exact_rows(normal * (1 + scale) + shift)
    if kind == "adaln":
        return (whole * step, z) if gated else whole * step
    u = linear(whole.flatten(0, 1), step.flatten(0, 1), s["w1"], s["b1"]).to(s["x"].dtype).double()
    whole, step = _exact_rows(_exact_gelu(u))
    return linear(whole, step, s["w2"], s["b2"]).unflatten(0, z.shape[:2]), z
