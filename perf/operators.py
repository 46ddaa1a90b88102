"""Cases for timing and comparing the 8-bit linear path: RMS norm (16-bit or 8-bit output,
residual added), row quantisation, the int8 x int8 linear layer, and a block of them.

`run` computes the operators with elementary torch operations in 32 bits (`own` false) or
calls the library's entry points (`own` true). What is held in 8 bits is returned as the
values it stands for, in the activations' 16-bit type, next to its fp32 scales.
"""
import math
import os
import sys

import torch

own = False

EPS = 1e-6
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
HERE = os.path.dirname(os.path.abspath(__file__))

#: bounds of the drawn cases: elements of a row operator, products and outputs of a linear layer
ROW_ELEMS = 8192 * 4096
PRODUCTS = 8192 * 4096 * 4096
OUTPUTS = 68451 * 1536


def listed():
    return [
        # the norm in front of a layer when one token of each of 16 sequences is processed
        {"name": "norm 16x4096 bf16", "op": "norm", "m": 16, "d": 4096, "type": "bf16", "residual": True},
        # 16-bit norm of a large batch, width odd: rows start at every alignment
        {"name": "norm 20000x1023 f16", "op": "norm", "m": 20000, "d": 1023, "type": "f16", "residual": False},
        # a corpus batch of 1,024 sentences (68,451 tokens) at the encoder's width
        {"name": "norm_i8 68451x384 f16", "op": "norm_i8", "m": 68451, "d": 384, "type": "f16", "residual": True},
        # a long prompt's hidden states
        {"name": "norm_i8 8192x4096 bf16", "op": "norm_i8", "m": 8192, "d": 4096, "type": "bf16", "residual": True},
        # the GELU output of 32 sentences of 512 tokens, before the second FFN layer
        {"name": "quantize 16384x1536 f16", "op": "quantize", "m": 16384, "d": 1536, "type": "f16"},
        # one sentence's attention output, a width that ends inside a vector
        {"name": "quantize 77x1000 bf16", "op": "quantize", "m": 77, "d": 1000, "type": "bf16"},
        # a single token: the weights' bytes are the work
        {"name": "linear 1x4096x4096 bf16", "op": "linear", "m": 1, "n": 4096, "k": 4096, "type": "bf16", "bias": False,
         "gelu": False},
        # a short query batch against a wide layer
        {"name": "linear 129x8192x2048 f16", "op": "linear", "m": 129, "n": 8192, "k": 2048, "type": "f16",
         "bias": True, "gelu": False},
        # odd in every direction
        {"name": "linear 1001x999x777 f16", "op": "linear", "m": 1001, "n": 999, "k": 777, "type": "f16", "bias": True,
         "gelu": False},
        # the encoder's first FFN layer over a corpus batch
        {"name": "linear 68451x1536x384 gelu", "op": "linear", "m": 68451, "n": 1536, "k": 384, "type": "f16",
         "bias": True, "gelu": True},
        # the largest product: a prompt of 8,192 tokens
        {"name": "linear 8192x4096x4096 bf16", "op": "linear", "m": 8192, "n": 4096, "k": 4096, "type": "bf16",
         "bias": False, "gelu": False},
        # norm -> up -> GELU -> quantise -> down, 8 x 128 tokens
        {"name": "ffn 1024x1024x4096 f16", "op": "ffn", "m": 1024, "d": 1024, "f": 4096, "type": "f16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm_i8", "quantize", "linear", "linear", "linear", "ffn"])
    kind = rng.choice(["f16", "bf16"])
    # widths: multiples of 8 or of nothing
    width = lambda lo, hi: (lambda v: v if rng.random() < 0.3 else max(8, v // 8 * 8))(_log(rng, lo, hi))
    if op in ("norm", "norm_i8", "quantize"):
        d = width(64, 16384)
        c = {"op": op, "m": _log(rng, 1, min(70000, ROW_ELEMS // d)), "d": d, "type": kind}
        return c if op == "quantize" else {**c, "residual": rng.random() < 0.6}
    if op == "linear":
        n, k = width(64, 8192), width(64, 8192)
        m = _log(rng, 1, max(1, min(70000, PRODUCTS // (n * k), OUTPUTS // n)))
        return {"op": op, "m": m, "n": n, "k": k, "type": kind, "bias": rng.random() < 0.5, "gelu": rng.random() < 0.3}
    return {"op": op, "m": _log(rng, 1, 4096), "d": width(128, 2048), "f": width(128, 8192), "type": kind}


# ------------------------------------------------------------------------------ inputs
def _activations(g, m, d, dtype):
    """Rows of different size, some channels eight times the others' as residual streams have them."""
    x = torch.randn(m, d, generator=g, device="cuda")
    x *= torch.exp(0.3 * torch.randn(m, 1, generator=g, device="cuda"))
    x *= 1 + 7 * (torch.rand(d, generator=g, device="cuda") < 0.01).float()
    return x.to(dtype)


def _int8_rows(g, rows, k, spread):
    """int8 [rows, k] with row strides of whole 16 bytes and one scale per row, as quantising normal values gives."""
    x = torch.randn(rows, k, generator=g, device="cuda")
    top = x.abs().amax(1, keepdim=True)
    q = torch.empty(rows, (k + 15) // 16 * 16, dtype=torch.int8, device="cuda")[:, :k]
    q.copy_(torch.round(x * (127 / top)))
    return q, (top[:, 0] / 127 * spread).contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, m = TYPES[case["type"]], case["m"]
    s = {"case": case, "dtype": dtype}
    if case["op"] in ("norm", "norm_i8", "quantize", "ffn"):
        d = case["d"]
        s["x"] = _activations(g, m, d, dtype)
        if case["op"] != "quantize":
            s["weight"] = (1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(dtype)
            s["residual"] = _activations(g, m, d, dtype) if case.get("residual", True) else None
    if case["op"] == "linear":
        n, k = case["n"], case["k"]
        s["a"], s["a_scale"] = _int8_rows(g, m, k, 1.0)
        s["w"], s["w_scale"] = _int8_rows(g, n, k, k**-0.5)
        s["bias"] = (0.1 * torch.randn(n, generator=g, device="cuda")).to(dtype) if case["bias"] else None
    if case["op"] == "ffn":
        d, f = case["d"], case["f"]
        s["up"], s["up_scale"] = _int8_rows(g, f, d, d**-0.5)
        s["down"], s["down_scale"] = _int8_rows(g, d, f, f**-0.5)
        s["up_bias"] = (0.1 * torch.randn(f, generator=g, device="cuda")).to(dtype)
        s["down_bias"] = (0.1 * torch.randn(d, generator=g, device="cuda")).to(dtype)
    return s


# ------------------------------------------------------------------------------ plain forms
def _norm(x, weight, residual):
    v = x.float()
    if residual is not None:
        v = v + residual.float()
    return v * torch.rsqrt((v * v).mean(1, keepdim=True) + EPS) * weight.float(), v


def _quantize(y):
    scale = y.abs().amax(1, keepdim=True) / 127
    return torch.round(y / torch.where(scale == 0, 1.0, scale)), scale


def _linear(q, q_scale, w, w_scale, bias, gelu):
    y = (q.float() @ w.float().T) * q_scale[:, None] * w_scale
    if bias is not None:
        y = y + bias.float()
    return 0.5 * y * (1 + torch.erf(y * 0.5**0.5)) if gelu else y


def _plain(s):
    op, dtype = s["case"]["op"], s["dtype"]
    if op == "norm":
        y, v = _norm(s["x"], s["weight"], s["residual"])
        return y.to(dtype) if s["residual"] is None else (y.to(dtype), v.to(dtype))
    if op == "norm_i8":
        y, v = _norm(s["x"], s["weight"], s["residual"])
        q, scale = _quantize(y)
        out = ((q * scale).to(dtype), scale[:, 0])
        return out if s["residual"] is None else (*out, v.to(dtype))
    if op == "quantize":
        q, scale = _quantize(s["x"].float())
        return (q * scale).to(dtype), scale[:, 0]
    if op == "linear":
        return _linear(s["a"], s["a_scale"], s["w"], s["w_scale"], s["bias"], s["case"]["gelu"]).to(dtype)
    y, v = _norm(s["x"], s["weight"], s["residual"])
    q, scale = _quantize(y)
    h = _linear(q, scale[:, 0], s["up"], s["up_scale"], s["up_bias"], True).to(dtype)
    q, scale = _quantize(h.float())
    return _linear(q, scale[:, 0], s["down"], s["down_scale"], s["down_bias"], False).to(dtype), v.to(dtype)


# ------------------------------------------------------------------------------ the library's calls
def _bbh():
    package = os.path.join(os.path.dirname(HERE), "bert-by-hand_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import bbh

    return bbh


def _own(s):
    bbh = sys.modules.get("bbh") or _bbh()
    op, dtype = s["case"]["op"], s["dtype"]
    if op == "norm":
        return bbh.rmsnorm(s["x"], s["weight"], EPS, residual=s["residual"])
    if op == "norm_i8":
        q, scale, *v = bbh.rmsnorm_i8(s["x"], s["weight"], EPS, residual=s["residual"])
        return (bbh.dequantize_i8(q, scale, dtype), scale, *v)
    if op == "quantize":
        q, scale = bbh.quantize_i8(s["x"])
        return bbh.dequantize_i8(q, scale, dtype), scale
    if op == "linear":
        return bbh.linear_i8(s["a"], s["a_scale"], s["w"], s["w_scale"], s["bias"], gelu=s["case"]["gelu"], dtype=dtype)
    q, scale, v = bbh.rmsnorm_i8(s["x"], s["weight"], EPS, residual=s["residual"])
    h = bbh.linear_i8(q, scale, s["up"], s["up_scale"], s["up_bias"], gelu=True, dtype=dtype)
    q, scale = bbh.quantize_i8(h)
    return bbh.linear_i8(q, scale, s["down"], s["down_scale"], s["down_bias"], dtype=dtype), v


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------ least work
def work(case):
    op, m = case["op"], case["m"]
    if op == "linear":
        n, k = case["n"], case["k"]
        return {"bytes": m * k + n * k + 4 * m + 4 * n + (2 * n if case["bias"] else 0) + 2 * m * n,
                "flops": 2 * m * n * k}
    d = case["d"]
    if op == "quantize":
        return {"bytes": 4 * m * d + 4 * m, "flops": 3 * m * d}
    if op == "ffn":
        f = case["f"]
        return {"bytes": 4 * m * d + 2 * d + 2 * d * f + 4 * (d + f) + 2 * (d + f) + 4 * m * d, "flops": 4 * m * d * f}
    r = 2 if case["residual"] else 1
    return {"bytes": r * 4 * m * d + 2 * d + (4 * m if op == "norm_i8" else 0), "flops": 6 * m * d}


# ------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    f64 = lambda t: None if t is None else t.to(torch.float64)
    dtype = s["dtype"]

    def eight_bits(t):  # the integers and what one of them stands for
        step = torch.linalg.vector_norm(t, float("inf"), dim=1) / 127.0
        return torch.where(step[:, None] > 0, t / step[:, None], 0.0).round(), step

    def product(a, sa, w, sw, bias, gelu):
        z = torch.einsum("mk,nk->mn", a, f64(w)) * torch.outer(f64(sa), f64(sw))
        if bias is not None:
            z = z + f64(bias)
        return z * torch.special.erfc(-z / math.sqrt(2.0)) / 2 if gelu else z

    if case["op"] == "linear":
        return product(f64(s["a"]), s["a_scale"], s["w"], s["w_scale"], s["bias"], case["gelu"])
    x = f64(s["x"])
    if case["op"] == "quantize":
        q, step = eight_bits(x)
        return q * step[:, None], step
    total = x if s["residual"] is None else x + f64(s["residual"])
    y = total / torch.sqrt(total.square().sum(1, keepdim=True) / case["d"] + EPS) * f64(s["weight"])
    if case["op"] == "norm":
        return y if s["residual"] is None else (y, total)
    q, step = eight_bits(y)
    if case["op"] == "norm_i8":
        return (q * step[:, None], step) if s["residual"] is None else (q * step[:, None], step, total)
    h = f64(product(q, step, s["up"], s["up_scale"], s["up_bias"], True).to(dtype))  # the layer's 16-bit output
    q, step = eight_bits(h)
    return product(q, step, s["down"], s["down_scale"], s["down_bias"], False), total
