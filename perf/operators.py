"""The 8-bit integer operators of the sentence encoder: what is measured, and their plain forms.

  linear   y = x . w^T of int8 rows, times a scale per token and a scale per channel, plus a bias
  norm     x + residual -> LayerNorm or RMS norm -> int8 rows with a scale per token
  quant    activation (none or erf-GELU) -> int8 rows with a scale per token

``own`` False computes them with elementary torch operations in 32 bits, True calls the
framework.  8-bit results are returned as the values that they stand for, in 16 bits.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}
MOST_LINEAR = 65536 * 4096 * 1024      # token x feature x depth of the largest listed product
MOST_ROWS = 65521 * 4096               # elements of the largest listed row operator
TINY = 2.0 ** -100                     # a row with no larger magnitude counts as zeros


def listed():
    return [
        # one token through a 1024 -> 4096 projection: the smallest call, a latency
        dict(name="linear_1_token", op="linear", rows=1, depth=1024, features=4096, out="f16", bias=True),
        # the q|k|v projection of a 384-wide encoder for one search query of 14 tokens
        dict(name="linear_query", op="linear", rows=14, depth=384, features=1152, out="f16", bias=True),
        # a handful of documents, every size odd, wide results in 32 bits
        dict(name="linear_odd", op="linear", rows=613, depth=999, features=2051, out="f32", bias=True),
        # q|k|v of a 768-wide encoder over an ingest batch with its padding dropped
        dict(name="linear_ingest", op="linear", rows=21853, depth=768, features=2304, out="f16", bias=True),
        # the second FFN product of a 1024-wide encoder over a very large ingest batch
        dict(name="linear_large", op="linear", rows=65536, depth=4096, features=1024, out="bf16", bias=True),
        # one token of a pre-norm model
        dict(name="norm_1_token", op="norm", rows=1, cols=1024, norm="rms", x="bf16", residual="bf16",
             bias=False, sum=True, keep="none"),
        # one query between a 384-wide encoder's sublayers
        dict(name="norm_query", op="norm", rows=37, cols=384, norm="layer", x="f16", residual="f32",
             bias=True, sum=False, keep="f32"),
        # an ingest batch between a 768-wide encoder's sublayers
        dict(name="norm_ingest", op="norm", rows=32749, cols=768, norm="layer", x="f16", residual="f32",
             bias=True, sum=False, keep="f32"),
        # wide rows of a pre-norm model, its residual stream updated
        dict(name="norm_large", op="norm", rows=65521, cols=4096, norm="rms", x="bf16", residual="bf16",
             bias=False, sum=True, keep="none"),
        # the FFN activation of one token
        dict(name="quant_1_token", op="quant", rows=1, cols=4096, act="gelu", x="f16"),
        # attention results of a few documents, an odd width
        dict(name="quant_odd", op="quant", rows=1021, cols=1531, act="none", x="bf16"),
        # the FFN activation of a very large ingest batch
        dict(name="quant_large", op="quant", rows=65521, cols=4096, act="gelu", x="f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "norm", "quant"])
    rows = _log(rng, 1, 65536)
    if op == "linear":
        depth, features = _log(rng, 16, 4096), _log(rng, 16, 4608)
        rows = max(1, min(rows, MOST_LINEAR // (depth * features)))
        return dict(op=op, rows=rows, depth=depth, features=features,
                    out=rng.choice(["f16", "bf16", "f32"]), bias=rng.random() < 0.75)
    cols = _log(rng, 17, 8192)
    rows = max(1, min(rows, MOST_ROWS // cols))
    if op == "quant":
        return dict(op=op, rows=rows, cols=cols, act=rng.choice(["none", "gelu"]),
                    x=rng.choice(["f16", "bf16", "f32"]))
    residual = rng.choice(["none", "f16", "bf16", "f32"])
    return dict(op=op, rows=rows, cols=cols, norm=rng.choice(["layer", "rms"]),
                x=rng.choice(["f16", "bf16", "f32"]), residual=residual, bias=rng.random() < 0.5,
                sum=residual != "none" and rng.random() < 0.5,
                keep=rng.choice(["none", "f16", "bf16", "f32"]))


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _int8_rows(g, rows, cols):
    """Rows as a quantiser leaves them: normal values, 16-byte row strides."""
    stride = (cols + 15) // 16 * 16
    q = torch.randn(rows, stride, generator=g, device="cuda").mul_(32).round_().clamp_(-127, 127)
    return q.to(torch.int8)[:, :cols]


def _activations(g, rows, cols, dtype, spread):
    """Normal values with some wide channels, as trained encoders have them."""
    wide = 1 + 4 * (torch.rand(cols, generator=g, device="cuda") < 0.02).float()
    return torch.randn(rows, cols, generator=g, device="cuda").mul_(wide * spread).to(dtype)


def prepare(case, seed):
    g = _generator(seed)
    if case["op"] == "linear":
        t, k, n = case["rows"], case["depth"], case["features"]
        bias = torch.randn(n, generator=g, device="cuda") * 0.1 if case["bias"] else None
        return dict(case=case, x=_int8_rows(g, t, k), w=_int8_rows(g, n, k), bias=bias,
                    x_scale=(0.5 + torch.rand(t, generator=g, device="cuda")) / 32,
                    w_scale=(0.5 + torch.rand(n, generator=g, device="cuda")) / (32 * math.sqrt(k)))
    t, h = case["rows"], case["cols"]
    state = dict(case=case, x=_activations(g, t, h, DTYPES[case["x"]], 1.0))
    if case["op"] == "norm":
        if case["residual"] != "none":
            state["residual"] = _activations(g, t, h, DTYPES[case["residual"]], 1.5)
        state["weight"] = 1 + 0.1 * torch.randn(h, generator=g, device="cuda")
        state["bias"] = 0.1 * torch.randn(h, generator=g, device="cuda") if case["bias"] else None
    return state


def _value_dtype(case):
    return torch.bfloat16 if case["x"] == "bf16" else torch.float16


def _round_rows(v, dtype):
    """The int8 grid of each row, as values: scale = max|v| / 127, ties to even."""
    a = v.abs().amax(1, keepdim=True)
    zero = a < TINY
    q = torch.round(v * (127 / torch.where(zero, torch.ones_like(a), a)))
    return (torch.where(zero, torch.zeros_like(q), q) * (a / 127)).to(dtype)


def _normed(h, state, eps):
    if state["case"]["norm"] == "layer":
        h = h - h.mean(1, keepdim=True)
    n = h * torch.rsqrt((h * h).mean(1, keepdim=True) + eps) * state["weight"].to(h.dtype)
    return n if state["bias"] is None else n + state["bias"].to(h.dtype)


EPS = 1e-6


def _plain(state):
    case = state["case"]
    if case["op"] == "linear":
        y = (state["x"].float() @ state["w"].float().T) * state["x_scale"][:, None] * state["w_scale"]
        return (y if state["bias"] is None else y + state["bias"]).to(DTYPES[case["out"]])
    x = state["x"].float()
    if case["op"] == "quant":
        if case["act"] == "gelu":
            x = 0.5 * x * (1 + torch.erf(x * math.sqrt(0.5)))
        return {"value": _round_rows(x, _value_dtype(case))}
    h = x + state["residual"].float() if "residual" in state else x
    n = _normed(h, state, EPS)
    out = {"value": _round_rows(n, _value_dtype(case))}
    if case["sum"]:
        out["sum"] = h.to(DTYPES[case["residual"]])
    if case["keep"] != "none":
        out["normed"] = n.to(DTYPES[case["keep"]])
    return out


def _framework():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    path = os.path.join(root, "hc-rag_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import hcrag_amd
    return hcrag_amd


_package = None


def _own(state):
    global _package
    if _package is None:
        _package = _framework()
    case = state["case"]
    if case["op"] == "linear":
        return _package.int8_linear(_package.Int8Rows(state["x"], state["x_scale"]),
                                    _package.Int8Rows(state["w"], state["w_scale"]),
                                    bias=state["bias"], dtype=DTYPES[case["out"]])
    if case["op"] == "quant":
        rows = _package.quantize_rows(state["x"], act=case["act"])
        return {"value": rows.dequantize(_value_dtype(case))}
    total = torch.empty_like(state["residual"]) if case["sum"] else None
    normed = None
    if case["keep"] != "none":
        normed = torch.empty(state["x"].shape, dtype=DTYPES[case["keep"]], device=state["x"].device)
    rows = _package.norm_quantize(state["x"], state["weight"], bias=state["bias"],
                                  residual=state.get("residual"), norm=case["norm"], eps=EPS,
                                  sum_out=total, norm_out=normed)
    out = {"value": rows.dequantize(_value_dtype(case))}
    if total is not None:
        out["sum"] = total
    if normed is not None:
        out["normed"] = normed
    return out


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    if case["op"] == "linear":
        t, k, n = case["rows"], case["depth"], case["features"]
        moved = t * k + n * k + 4 * t + 4 * n + (4 * n if case["bias"] else 0) + t * n * SIZE[case["out"]]
        return {"bytes": moved, "flops": 2 * t * k * n}
    t, h = case["rows"], case["cols"]
    each = SIZE[case["x"]] + 1
    if case["op"] == "quant":
        return {"bytes": t * (h * each + 4), "flops": (12 if case["act"] == "gelu" else 3) * t * h}
    if case["residual"] != "none":
        each += SIZE[case["residual"]] * (2 if case["sum"] else 1)
    if case["keep"] != "none":
        each += SIZE[case["keep"]]
    return {"bytes": t * (h * each + 4) + 4 * h * (2 if case["bias"] else 1), "flops": 10 * t * h}


def _exact_rows(v):
    """[rows, cols] float64 -> the values on each row's int8 grid, float64."""
    scale = v.abs().max(dim=1).values / 127
    steps = torch.zeros_like(v)
    some = scale * 127 >= TINY
    steps[some] = torch.round(v[some] / scale[some, None])
    return steps * scale[:, None]


def exact(case, seed):
    state = prepare(case, seed)
    d = torch.float64
    if case["op"] == "linear":
        # the sums are whole numbers below 2^53: exact in 64 bits in any order
        sums = torch.mm(state["x"].to(d), state["w"].to(d).t())
        y = sums * torch.outer(state["x_scale"].to(d), state["w_scale"].to(d))
        if state["bias"] is not None:
            y += state["bias"].to(d)
        return y
    x = state["x"].to(d)
    if case["op"] == "quant":
        if case["act"] == "gelu":
            x = x * torch.special.ndtr(x)
        return {"value": _exact_rows(x)}
    if "residual" in state:
        x = x + state["residual"].to(d)
    centre = x.sum(dim=1, keepdim=True) / case["cols"] if case["norm"] == "layer" else 0.0
    spread = ((x - centre) ** 2).sum(dim=1, keepdim=True) / case["cols"]
    n = (x - centre) / torch.sqrt(spread + EPS) * state["weight"].to(d)
    if state["bias"] is not None:
        n = n + state["bias"].to(d)
    out = {"value": _exact_rows(n)}
    if case["sum"]:
        out["sum"] = x
    if case["keep"] != "none":
        out["normed"] = n
    return out
