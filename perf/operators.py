"""The operators around and of a layer's product with FP8 weights, as a program
that serves a model calls them: the root-mean-square norm with the residual's
addition and an 8-bit output, the 8-bit rounding of rows, and the matrix
product of 8-bit rows with FP8 weights, its epilogue included.

listed() holds named cases, draw() more of the same ranges; prepare() makes
what such a program holds before the call, run() is one call (the plain form in
torch's elementary operations, or with `own` the framework's), work() what the
call cannot do without, exact() the result in 64 bits.

8-bit outputs are returned as float8_e4m3fn tensors (the values they stand
for), their row scales beside them.
"""
import math
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

EPS = 1e-6
FP8_MAX = 448.0
AMAX_MIN = 2.0 ** -100   # rows of zeros get the scale of this maximum


def listed():
    return [
        # -- norm + residual -> 8 bits, rows of the benchmark's 5120 columns ----
        # one token of a decoding step: latency
        {"name": "norm_1x5120", "op": "norm", "M": 1, "D": 5120, "residual": True},
        # a batch of prompts
        {"name": "norm_8192x5120", "op": "norm", "M": 8192, "D": 5120, "residual": True},
        # a first layer (no residual yet), odd row count, rows of no power of two
        {"name": "norm_odd", "op": "norm", "M": 1777, "D": 1296, "residual": False},
        # -- rows -> 8 bits: the gated product's output, 17408 columns -----------
        {"name": "quant_5x17408", "op": "quant", "M": 5, "D": 17408},
        {"name": "quant_8192x17408", "op": "quant", "M": 8192, "D": 17408},
        # -- matrix product with its epilogue ---------------------------------
        # one token through gate and up (17408 rows each) of a layer
        {"name": "up_1", "op": "linear", "M": 1, "C": 5120, "R": 34816, "gated": True,
         "act": "silu", "bias": False, "residual": False},
        # a few sequences' tokens through the down projection, residual added
        {"name": "down_7", "op": "linear", "M": 7, "C": 17408, "R": 5120, "gated": False,
         "act": "none", "bias": False, "residual": True},
        # a serving batch of tokens, one a sequence
        {"name": "up_97", "op": "linear", "M": 97, "C": 5120, "R": 34816, "gated": True,
         "act": "silu", "bias": False, "residual": False},
        # a small layer with bias and GELU, odd counts on every side
        {"name": "small_odd", "op": "linear", "M": 1003, "C": 1296, "R": 2187, "gated": False,
         "act": "gelu", "bias": True, "residual": False},
        # one prompt through the down projection
        {"name": "down_2048", "op": "linear", "M": 2048, "C": 17408, "R": 5120, "gated": False,
         "act": "none", "bias": True, "residual": True},
        # a batch of prompts through gate and up
        {"name": "up_8192", "op": "linear", "M": 8192, "C": 5120, "R": 34816, "gated": True,
         "act": "silu", "bias": False, "residual": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm", "quant", "linear", "linear", "linear"))
    if op != "linear":
        d = 16 * _log_int(rng, 4, 1088)
        m = min(_log_int(rng, 1, 16384), 8192 * 17408 // d)
        case = {"op": op, "M": m, "D": d}
        if op == "norm":
            case["residual"] = rng.random() < 0.75
        return case
    most = 34816 * 5120
    c = 16 * _log_int(rng, 16, 1088)
    r = min(_log_int(rng, 256, 34816), most // c)
    gated = rng.random() < 0.4
    r -= r % 2 if gated else 0
    m = _log_int(rng, 1, 8192)
    return {"op": "linear", "M": m, "C": c, "R": r, "gated": gated,
            "act": rng.choice(("none", "relu", "silu", "gelu", "gelu_tanh")),
            "bias": rng.random() < 0.5, "residual": rng.random() < 0.5}


# ---------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _activations(g, m, d):
    """Rows of a residual stream: magnitudes differ from row to row, and a few
    columns are an order of magnitude larger than the others."""
    rows = torch.exp(0.5 * _randn(g, m, 1))
    cols = torch.where(torch.rand(d, generator=g, device="cuda") < 0.01, 12.0, 1.0)
    return _randn(g, m, d).mul_(rows).mul_(cols)


def _rows_to_fp8(x):
    """E4M3FN bytes of x (overwritten) and its row scales."""
    scale = x.abs().amax(dim=1).div_(FP8_MAX)
    return x.div_(scale[:, None]).to(torch.float8_e4m3fn).view(torch.uint8), scale


def prepare(case, seed):
    g = _gen(seed)
    m = case["M"]
    if case["op"] == "norm":
        d = case["D"]
        s = {"x": _activations(g, m, d).to(torch.bfloat16),
             "weight": _randn(g, d).mul_(0.2).add_(1.0).to(torch.bfloat16),
             "residual": _activations(g, m, d).to(torch.bfloat16) if case["residual"] else None}
    elif case["op"] == "quant":
        # a gated product's rows: heavy-tailed, many values near zero
        d = case["D"]
        s = {"x": _randn(g, m, d).mul_(_randn(g, m, d)).to(torch.bfloat16)}
    else:
        c, r = case["C"], case["R"]
        n = r // 2 if case["gated"] else r
        a, a_scale = _rows_to_fp8(_activations(g, m, c))
        w, w_scale = _rows_to_fp8(_randn(g, r, c).mul_(0.02))
        s = {"a": a, "a_scale": a_scale, "w": w, "w_scale": w_scale,
             "bias": _randn(g, r).to(torch.bfloat16) if case["bias"] else None,
             "residual": _randn(g, m, n).to(torch.bfloat16) if case["residual"] else None,
             "act": case["act"], "gated": case["gated"]}
    s["op"] = case["op"]
    return s


# -- plain forms: elementary operations in 32 bits, rounded once at the end ------


def _fp8(b):
    return b.view(torch.float8_e4m3fn).to(torch.float32)


def _plain_quant(y):
    scale = y.abs().amax(dim=1).clamp(min=AMAX_MIN) / FP8_MAX
    return [(y / scale[:, None]).to(torch.float8_e4m3fn), scale]


def _plain_act(v, act):
    if act == "relu":
        return torch.clamp(v, min=0.0)
    if act == "silu":
        return v / (1.0 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    return v


def _plain(s):
    if s["op"] == "quant":
        return _plain_quant(s["x"].to(torch.float32))
    if s["op"] == "norm":
        h = s["x"].to(torch.float32)
        if s["residual"] is not None:
            h = h + s["residual"].to(torch.float32)
        y = h * torch.rsqrt((h * h).mean(dim=1, keepdim=True) + EPS) * s["weight"].to(torch.float32)
        return [*_plain_quant(y), h.to(torch.bfloat16)]
    v = _fp8(s["a"]) @ _fp8(s["w"]).t()
    v = v * s["a_scale"][:, None] * s["w_scale"]
    if s["bias"] is not None:
        v = v + s["bias"].to(torch.float32)
    if s["gated"]:
        n = v.shape[1] // 2
        v = _plain_act(v[:, :n], s["act"]) * v[:, n:]
    else:
        v = _plain_act(v, s["act"])
    if s["residual"] is not None:
        v = v + s["residual"].to(torch.float32)
    return v.to(torch.bfloat16)


def _framework():
    path = os.path.join(_ROOT, "tans-vectoradd_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import rans_vectoradd
    return rans_vectoradd


def run(state):
    s = state
    if not own:
        return _plain(s)
    R = _framework()
    if s["op"] == "norm":
        q, scale, h = R.fp8_rmsnorm(s["x"], s["weight"], s["residual"], eps=EPS)
        return [q.view(torch.float8_e4m3fn), scale, h]
    if s["op"] == "quant":
        q, scale = R.fp8_quantize_rows(s["x"])
        return [q.view(torch.float8_e4m3fn), scale]
    return R.fp8_linear(s["a"], s["a_scale"], s["w"], s["w_scale"], bias=s["bias"],
                        activation=s["act"], residual=s["residual"], gated=s["gated"])


# ---------------------------------------------------------------------------


def work(case):
    """Bytes: inputs once, outputs once.  Operations: the product's; for the
    norm the square, sum, two products and the 8-bit division."""
    m = case["M"]
    if case["op"] == "quant":
        n = m * case["D"]
        return {"bytes": 3 * n + 4 * m, "flops": 2 * n}
    if case["op"] == "norm":
        n = m * case["D"]
        per = 7 if case["residual"] else 3   # x, q; the residual read and the sum written
        return {"bytes": per * n + 2 * case["D"] + 4 * m, "flops": 6 * n}
    c, r = case["C"], case["R"]
    n = r // 2 if case["gated"] else r
    b = m * c + r * c + 4 * m + 4 * r + 2 * m * n
    b += 2 * r if case["bias"] else 0
    b += 2 * m * n if case["residual"] else 0
    return {"bytes": b, "flops": 2 * m * r * c}


def _f64(b):
    """The values of E4M3FN bytes from the format's definition: sign, 4 exponent
    bits (bias 7), 3 mantissa bits; exponent 0 is subnormal."""
    i = torch.arange(256, dtype=torch.float64, device="cuda")
    sign = torch.where(i >= 128, -1.0, 1.0).double()
    e = torch.floor(i / 8) % 16
    f = i % 8
    mag = torch.where(e > 0, (1 + f / 8) * torch.pow(2.0, e - 7), f / 8 * 2.0 ** -6)
    return (sign * mag)[b.to(torch.int32)]


def _exact_rows(y):
    top = torch.clamp(y.abs().max(dim=1).values, min=AMAX_MIN)
    scale = top / FP8_MAX
    return [y / scale.unsqueeze(1), scale]


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "quant":
        return _exact_rows(s["x"].double())
    if s["op"] == "norm":
        h = s["x"].double()
        if s["residual"] is not None:
            h += s["residual"].double()
        rms = torch.sqrt(h.square().sum(dim=1) / case["D"] + EPS)
        return [*_exact_rows(s["weight"].double() * (h / rms.unsqueeze(1))), h]
    a = _f64(s["a"]) * s["a_scale"].double().unsqueeze(1)
    wt = (_f64(s["w"]) * s["w_scale"].double().unsqueeze(1)).t()
    v = torch.matmul(a, wt)
    del a, wt
    if s["bias"] is not None:
        v += s["bias"].double()
    up = None
    if s["gated"]:
        v, up = v.chunk(2, dim=1)
    act = s["act"]
    if act == "relu":
        v = torch.where(v > 0, v, torch.zeros_like(v))
    elif act == "silu":
        v = v * torch.sigmoid(v)
    elif act == "gelu":
        v = v * torch.special.ndtr(v)
    elif act == "gelu_tanh":
        # (1 + tanh(u)) / 2 = sigmoid(2 u)
        v = v * torch.sigmoid(math.sqrt(8.0 / math.pi) * (v + 0.044715 * v.pow(3)))
    if up is not None:
        v = v * up
    if s["residual"] is not None:
        v = v + s["residual"].double()
    return v
