"""The 8-bit projection path: RMS norm with the residual's addition, rows to 8 bits, the product of 8-bit rows.

A decoder layer's projections with 8-bit weights and activations: the hidden state is normed and quantised a row (token)
at a time, the weights were quantised a row (output channel) at a time, the product of the two runs in integers and is
scaled back.  ``op`` says which operator a case is:

* ``norm``    ``add_rms_norm``: s = x + residual, y = s * rsqrt(mean(s^2) + eps) * weight; y comes in the input's type or
              in 8 bits with a scale for each row, s in the input's type
* ``quant``   ``quantize_int8``: a row's scale is its largest magnitude over 127, its values are rounded to multiples of it
* ``linear``  ``int8_linear``: the integer product, times the token's scale, times the channel's, plus bias, plus residual

Rows held in 8 bits are returned as the values they stand for, in bfloat16 (a value has seven bits and a sign; what the
scale has beyond that is returned with the scales, which are float32).

Hidden states are Gaussian with channels of different spread, as trained models have them; norm weights lie around one.
The shapes are those of this repository's benchmark and tests (embed 512, 576, 4096, 8192), rows are tokens: one for each
state of a decode step, states times tokens for a chunk of a prefill.
"""
import math
import os
import sys

import torch

own = False

EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    def norm(name, rows, dim, dtype="bf16", residual=True, int8=True):
        return dict(name=name, op="norm", rows=rows, dim=dim, dtype=dtype, residual=residual, int8=int8)

    def quant(name, rows, dim, dtype="bf16"):
        return dict(name=name, op="quant", rows=rows, dim=dim, dtype=dtype)

    def linear(name, rows, k, n, dtype="bf16", bias=False, residual=False):
        return dict(name=name, op="linear", rows=rows, k=k, n=n, dtype=dtype, bias=bias, residual=residual)

    return [
        # the smallest call: one sequence, one token, the small layer
        norm("norm_int8_b1_d512", 1, 512),
        # a decode step's rows in front of the input projection, 32 states of the 7B shape
        norm("norm_int8_b32_d4096", 32, 4096),
        # single precision without 8 bits, rows that start on no vector boundary
        norm("norm_f32_2047x577", 2047, 577, dtype="f32", int8=False),
        # a chunk of 512 tokens for 32 states of the 7B shape
        norm("norm_int8_prefill_d4096", 16384, 4096),
        # a decode step's heads in front of the output projection, 64 states of the 70B shape
        quant("quant_b64_d8192", 64, 8192),
        # the heads of a prefill chunk
        quant("quant_prefill_d4096", 16384, 4096),
        # the smallest call: the fused input projection of the small layer for one token
        linear("linear_in_b1_d512", 1, 512, 777, bias=True),
        # the fused input projection of the 7B shape for a decode step (the width is odd)
        linear("linear_in_b32_d4096", 32, 4096, 6177, bias=True),
        # the output projection of the 70B shape for an odd number of states, the residual in its epilogue
        linear("linear_out_b100_d8192", 100, 8192, 8192, residual=True),
        # the input projection of a small single-precision layer over a ragged prompt
        linear("linear_in_2047_d576_f32", 2047, 576, 970, dtype="f32", bias=True),
        # the input projection of the 7B shape over a prefill chunk
        linear("linear_in_prefill_d4096", 16384, 4096, 6177, bias=True),
        # the output projection of the 70B shape over a prefill chunk
        linear("linear_out_prefill_d8192", 8192, 8192, 8192, residual=True),
    ]


def draw(rng):
    def span(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    def width(lo, hi):      # half of the widths are multiples of 64, as in most models
        n = span(lo, hi)
        return max(64, n // 64 * 64) if rng.random() < 0.5 else n

    op = rng.choice(("norm", "quant", "linear"))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    rows = span(1, 16384)
    if op == "linear":
        k, n = width(64, 8192), width(64, 8192)
        rows = min(rows, 8192 ** 3 // (k * n))
        return dict(op=op, rows=rows, k=k, n=n, dtype=dtype, bias=rng.random() < 0.5, residual=rng.random() < 0.5)
    dim = width(64, 8192)
    rows = max(1, min(rows, 16384 * 4096 // (dim * (2 if dtype == "f32" else 1))))
    if op == "quant":
        return dict(op=op, rows=rows, dim=dim, dtype=dtype)
    return dict(op=op, rows=rows, dim=dim, dtype=dtype, residual=rng.random() < 0.7, int8=rng.random() < 0.7)


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _hidden(gen, rows, dim, dtype):
    """Hidden states: Gaussian, each channel with its own spread."""
    return (_randn(gen, rows, dim) * torch.exp(0.5 * _randn(gen, dim))).to(TYPES[dtype])


def _rows_of_int8(gen, rows, k):
    """8-bit rows as a quantised Gaussian has them, each row's largest value at 127; rows start every 16 bytes."""
    x = _randn(gen, rows, k)
    x *= 127.0 / x.abs().amax(1, keepdim=True)
    values = torch.zeros(rows, (k + 15) // 16 * 16, device="cuda", dtype=torch.int8)[:, :k]
    values.copy_(x.round_())
    return values, 0.01 + 0.02 * torch.rand(rows, generator=gen, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if case["op"] == "linear":
        dt = TYPES[case["dtype"]]
        s["x"], s["x_scale"] = _rows_of_int8(gen, case["rows"], case["k"])
        s["w"], s["w_scale"] = _rows_of_int8(gen, case["n"], case["k"])
        s["w_scale"] *= 1.0 / math.sqrt(case["k"])
        s["b"] = _randn(gen, case["n"]).to(dt) if case["bias"] else None
        s["r"] = _randn(gen, case["rows"], case["n"]).to(dt) if case["residual"] else None
        return s
    s["x"] = _hidden(gen, case["rows"], case["dim"], case["dtype"])
    if case["op"] == "norm":
        s["w"] = (1.0 + 0.1 * _randn(gen, case["dim"])).to(TYPES[case["dtype"]])
        s["r"] = _hidden(gen, case["rows"], case["dim"], case["dtype"]) if case["residual"] else None
    return s


def run(state):
    return _own(state) if own else _plain(state)


# ---- the framework's calls ---------------------------------------------------------------------
def _own(s):
    package = os.path.join(os.getcwd(), "coda-gqa-l_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    from coda_gqa_l_b200 import Int8Rows, add_rms_norm, int8_linear, quantize_int8

    if s["op"] == "norm":
        y, h = add_rms_norm(s["x"], s["w"], residual=s["r"], eps=EPS, int8=s["int8"])
        out = {"values": y.dequantize(torch.bfloat16), "scale": y.scale} if s["int8"] else {"y": y}
        return {**out, "h": h} if s["residual"] else out
    if s["op"] == "quant":
        q = quantize_int8(s["x"])
        return {"values": q.dequantize(torch.bfloat16), "scale": q.scale}
    return int8_linear(Int8Rows(s["x"], s["x_scale"]), Int8Rows(s["w"], s["w_scale"]), s["b"], residual=s["r"],
                       dtype=TYPES[s["dtype"]])


# ---- the plain forms ----------------------------------------------------------------------------
def _to_8_bits_and_back(y):
    scale = y.abs().amax(1) / 127.0
    q = torch.round(y / scale[:, None])
    return {"values": (q * scale[:, None]).to(torch.bfloat16), "scale": scale}


def _plain(s):
    if s["op"] == "quant":
        return _to_8_bits_and_back(s["x"].float())
    if s["op"] == "norm":
        h = s["x"].float() if s["r"] is None else s["x"].float() + s["r"].float()
        y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * s["w"].float()
        out = _to_8_bits_and_back(y) if s["int8"] else {"y": y.to(s["x"].dtype)}
        return {**out, "h": h.to(s["x"].dtype)} if s["residual"] else out
    # a product of 8-bit values has 14 bits and the sums of these distributions stay under 2^24: exact in float32
    y = (s["x"].float() @ s["w"].float().t()) * s["x_scale"][:, None] * s["w_scale"]
    if s["b"] is not None:
        y = y + s["b"].float()
    if s["r"] is not None:
        y = y + s["r"].float()
    return y.to(TYPES[s["dtype"]])


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "linear":
        m, n, k = case["rows"], case["n"], case["k"]
        return {"bytes": m * k + n * k + 4 * (m + n) + e * m * n * (2 if case["residual"] else 1) + (e * n if case["bias"] else 0),
                "flops": 2.0 * m * n * k}
    n = case["rows"] * case["dim"]
    if case["op"] == "quant":
        return {"bytes": n * (e + 2) + 4 * case["rows"], "flops": 4.0 * n}
    out = 2 * n + 4 * case["rows"] if case["int8"] else e * n
    return {"bytes": n * e * (3 if case["residual"] else 1) + e * case["dim"] + out, "flops": 8.0 * n}


# ---- the definitions in 64 bits -------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)

    def held(rows):          # multiples of a 127th of the row's largest magnitude
        step = rows.abs().max(dim=1, keepdim=True).values.div(127)
        return {"values": rows.div(step).round().mul(step), "scale": step.squeeze(1)}

    if case["op"] == "linear":
        acc = torch.matmul(s["x"].double(), s["w"].double().transpose(0, 1))
        acc *= torch.outer(s["x_scale"].double(), s["w_scale"].double())
        for extra in (s["b"], s["r"]):
            if extra is not None:
                acc += extra.double()
        return acc
    x = s["x"].double()
    if case["op"] == "quant":
        return held(x)
    if case["residual"]:
        x = x.add(s["r"].double())
    length = x.square().sum(dim=1, keepdim=True).div(case["dim"]).add(EPS).sqrt()
    y = x.div(length).mul(s["w"].double())
    out = held(y) if case["int8"] else {"y": y}
    if case["residual"]:
        out["h"] = x
    return out
