"""Workloads of the 8-bit integer operators: the scaled matrix product, the root-mean-square norm with the residual's addition and an
8-bit output, and the quantisation of rows (with its way back).

Every case is a dict of plain values; `prepare` makes what a program holds before the call, `run` is one call as a program makes it
(`own`: through `dynamicscaler_amd.ops`, otherwise the plain form in elementary torch operations), `exact` the same in 64 bits.

Definitions (rows m, columns n, inner index k; rint rounds halves to even):

  product   out[m, n] = act(a_scale[m] * w_scale[n] * sum_k A[m, k] W[n, k] + bias[n]) + residual[m, n]
            act = identity, SiLU, or GEGLU: W's rows come in groups of 64 = 32 value rows, then their 32 gate rows, and
            out[m, j] = value_j * gelu(gate_j) (exact erf form), half as many columns
  norm      h = x + residual;  y = h * gamma / sqrt(mean(h^2) + eps);  out: y itself, or q = rint(127 y / max|y|) with
            scale = max|y| / 127 of each row;  the sum h goes back to the residual stream in the residual's type, the norm itself
            reads it unrounded
  quantize  scale = max|x| / 127 of each row, q = rint(127 x / max|x|)

8-bit results are returned as the values they stand for, q * scale.
"""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "f32": torch.float32}
SIZE = {"f16": 2, "f32": 4}
EPS = 1e-6

MOST_FLOPS = 2.0 * 40960 * 1280 * 10240       # the largest listed product
MOST_BYTES = 655360 * 320 * 9                 # ... and the most bytes of a listed product (its level-0 rows)
MOST_VALUES = 655360 * 320                    # values of the largest listed norm / quantisation


def _product(m, k, n, out="f16", residual=None, bias=True, act="none", lda_extra=0):
    return {"op": "product", "m": m, "k": k, "n": n, "out": out, "residual": residual, "bias": bias, "act": act, "lda_extra": lda_extra}


def _norm(m, n, x="f16", residual="f16", out="i8"):
    return {"op": "norm", "m": m, "n": n, "x": x, "residual": residual, "out": out}


def _quantize(m, n, x="f16"):
    return {"op": "quantize", "m": m, "n": n, "x": x}


def listed():
    return [
        # one token through the second layer of a time-embedding MLP: the smallest call, its latency counts
        dict(_product(1, 1280, 1280, act="silu"), name="product one token"),
        # sixteen single tokens through a feed-forward's second layer: the weights are read once for all of them
        dict(_product(16, 5120, 1280, residual="f16"), name="product sixteen tokens"),
        # one prompt through the first layer of the text tower's MLP
        dict(_product(77, 1024, 4096), name="product prompt"),
        # ragged sizes: nothing is a multiple of anything, the residual stream in 32 bits
        dict(_product(2057, 1273, 997, out="f32", residual="f32"), name="product ragged"),
        # the output projection of the highest resolution's attention (16 tile evaluations x 16 frames x 40 x 64 rows) onto the fp32
        # residual stream: short inner axis, bound by memory
        dict(_product(655360, 320, 320, out="f32", residual="f32"), name="product level 0"),
        # the GEGLU projection of the quarter resolution (16 x 16 x 10 x 16 rows): the largest product, bound by the matrix cores
        dict(_product(40960, 1280, 10240, act="geglu"), name="product geglu level 2"),
        # one token's norm in front of a product
        dict(_norm(1, 1280), name="norm one token"),
        # ragged rows, fp32 residual stream
        dict(_norm(3001, 1283, residual="f32"), name="norm ragged"),
        # every row of the highest resolution, fp32 residual stream: many short rows
        dict(_norm(655360, 320, residual="f32"), name="norm level 0"),
        # a few tokens' activations in front of the second feed-forward layer
        dict(_quantize(16, 5120), name="quantize sixteen tokens"),
        # ragged fp32 rows
        dict(_quantize(4099, 641, x="f32"), name="quantize ragged"),
        # the feed-forward's hidden rows at the quarter resolution
        dict(_quantize(40960, 5120), name="quantize level 2"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["product", "product", "norm", "quantize"])
    even = rng.random() < 0.5                  # half of the draws have whole 16s along the rows, half are odd
    rows = _log(rng, 1, 200000)

    def width(lo, hi):
        w = _log(rng, lo, hi)
        return max(16, w // 16 * 16) if even else w | 1

    if op == "product":
        k, act = width(16, 8192), rng.choice(["none", "none", "silu", "geglu"])
        n = max(64, _log(rng, 64, 10240) // 64 * 64) if act == "geglu" else width(16, 8192)
        c = _product(rows, k, n, out=rng.choice(["f16", "f32"]), residual=rng.choice([None, "f16", "f32"]) if act == "none" else None,
                     bias=rng.random() < 0.7, act=act, lda_extra=rng.choice([0, 0, 64]))
        while work(c)["flops"] > MOST_FLOPS or work(c)["bytes"] > MOST_BYTES:
            c["m"] = max(1, c["m"] * 2 // 3)
        return c
    n = width(64, 16384)
    rows = max(1, min(rows, MOST_VALUES // n))
    if op == "norm":
        return _norm(rows, n, x=rng.choice(["f16", "f16", "f32"]), residual=rng.choice([None, "f16", "f32"]), out=rng.choice(["i8", "i8", "f16", "f32"]))
    return _quantize(rows, n, x=rng.choice(["f16", "f16", "f32"]))


def _columns(case):
    return case["n"] // 2 if case["act"] == "geglu" else case["n"]


def work(case):
    m, n = case["m"], case["n"]
    if case["op"] == "product":
        k, cols = case["k"], _columns(case)
        held = m * k + n * k + 4 * (m + n) + (4 * n if case["bias"] else 0) + m * cols * (SIZE[case["out"]] + SIZE.get(case["residual"], 0))
        return {"bytes": held, "flops": 2 * m * n * k}
    if case["op"] == "norm":                   # x and the residual in, the sum and the result (8-bit ones as their values) out
        out = {"i8": 2 * m * n + 4 * m, "f16": 2 * m * n, "f32": 4 * m * n}[case["out"]]
        return {"bytes": m * n * (SIZE[case["x"]] + 2 * SIZE.get(case["residual"], 0)) + 4 * n + out, "flops": 8 * m * n}
    return {"bytes": 2 * m * n * SIZE[case["x"]] + 4 * m, "flops": 4 * m * n}


def _rows_i8(shape, gen, dev):
    """8-bit rows as a quantisation of normal values leaves them (the largest of a row is +-127), and their scales."""
    v = torch.randn(shape, generator=gen, device=dev)
    top = v.abs().amax(dim=1, keepdim=True)
    return torch.round(v * (127.0 / top)).to(torch.int8), (top[:, 0] / 127.0)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    m, n = case["m"], case["n"]

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(shape, generator=gen, device=dev) * scale).to(dtype)

    s = {"case": dict(case)}
    if case["op"] == "product":
        k, pad = case["k"], case["lda_extra"]
        a, s["a_scale"] = _rows_i8((m, k), gen, dev)
        if pad:                                # a column slice of a wider matrix, as a fused projection's result gives it
            wide = torch.zeros((m, k + pad), dtype=torch.int8, device=dev)
            wide[:, :k] = a
            a = wide[:, :k]
        s["a"] = a
        s["w"], w_scale = _rows_i8((n, k), gen, dev)
        s["w_scale"] = w_scale / math.sqrt(k)  # results of order one, as trained projections give
        s["bias"] = normal(n, scale=0.1) if case["bias"] else None
        s["residual"] = normal(m, _columns(case), dtype=DTYPES[case["residual"]]) if case["residual"] else None
        return s
    channel = torch.exp(normal(n, scale=0.7))  # a few channels are several times larger than the others, as in trained streams
    x = normal(m, n)
    x *= channel
    s["x"] = x.to(DTYPES[case["x"]])
    if case["op"] == "norm":
        s["gamma"] = 1.0 + normal(n, scale=0.2)
        s["residual"] = normal(m, n, dtype=DTYPES[case["residual"]], scale=2.0) if case["residual"] else None
    return s


# ------------------------------------------------------------------------------------------------ the framework's calls
def _run_own(s):
    from dynamicscaler_amd import ops
    from dynamicscaler_amd._lib import DS_EPI_GEGLU, DS_EPI_SILU
    c = s["case"]
    if c["op"] == "product":
        act = {"none": 0, "silu": DS_EPI_SILU, "geglu": DS_EPI_GEGLU}[c["act"]]
        return ops.gemm_i8(s["a"], s["w"], s["a_scale"], s["w_scale"], bias=s["bias"], residual=s["residual"], epilogue=act,
                           out_dtype=DTYPES[c["out"]])
    if c["op"] == "norm":
        if c["out"] == "i8":
            q, scale, h = ops.rmsnorm_i8(s["x"], s["gamma"], eps=EPS, residual=s["residual"])
            return {"values": ops.dequantize_rows_i8(q, scale, dtype=torch.float16), "scale": scale, "sum": h}
        y, h = ops.rmsnorm(s["x"], s["gamma"], eps=EPS, residual=s["residual"], out_dtype=DTYPES[c["out"]])
        return {"values": y, "sum": h}
    q, scale = ops.quantize_rows_i8(s["x"])
    return {"values": ops.dequantize_rows_i8(q, scale, dtype=DTYPES[c["x"]]), "scale": scale}


# ------------------------------------------------------------------------------------------------ the plain form
def _quantized(t, root):
    """Values and scales of rows `t` (root: a factor of each row's scale).  The quotient is formed in the type of `t`."""
    top = t.abs().amax(dim=1, keepdim=True)
    q = torch.round(torch.where(top > 0, 127 * t / top, torch.zeros_like(t)))
    scale = top * root / 127
    return q * scale, scale[:, 0]


def _run_plain(s):
    c = s["case"]
    if c["op"] == "product":
        v = s["a"].float() @ s["w"].float().t()
        v = v * s["a_scale"][:, None] * s["w_scale"]
        if s["bias"] is not None:
            v = v + s["bias"]
        if c["act"] == "silu":
            v = v / (1 + torch.exp(-v))
        elif c["act"] == "geglu":
            v = v.view(c["m"], c["n"] // 64, 2, 32)
            gate = v[:, :, 1]
            v = (v[:, :, 0] * (0.5 * gate * (1 + torch.erf(gate * math.sqrt(0.5))))).reshape(c["m"], c["n"] // 2)
        if s["residual"] is not None:
            v = v + s["residual"].float()
        return v.to(DTYPES[c["out"]])
    # 8-bit roundings: in 64 bits, since 32 put values that lie next to the middle of two steps on the wrong side; fp16 rows without a
    # sum or a product before the rounding are exact in 32
    if c["op"] == "norm":
        t = torch.float64 if c["out"] == "i8" else torch.float32
        h = s["x"].to(t)
        if s["residual"] is not None:
            h = h + s["residual"]
        root = torch.rsqrt((h * h).mean(dim=1, keepdim=True) + EPS)
        back = h.to(DTYPES[c["residual"]]) if c["residual"] else None
        if c["out"] == "i8":
            values, scale = _quantized(h * s["gamma"], root)
            return {"values": values.to(torch.float16), "scale": scale.to(torch.float32), "sum": back}
        return {"values": (h * root * s["gamma"]).to(DTYPES[c["out"]]), "sum": back}
    x = s["x"].double() if c["x"] == "f32" else s["x"].float()
    values, scale = _quantized(x, 1.0)
    return {"values": values.to(s["x"].dtype), "scale": scale.to(torch.float32)}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------------------ 64 bits, from the definitions above
def _exact_rows_i8(t):
    """q of rows t, and max|t| of each row."""
    top, _ = torch.max(torch.abs(t), dim=1)
    ratio = torch.div(t * 127.0, torch.clamp(top, min=torch.finfo(torch.float64).tiny)[:, None])
    return torch.round(ratio), top


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "product":
        rows, parts = max(1, (1 << 28) // case["n"]), []
        w = torch.mul(s["w"].to(torch.float64), s["w_scale"].to(torch.float64)[:, None]).t().contiguous()
        for at in range(0, case["m"], rows):
            u = torch.mul(s["a"][at:at + rows].to(torch.float64), s["a_scale"][at:at + rows].to(torch.float64)[:, None])
            z = torch.matmul(u, w)
            if s["bias"] is not None:
                z += s["bias"].to(torch.float64)
            if case["act"] == "silu":
                z *= torch.sigmoid(z)
            elif case["act"] == "geglu":
                pair = z.unflatten(1, (-1, 64))
                value, gate = pair[..., :32], pair[..., 32:]
                z = (value * gate * torch.erfc(gate / -math.sqrt(2.0)) / 2).flatten(1)
            if s["residual"] is not None:
                z += s["residual"][at:at + rows].to(torch.float64)
            parts.append(z)
        return torch.cat(parts)
    h = s["x"].to(torch.float64)
    if case["op"] == "quantize":
        q, top = _exact_rows_i8(h)
        return {"values": q * (top / 127.0)[:, None], "scale": top / 127.0}
    back = None
    if s["residual"] is not None:
        h = torch.add(h, s["residual"].to(torch.float64))
        back = h
    length = torch.sqrt(torch.linalg.vector_norm(h, dim=1) ** 2 / case["n"] + EPS)
    if case["out"] == "i8":
        q, top = _exact_rows_i8(h * s["gamma"].to(torch.float64))
        scale = top / length / 127.0
        return {"values": q * scale[:, None], "scale": scale, "sum": back}
    return {"values": h * s["gamma"].to(torch.float64) / length[:, None], "sum": back}
