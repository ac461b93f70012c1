"""Cases for timing the operators of serving in 8 bits: rows and weights turned into e4m3 with a scale for each block of
128, the RMS norm that leaves its rows so, and the linear map that takes both so.

``own`` False computes them in their plain form, elementary torch operations in 32 bits; ``own`` True makes the calls
that a user makes of ``ccq_amd``.  A case is a dict of plain values:

  op      "quantize" quantize_fp8    "norm" rms_norm_fp8    "linear" fp8_linear
  quantize: rows, D, dtype of the rows
  norm:     rows, D, dtype of the rows and the stream, wdtype of the weight, residual (the block's residual stream is
            added and returned)
  linear:   M, K, N (outputs), act, bias, residual, dtype of the output and of bias and residual, or "fp8": the output
            is in 8 bits with scales again, for the next map

Rows in 8 bits are a pair: values (e4m3) and scales (e8m0, powers of two), one of 128 consecutive elements of a row.
"""

import math

import torch

own = False

DEV = "cuda"
EPS = 1e-5
BLOCK = 128
MOST = 448.0  # largest number of e4m3


def listed():
    return [
        # One token of sixteen sequences: the norm ahead of a decode step's projections. Latency.
        dict(name="norm_decode", op="norm", rows=16, D=1024, dtype="bfloat16", wdtype="bfloat16", residual=True),
        # A block's norm over a long prompt with the residual stream added in it (8 sequences of 4096 tokens).
        dict(name="norm_prompt", op="norm", rows=32768, D=1024, dtype="bfloat16", wdtype="bfloat16", residual=True),
        # A small model kept in 32 bits with an odd width: rows that no wide load fits, a last block that is not whole.
        dict(name="norm_odd", op="norm", rows=1531, D=777, dtype="float32", wdtype="float32", residual=True),
        # The mixers' outputs of a prompt ahead of their projection (4 sequences of 4096 tokens).
        dict(name="quantize_rows", op="quantize", rows=16384, D=2048, dtype="bfloat16"),
        # A head's weight in 32 bits, once, when a model is loaded.
        dict(name="quantize_weight", op="quantize", rows=32000, D=1024, dtype="float32"),
        # One token of sixteen sequences through a gated MLP's up projection, on to the next. Latency.
        dict(name="linear_decode", op="linear", M=16, K=1024, N=2816, act="swiglu", bias=False, residual=False, dtype="fp8"),
        # One token of one sequence through the head, logits in 32 bits: the weight's bytes.
        dict(name="linear_head", op="linear", M=1, K=1024, N=32000, act="", bias=False, residual=False, dtype="float32"),
        # A decode step of a large batch, the output projection with the residual stream.
        dict(name="linear_batch", op="linear", M=256, K=2048, N=1024, act="", bias=False, residual=True, dtype="bfloat16"),
        # The gated MLP's up projection of a prompt (4 sequences of 4096 tokens), on to the next.
        dict(name="linear_up_prompt", op="linear", M=16384, K=1024, N=2816, act="swiglu", bias=False, residual=False,
             dtype="fp8"),
        # Its down projection over a longer prompt, with the residual stream added.
        dict(name="linear_down_prompt", op="linear", M=32768, K=2816, N=1024, act="", bias=False, residual=True,
             dtype="bfloat16"),
        # A classical MLP on a ragged batch in half precision: odd rows, odd widths.
        dict(name="linear_odd", op="linear", M=1531, K=1000, N=777, act="gelu", bias=True, residual=False, dtype="float16"),
        # A large square map: the matrix cores.
        dict(name="linear_large", op="linear", M=8192, K=8192, N=8192, act="", bias=False, residual=False, dtype="bfloat16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "quantize", "linear", "linear"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if op != "linear":
        D = _log(rng, 32, 8192)
        if rng.random() < 0.5:
            D = -(-D // 32) * 32
        rows = min(_log(rng, 1, 65536), 32768 * 2048 // D)
        if op == "quantize":
            return dict(op=op, rows=rows, D=D, dtype=dtype)
        return dict(op=op, rows=rows, D=D, dtype=dtype, wdtype=rng.choice([dtype, "float32"]), residual=rng.random() < 0.5)
    K, N = _log(rng, 32, 8192), _log(rng, 16, 8192)
    if rng.random() < 0.6:
        K, N = -(-K // 32) * 32, -(-N // 32) * 32
    act = rng.choice(["", "relu", "silu", "gelu", "gelu_tanh", "swiglu"])
    outs = 2 * N if act == "swiglu" else N
    M = min(_log(rng, 1, 32768), 8192 ** 3 // 2 // (K * outs))
    dtype = rng.choice([dtype, "fp8"])
    return dict(op=op, M=M, K=K, N=N, act=act, bias=rng.random() < 0.5, residual=dtype != "fp8" and rng.random() < 0.4,
                dtype=dtype)


# ---- inputs ----------------------------------------------------------------------------------------------------

def _blocks(t):
    """[rows, D] as [rows, blocks, 128], zeros behind D."""
    rows, D = t.shape
    n = -(-D // BLOCK)
    return torch.nn.functional.pad(t, (0, n * BLOCK - D)).view(rows, n, BLOCK)


def _quantized(t):
    """Rows in 32 bits as (values, scales): the least power of two that brings a block's largest within e4m3."""
    rows, D = t.shape
    b = _blocks(t)
    m, e = torch.frexp(b.abs().amax(-1, keepdim=True))
    e = (e - torch.where(m <= 0.875, 9, 8)).clamp_min(-126)  # 448 = 0.875 * 2^9
    e = torch.where(m == 0, -126, e).int()
    scale = ((e + 127) << 23).view(torch.float32)
    values = (b / scale).view(rows, -1)[:, :D].to(torch.float8_e4m3fn)
    return values, scale[..., 0].to(torch.float8_e8m0fnu)


def _kept(pair):
    """The pair as a program keeps it: rows from multiples of 16 bytes on, their scales from multiples of 4."""
    out = []
    for t, n in zip(pair, (16, 4)):
        rows, D = t.shape
        room = torch.zeros(rows, -(-D // n) * n, dtype=torch.uint8, device=t.device)
        room[:, :D] = t.view(torch.uint8)
        out.append(room.view(t.dtype)[:, :D])
    return tuple(out)


def _rows(rnd, R, D):
    # a residual stream: channels of different scale and a common offset, as trained blocks have them
    return rnd(R, D) * torch.exp(0.5 * rnd(D)) + 0.3


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def rnd(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)

    x = {}
    if c["op"] == "linear":
        M, K, N = c["M"], c["K"], c["N"]
        outs = 2 * N if c["act"] == "swiglu" else N
        rest = torch.bfloat16 if c["dtype"] == "fp8" else getattr(torch, c["dtype"])
        x["x"] = _kept(_quantized(rnd(M, K) * torch.exp(0.5 * rnd(K))))
        x["weight"] = _kept(_quantized(rnd(outs, K) / math.sqrt(K)))
        if c["bias"]:
            x["bias"] = (0.1 * rnd(outs)).to(rest)
        if c["residual"]:
            x["residual"] = rnd(M, N).to(rest)
        return {"case": dict(c), "x": x}
    dtype = getattr(torch, c["dtype"])
    if c["op"] == "quantize":
        x["x"] = _rows(rnd, c["rows"], c["D"]).to(dtype)
        return {"case": dict(c), "x": x}
    x["x"] = _rows(rnd, c["rows"], c["D"]).to(dtype)
    x["weight"] = (1 + 0.1 * rnd(c["D"])).to(getattr(torch, c["wdtype"]))
    if c["residual"]:
        x["residual"] = (0.5 * rnd(c["rows"], c["D"])).to(dtype)
    return {"case": dict(c), "x": x}


# ---- the plain forms -------------------------------------------------------------------------------------------

def _plain_quantize(c, x):
    values, scales = _quantized(x["x"].float())
    return {"values": values, "scales": scales}


def _plain_norm(c, x):
    s = x["x"]
    if c["residual"]:
        s = (s.float() + x["residual"].float()).to(s.dtype)  # the stream as the next block reads it
    f = s.float()
    y = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + EPS) * x["weight"].float()
    values, scales = _quantized(y)
    out = {"values": values, "scales": scales}
    if c["residual"]:
        out["s"] = s
    return out


def _meant(pair):
    """The numbers that a pair stands for, in 32 bits."""
    values, scales = pair
    return values.float() * scales.float().repeat_interleave(BLOCK, 1)[:, :values.shape[1]]


def _plain_act(act, z):
    if act == "relu":
        return z.clamp_min(0)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return z * 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "swiglu":
        gate, up = z.chunk(2, -1)
        return gate * torch.sigmoid(gate) * up
    return z


def _plain_linear(c, x):
    z = _meant(x["x"]) @ _meant(x["weight"]).T
    if c["bias"]:
        z = z + x["bias"].float()
    y = _plain_act(c["act"], z)
    if c["residual"]:
        y = y + x["residual"].float()
    if c["dtype"] != "fp8":
        return {"y": y.to(getattr(torch, c["dtype"]))}
    values, scales = _quantized(y)
    return {"values": values, "scales": scales}


# ---- the framework's calls -------------------------------------------------------------------------------------

def _own_quantize(c, x):
    from ccq_amd import quantize_fp8
    q = quantize_fp8(x["x"])
    return {"values": q.values, "scales": q.scales}


def _own_norm(c, x):
    from ccq_amd import rms_norm_fp8
    if c["residual"]:
        y, s = rms_norm_fp8(x["x"], x["weight"], eps=EPS, residual=x["residual"])
        return {"values": y.values, "scales": y.scales, "s": s}
    y = rms_norm_fp8(x["x"], x["weight"], eps=EPS)
    return {"values": y.values, "scales": y.scales}


def _own_linear(c, x):
    from ccq_amd import Fp8Rows, fp8_linear
    a, w = Fp8Rows(*x["x"]), Fp8Rows(*x["weight"])
    if c["dtype"] == "fp8":
        y = fp8_linear(a, w, x.get("bias"), activation=c["act"] or None, quantize=True)
        return {"values": y.values, "scales": y.scales}
    return {"y": fp8_linear(a, w, x.get("bias"), activation=c["act"] or None, residual=x.get("residual"),
                            dtype=getattr(torch, c["dtype"]))}


def run(state):
    c, x = state["case"], state["x"]
    with torch.no_grad():
        if own:
            return {"linear": _own_linear, "norm": _own_norm, "quantize": _own_quantize}[c["op"]](c, x)
        return {"linear": _plain_linear, "norm": _plain_norm, "quantize": _plain_quantize}[c["op"]](c, x)


# ---- what a pass cannot do without -----------------------------------------------------------------------------

def _size(dtype):
    return {"fp8": 1, "float32": 4}.get(dtype, 2)


def work(case):
    c = case
    if c["op"] == "linear":
        M, K, N = c["M"], c["K"], c["N"]
        outs = 2 * N if c["act"] == "swiglu" else N
        rest = 2 if c["dtype"] == "fp8" else _size(c["dtype"])
        n = (M + outs) * (K + -(-K // BLOCK)) + M * N * _size(c["dtype"])
        n += (outs * rest if c["bias"] else 0) + (M * N * rest if c["residual"] else 0)
        n += M * -(-N // BLOCK) if c["dtype"] == "fp8" else 0
        return {"bytes": n, "flops": 2 * M * outs * K}
    R, D, size = c["rows"], c["D"], _size(c["dtype"])
    n = R * D * size + R * (D + -(-D // BLOCK))
    if c["op"] == "quantize":
        return {"bytes": n, "flops": 4 * R * D}
    n += (2 * R * D * size if c["residual"] else 0) + D * _size(c["wdtype"])
    return {"bytes": n, "flops": 10 * R * D}


# ---- the operators' definitions in 64 bits ---------------------------------------------------------------------

def _exact_quantize(y):
    """Rows in 64 bits: the values and scales that the format's definition gives."""
    rows, D = y.shape
    n = (D + BLOCK - 1) // BLOCK
    values, scales = torch.empty_like(y), torch.empty(rows, n, dtype=torch.float64, device=y.device)
    for b in range(n):
        part = y[:, b * BLOCK:(b + 1) * BLOCK]
        e = torch.ceil(torch.log2(part.abs().max(-1).values / MOST))
        for near in (-1.0, 0.0):  # a logarithm next to a whole number may fall on its other side
            e = torch.where(part.abs().max(-1).values <= MOST * torch.exp2(e + near), e + near, e)
        e = torch.where(part.abs().max(-1).values > MOST * torch.exp2(e), e + 1, e).clamp_min(-126.0)
        scales[:, b] = torch.exp2(e)
        v = part / scales[:, b:b + 1]
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)  # 3 bits behind the first one
        values[:, b * BLOCK:(b + 1) * BLOCK] = torch.round(v / step) * step
    return {"values": values, "scales": scales}


def _exact_norm(c, x):
    s = x["x"].double()
    if c["residual"]:
        s = (s + x["residual"].double()).to(x["x"].dtype).double()
    sigma = torch.sqrt(s.square().sum(-1, keepdim=True) / s.shape[-1] + EPS)
    out = _exact_quantize(s / sigma * x["weight"].double())
    if c["residual"]:
        out["s"] = s
    return out


def _exact_rows(pair):
    values, scales = pair
    at = torch.arange(values.shape[1], device=values.device) // BLOCK
    return values.double() * scales.double()[:, at]


def _exact_act(act, z):
    if act == "relu":
        return torch.where(z > 0, z, 0.0)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return z * 0.5 * torch.special.erfc(-z / math.sqrt(2))
    if act == "gelu_tanh":
        return z / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))  # (1 + tanh v) / 2
    if act == "swiglu":
        half = z.shape[-1] // 2
        return z[:, :half] / (1 + torch.exp(-z[:, :half])) * z[:, half:]
    return z


def _exact_linear(c, x):
    z = torch.nn.functional.linear(_exact_rows(x["x"]), _exact_rows(x["weight"]),
                                   x["bias"].double() if c["bias"] else None)
    y = _exact_act(c["act"], z)
    if c["residual"]:
        y = y + x["residual"].double()
    return _exact_quantize(y) if c["dtype"] == "fp8" else {"y": y}


def exact(case, seed):
    x = prepare(case, seed)["x"]
    with torch.no_grad():
        if case["op"] == "quantize":
            return _exact_quantize(x["x"].double())
        return (_exact_linear if case["op"] == "linear" else _exact_norm)(case, x)
