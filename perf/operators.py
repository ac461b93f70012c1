"""Cases for timing the operators around the token mixers: the block norms, the projections with their epilogues,
and the log probabilities of given tokens, each forward alone (serving, scoring) and forward with gradients.

``own`` False computes them in their plain form, elementary torch operations in 32 bits; ``own`` True makes the calls
that a user makes of ``ccq_amd``.  A case is a dict of plain values:

  op      "layer" layer_norm    "rms" rms_norm    "linear" fused_linear    "logprobs" token_logprobs
  train   forward and the gradients of every input (True), or the forward alone (False)
  dtype   type of activations and matrices (norms: weights in ``wdtype``)
  norms:    rows, D, residual (the block's residual stream is added and returned)
  linear:   M, K, N (outputs), act, bias, residual
  logprobs: rows, V, top (alternatives a row), ignored (share of rows without a token), pad (entries at the end
            of the vocabulary that are masked with -inf)
"""

import math

import torch

own = False

DEV = "cuda"
EPS = 1e-5
IGNORE = -100


def listed():
    return [
        # One token of sixteen sequences: the norm ahead of a decode step's projections. Latency.
        dict(name="rms_decode", op="rms", train=False, rows=16, D=1024, dtype="bfloat16", wdtype="bfloat16",
             residual=True),
        # A block's norm in training with the residual stream added in it (8 sequences of 4096 tokens).
        dict(name="rms_train", op="rms", train=True, rows=32768, D=1024, dtype="bfloat16", wdtype="bfloat16",
             residual=True),
        # Layer norm in training at the layers' default width, weights kept in 32 bits.
        dict(name="layer_train", op="layer", train=True, rows=32768, D=2048, dtype="bfloat16", wdtype="float32",
             residual=False),
        # A small experiment in 32 bits with an odd width: rows that no wide load fits.
        dict(name="layer_odd", op="layer", train=True, rows=1531, D=777, dtype="float32", wdtype="float32",
             residual=True),
        # One token of sixteen sequences through a gated MLP's up projection. Latency, and the weight's bytes.
        dict(name="linear_decode", op="linear", train=False, M=16, K=1024, N=2816, dtype="bfloat16", act="swiglu",
             bias=False, residual=False),
        # The gated MLP's up projection of a training step (4 sequences of 4096 tokens).
        dict(name="linear_up_train", op="linear", train=True, M=16384, K=1024, N=2816, dtype="bfloat16",
             act="swiglu", bias=False, residual=False),
        # Its down projection over a long prompt, with the residual stream added.
        dict(name="linear_down_prompt", op="linear", train=False, M=32768, K=2816, N=1024, dtype="bfloat16", act="",
             bias=False, residual=True),
        # Fine-tuning a classical MLP on a ragged batch in half precision: odd rows, odd widths.
        dict(name="linear_odd", op="linear", train=True, M=1531, K=1000, N=777, dtype="float16", act="gelu",
             bias=True, residual=False),
        # Sampling: one position of sixteen sequences, the chosen tokens' log probabilities and 20 alternatives.
        dict(name="logprobs_decode", op="logprobs", train=False, rows=16, V=32000, dtype="bfloat16", top=20,
             ignored=0.0, pad=0),
        # Training on 4 sequences of 4096 tokens: the loss and the entropy with the logits' gradient.
        dict(name="logprobs_train", op="logprobs", train=True, rows=16384, V=32000, dtype="bfloat16", top=0,
             ignored=0.05, pad=0),
        # Scoring an answer under its prompt, in 32 bits: odd vocabulary with masked padding, half the rows prompt.
        dict(name="logprobs_score", op="logprobs", train=False, rows=1531, V=32007, dtype="float32", top=5,
             ignored=0.5, pad=7),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["layer", "rms", "linear", "logprobs"])
    train = rng.random() < 0.5
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if op in ("layer", "rms"):
        D = _log(rng, 32, 8192)
        if rng.random() < 0.5:
            D = -(-D // 32) * 32
        rows = min(_log(rng, 1, 65536), 32768 * 2048 // D)
        return dict(op=op, train=train, rows=rows, D=D, dtype=dtype, wdtype=rng.choice([dtype, "float32"]),
                    residual=rng.random() < 0.5)
    if op == "linear":
        K, N = _log(rng, 32, 4096), _log(rng, 16, 4096)
        if rng.random() < 0.6:
            K, N = -(-K // 32) * 32, -(-N // 32) * 32
        act = rng.choice(["", "relu", "silu", "gelu", "gelu_tanh", "swiglu"])
        outs = 2 * N if act == "swiglu" else N
        M = min(_log(rng, 1, 32768), 16384 * 1024 * 5632 // (K * outs))
        return dict(op=op, train=train, M=M, K=K, N=N, dtype=rng.choice(["bfloat16", "float16"]), act=act,
                    bias=rng.random() < 0.5, residual=rng.random() < 0.4)
    V = _log(rng, 500, 160000)
    if rng.random() < 0.5:
        V = -(-V // 64) * 64
    rows = max(1, min(_log(rng, 1, 16384), 16384 * 16000 // V))
    return dict(op=op, train=train, rows=rows, V=V, dtype=dtype, top=0 if train else rng.choice([0, 1, 5, 20, 32]),
                ignored=rng.choice([0.0, 0.05, 0.5]), pad=rng.choice([0, 0, 7]))


def _norm_inputs(c, rnd, dtype):
    R, D = c["rows"], c["D"]
    wdtype = getattr(torch, c["wdtype"])
    # a residual stream: channels of different scale and a common offset, as trained blocks have them
    scale = torch.exp(0.5 * rnd(D))
    x = {"x": (rnd(R, D) * scale + 0.3).to(dtype), "weight": (1 + 0.1 * rnd(D)).to(wdtype)}
    if c["op"] == "layer":
        x["bias"] = (0.1 * rnd(D)).to(wdtype)
    if c["residual"]:
        x["residual"] = (0.5 * rnd(R, D)).to(dtype)
    if c["train"]:
        x["dy"] = rnd(R, D).to(dtype)
        if c["residual"]:
            x["ds"] = rnd(R, D).to(dtype)
    return x


def _linear_inputs(c, rnd, dtype):
    M, K, N = c["M"], c["K"], c["N"]
    outs = 2 * N if c["act"] == "swiglu" else N
    x = {"x": rnd(M, K).to(dtype), "weight": (rnd(outs, K) / math.sqrt(K)).to(dtype)}
    if c["bias"]:
        x["bias"] = (0.1 * rnd(outs)).to(dtype)
    if c["residual"]:
        x["residual"] = rnd(M, N).to(dtype)
    if c["train"]:
        x["dy"] = rnd(M, N).to(dtype)
    return x


def _logprob_inputs(c, rnd, dtype, gen):
    R, V = c["rows"], c["V"]
    # logits of a language model: a few tokens far above the rest; the tokens are likely ones
    logits = rnd(R, V)
    logits.mul_(2.0)
    near = torch.randint(0, V, (R, 8), generator=gen, device=DEV)
    logits.scatter_add_(1, near, 4.0 + 3.0 * rnd(R, 8))
    ids = near[:, 0].clone()
    if c["pad"]:
        logits[:, V - c["pad"]:] = -math.inf
        ids.clamp_(max=V - c["pad"] - 1)
    skip = torch.rand(R, generator=gen, device=DEV) < c["ignored"]
    ids[skip] = IGNORE
    x = {"logits": logits.to(dtype), "ids": ids}
    if c["train"]:
        x["dlogp"], x["dent"] = -torch.rand(R, generator=gen, device=DEV), 0.01 * rnd(R)
    return x


_GRADS = {"layer": ("x", "weight", "bias"), "rms": ("x", "weight"), "linear": ("x", "weight", "bias", "residual"),
          "logprobs": ("logits",)}


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def rnd(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)

    dtype = getattr(torch, case["dtype"])
    if case["op"] == "linear":
        x = _linear_inputs(case, rnd, dtype)
    elif case["op"] == "logprobs":
        x = _logprob_inputs(case, rnd, dtype, gen)
    else:
        x = _norm_inputs(case, rnd, dtype)
    if case["train"]:
        for name in _GRADS[case["op"]] + ("residual",):
            if name in x:
                x[name].requires_grad_()
    return {"case": dict(case), "x": x}


# ---- the plain forms -------------------------------------------------------------------------------------------

def _plain_norm(c, x):
    dtype, layer = x["x"].dtype, c["op"] == "layer"
    s = x["x"]
    if c["residual"]:
        s = (s.float() + x["residual"].float()).to(dtype)  # the stream as the next block reads it
    f, w = s.float(), x["weight"].float()
    if layer:
        f = f - f.mean(-1, keepdim=True)
    rstd = torch.rsqrt((f * f).mean(-1, keepdim=True) + EPS)
    h = f * rstd
    y = h * w
    if layer:
        y = y + x["bias"].float()
    out = {"y": y.to(dtype)}
    if c["residual"]:
        out["s"] = s
    if not c["train"]:
        return out
    dy = x["dy"].float()
    a = dy * w
    dx = a - h * (a * h).mean(-1, keepdim=True)
    if layer:
        dx = dx - a.mean(-1, keepdim=True)
    dx = dx * rstd
    if c["residual"]:
        dx = dx + x["ds"].float()
    out["dx"] = dx.to(dtype)
    if c["residual"]:
        out["dresidual"] = out["dx"]
    out["dweight"] = (dy * h).sum(0).to(x["weight"].dtype)
    if layer:
        out["dbias"] = dy.sum(0).to(x["bias"].dtype)
    return out


def _act(act, z):
    """The activation of ``z`` and, as a function of the gradient that arrives, the gradient of ``z``."""
    if act == "relu":
        return z.clamp_min(0), lambda d: d * (z > 0)
    if act == "silu":
        g = torch.sigmoid(z)
        return z * g, lambda d: d * (g * (1 + z * (1 - g)))
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, lambda d: d * (cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi)))
    if act == "gelu_tanh":
        b = math.sqrt(2 / math.pi)
        t = torch.tanh(b * (z + 0.044715 * z * z * z))
        return 0.5 * z * (1 + t), lambda d: d * (0.5 * (1 + t) + 0.5 * z * (1 - t * t) * b * (1 + 0.134145 * z * z))
    if act == "swiglu":
        gate, up = z.chunk(2, -1)
        g = torch.sigmoid(gate)
        return gate * g * up, lambda d: torch.cat([d * up * (g * (1 + gate * (1 - g))), d * gate * g], -1)
    return z, lambda d: d


def _plain_linear(c, x):
    dtype = x["x"].dtype
    f, w = x["x"].float(), x["weight"].float()
    z = f @ w.T
    if c["bias"]:
        z = z + x["bias"].float()
    y, back = _act(c["act"], z)
    if c["residual"]:
        y = y + x["residual"].float()
    out = {"y": y.to(dtype)}
    if not c["train"]:
        return out
    dz = back(x["dy"].float())
    out["dx"] = (dz @ w).to(dtype)
    out["dweight"] = (dz.T @ f).to(dtype)
    if c["bias"]:
        out["dbias"] = dz.sum(0).to(dtype)
    if c["residual"]:
        out["dresidual"] = x["dy"].to(dtype)
    return out


def _plain_top(c, logits, lse, keep):
    """The ``top`` largest log probabilities of each row, ties to the lowest index: the largest of distinct whole
    numbers, a logit's order above its index's."""
    V, k = c["V"], c["top"]
    b = (logits + 0.0).view(torch.int32).long()
    key = torch.where(b < 0, b ^ 0x7FFFFFFF, b) * (1 << 32) + (V - 1 - torch.arange(V, device=logits.device))
    at = V - 1 - (key.topk(k, -1).values & 0xFFFFFFFF)
    top = logits.gather(1, at) - lse
    return torch.where(keep, top, torch.zeros_like(top)), torch.where(keep, at, torch.full_like(at, -1))


def _plain_logprobs(c, x):
    f, ids = x["logits"].float(), x["ids"]
    keep = (ids != IGNORE)[:, None]
    at = ids.clamp_min(0)[:, None]
    u = f - f.amax(-1, keepdim=True)
    e = torch.exp(u)
    total = e.sum(-1, keepdim=True)
    logz = torch.log(total)
    p = e / total
    pu = torch.where(p > 0, p * u, torch.zeros_like(p))  # a masked entry has no share
    ent = logz - pu.sum(-1, keepdim=True)
    zero = torch.zeros_like(ent)
    out = {"logp": torch.where(keep, u.gather(1, at) - logz, zero)[:, 0], "entropy": torch.where(keep, ent, zero)[:, 0]}
    if c["top"]:
        out["top"], out["top_ids"] = _plain_top(c, f, f.amax(-1, keepdim=True) + logz, keep)
    if not c["train"]:
        return out
    dlogp, dent = torch.where(keep, x["dlogp"][:, None], zero), torch.where(keep, x["dent"][:, None], zero)
    dx = -p * dlogp - dent * (pu - p * logz + p * ent)
    dx.scatter_add_(1, at, dlogp)
    out["dlogits"] = dx.to(x["logits"].dtype)
    return out


# ---- the framework's calls -------------------------------------------------------------------------------------

def _own_norm(c, x):
    from ccq_amd import layer_norm, rms_norm
    r = x.get("residual")
    if c["op"] == "layer":
        got = layer_norm(x["x"], x["weight"], x["bias"], eps=EPS, residual=r)
    else:
        got = rms_norm(x["x"], x["weight"], eps=EPS, residual=r)
    y, s = got if r is not None else (got, None)
    out = {"y": y} if s is None else {"y": y, "s": s}
    if c["train"]:
        names = [n for n in ("x", "weight", "bias", "residual") if n in x]
        outs, grads = ([y], [x["dy"]]) if s is None else ([y, s], [x["dy"], x["ds"]])
        got = torch.autograd.grad(outs, [x[n] for n in names], grads)
        out.update(("d" + n, g) for n, g in zip(names, got))
    return out


def _own_linear(c, x):
    from ccq_amd import fused_linear
    y = fused_linear(x["x"], x["weight"], x.get("bias"), activation=c["act"] or None, residual=x.get("residual"))
    out = {"y": y}
    if c["train"]:
        names = [n for n in _GRADS["linear"] if n in x]
        got = torch.autograd.grad(y, [x[n] for n in names], x["dy"])
        out.update(("d" + n, g) for n, g in zip(names, got))
    return out


def _own_logprobs(c, x):
    from ccq_amd import token_logprobs
    got = token_logprobs(x["logits"], x["ids"], top_k=c["top"], ignore_index=IGNORE)
    out = {"logp": got.logprobs, "entropy": got.entropy}
    if c["top"]:
        out["top"], out["top_ids"] = got.top_logprobs, got.top_ids
    if c["train"]:
        out["dlogits"], = torch.autograd.grad([got.logprobs, got.entropy], [x["logits"]], [x["dlogp"], x["dent"]])
    return out


def run(state):
    c, x = state["case"], state["x"]
    if own:
        return {"linear": _own_linear, "logprobs": _own_logprobs}.get(c["op"], _own_norm)(c, x)
    with torch.no_grad():
        return {"linear": _plain_linear, "logprobs": _plain_logprobs}.get(c["op"], _plain_norm)(c, x)


# ---- what a pass cannot do without -----------------------------------------------------------------------------

def work(case):
    c = case
    size = 4 if c["dtype"] == "float32" else 2
    if c["op"] in ("layer", "rms"):
        R, D, res = c["rows"], c["D"], c["residual"]
        wsize = 4 if c["wdtype"] == "float32" else 2
        vectors = 2 if c["op"] == "layer" else 1
        acts = 4 if res else 2                                      # x (residual) in, y (s) out
        n = acts * R * D * size + vectors * D * wsize
        if c["train"]:                                              # dy (ds) in, dx out, the vectors' gradients
            n += (3 if res else 2) * R * D * size + vectors * D * wsize
        return {"bytes": n, "flops": (20 if c["train"] else 8) * R * D}
    if c["op"] == "linear":
        M, K, N = c["M"], c["K"], c["N"]
        outs = 2 * N if c["act"] == "swiglu" else N
        n = (M * K + outs * K + M * N * (2 if c["residual"] else 1) + (outs if c["bias"] else 0)) * size
        if c["train"]:
            n += (M * N + M * K + outs * K + (outs if c["bias"] else 0)) * size
        return {"bytes": n, "flops": (3 if c["train"] else 1) * 2 * M * outs * K}
    R, V = c["rows"], c["V"]
    read = R * (1.0 - c["ignored"])                                 # a row without a token need not be read
    n = read * V * size + R * 8 + R * 8 + R * c["top"] * 12
    flops = 5 * read * V
    if c["train"]:
        n += R * V * size + R * 8
        flops += 6 * read * V
    return {"bytes": n, "flops": flops}


# ---- the operators' definitions in 64 bits ---------------------------------------------------------------------

def _exact_norm(c, x):
    dtype = x["x"].dtype
    x = {n: t.detach() for n, t in x.items()}
    s = x["x"].double()
    if "residual" in x:
        s = (s + x["residual"].double()).to(dtype).double()
    n = s.shape[-1]
    mu = s.sum(-1, keepdim=True) / n if c["op"] == "layer" else torch.zeros(s.shape[0], 1, device=DEV, dtype=torch.float64)
    sigma = torch.sqrt((s - mu).square().sum(-1, keepdim=True) / n + EPS)
    w = x["weight"].double()
    y = (s - mu) / sigma * w
    if "bias" in x:
        y = y + x["bias"].double()
    out = {"y": y, "s": s if "residual" in x else None}
    if c["train"]:
        dh = x["dy"].double() * w
        # h = (s - mu) / sigma: through the quotient, then through sigma and mu
        dsigma = -(dh * (s - mu)).sum(-1, keepdim=True) / sigma.square()
        dx = dh / sigma + dsigma * (s - mu) / (n * sigma)
        if c["op"] == "layer":
            dx = dx - dh.sum(-1, keepdim=True) / (n * sigma)  # (the s - mu of a row sum to zero)
        if "ds" in x:
            dx = dx + x["ds"].double()
        out["dx"] = dx
        out["dresidual"] = dx if "residual" in x else None
        out["dweight"] = (x["dy"].double() * (s - mu) / sigma).sum(0)
        out["dbias"] = x["dy"].double().sum(0) if "bias" in x else None
    return {k: v for k, v in out.items() if v is not None}


def _act64(act, z):
    """Value and derivative (swiglu: the derivatives of both halves) in 64 bits."""
    if act == "relu":
        return torch.where(z > 0, z, 0.0), torch.where(z > 0, 1.0, 0.0).double()
    if act == "silu":
        q = 1 / (1 + torch.exp(-z))
        return z * q, q + z * q * (1 - q)
    if act == "gelu":
        q = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        return z * q, q + z * torch.exp(-z.square() / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        v = math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
        q = 1 / (1 + torch.exp(-2 * v))  # (1 + tanh v) / 2
        return z * q, q + z * 2 * q * (1 - q) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z.square())
    return z, torch.ones_like(z)


def _exact_linear(c, x):
    x = {n: t.detach().double() for n, t in x.items()}
    z = torch.nn.functional.linear(x["x"], x["weight"], x.get("bias"))
    if c["act"] == "swiglu":
        half = z.shape[-1] // 2
        v, d = _act64("silu", z[:, :half])
        y = v * z[:, half:]
    else:
        y, d = _act64(c["act"], z)
    out = {"y": y + x["residual"] if "residual" in x else y}
    if c["train"]:
        dy = x["dy"]
        dz = torch.cat([dy * z[:, half:] * d, dy * v], 1) if c["act"] == "swiglu" else dy * d
        out["dx"] = torch.mm(dz, x["weight"])
        out["dweight"] = torch.mm(dz.t(), x["x"])
        if "bias" in x:
            out["dbias"] = dz.sum(0)
        if "residual" in x:
            out["dresidual"] = dy
    return out


def _exact_logprobs(c, x):
    z, ids = x["logits"].detach().double(), x["ids"]
    live = ids != IGNORE
    lse = torch.logsumexp(z, -1)
    logp = z - lse[:, None]
    del z
    p = torch.exp(logp)
    plogp = torch.special.entr(p).neg_()  # p log p, nothing where p is nothing
    ent = -plogp.sum(-1)
    mine = torch.gather(logp, 1, torch.where(live, ids, 0)[:, None])[:, 0]
    out = {"logp": torch.where(live, mine, 0.0), "entropy": torch.where(live, ent, 0.0)}
    if c["top"]:
        order = torch.sort(logp, dim=-1, descending=True, stable=True)
        out["top"] = torch.where(live[:, None], order.values[:, :c["top"]], 0.0)
        out["top_ids"] = torch.where(live[:, None], order.indices[:, :c["top"]], -1)
    if c["train"]:
        a, b = (torch.where(live, x[n].double(), 0.0)[:, None] for n in ("dlogp", "dent"))
        # d H / d z_j = -p_j (log p_j + H), d logp / d z_j = [j = id] - p_j
        dz = plogp.addcmul_(p, ent[:, None]).mul_(-b)
        dz.addcmul_(p, a, value=-1)
        dz.scatter_add_(1, torch.where(live, ids, 0)[:, None], a)
        out["dlogits"] = dz
    return out


def exact(case, seed):
    x = prepare(case, seed)["x"]
    with torch.no_grad():
        return {"linear": _exact_linear, "logprobs": _exact_logprobs}.get(case["op"], _exact_norm)(case, x)
