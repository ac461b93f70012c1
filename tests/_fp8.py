"""The 8-bit rows' definition in 64 bits on the CPU, for the tests of quantize_fp8, rms_norm_fp8 and fp8_linear."""

import torch

BLOCK = 128


def exponent(most):
    """The scales' exponents of blocks with these largest magnitudes (float64): the least e >= -126 with most <= 448 * 2^e."""
    m, e = torch.frexp(most)           # most = m 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp_min(-126)
    return torch.where(most == 0, torch.full_like(e, -126), e)


def to_e4m3(v):
    """float64 numbers of magnitude up to 448 to the nearest e4m3, ties to even."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (e - 1).clamp_min(-6) - 3)
    return torch.round(v / step) * step


def blocks(x):
    D = x.shape[-1]
    n = -(-D // BLOCK)
    return torch.nn.functional.pad(x.double(), (0, n * BLOCK - D)).unflatten(-1, (n, BLOCK))


def quantized(x):
    """Values and scales (both float64) of finite rows."""
    D, b = x.shape[-1], blocks(x)
    scale = torch.ldexp(torch.ones(b.shape[:-1], dtype=torch.float64), exponent(b.abs().amax(-1)))
    return to_e4m3(b / scale[..., None]).flatten(-2)[..., :D], scale


def meant(values, scales):
    """The numbers that rows stand for, float64 on the CPU."""
    v, s = values.cpu().double(), scales.cpu().double()
    return v * s.repeat_interleave(BLOCK, -1)[..., :v.shape[-1]]


def check_rounded(values, scales, y, err, where=""):
    """values and scales are the 8-bit form of numbers within err (a tensor) of y (float64): the scale is that of a largest
    magnitude within its error, and each value lies between the roundings of y - err and y + err in that scale."""
    D = y.shape[-1]
    v, s = values.cpu().double(), scales.cpu().double()
    b, e = blocks(y), blocks(err.expand_as(y))
    lo = exponent((b.abs() - e).clamp_min(0).amax(-1))
    hi = exponent((b.abs() + e).amax(-1))
    got = torch.log2(s)
    assert bool(((got >= lo) & (got <= hi)).all()), (where, "scales")
    wide = s[..., None].expand_as(b).flatten(-2)[..., :D]
    low, high = to_e4m3((y - err) / wide), to_e4m3((y + err) / wide)
    # (beside the rounded bounds themselves nothing is allowed)
    bad = ~((v >= low) & (v <= high.clamp_max(448.0).clamp_min(-448.0)) | (v == low.clamp(-448.0, 448.0)))
    assert not bool(bad.any()), (where, int(bad.sum()), y[bad][:4], (v * wide)[bad][:4])


def random_rows(gen, rows, D, scale=1.0):
    """Finite rows as (values float8, scales e8m0) on the CPU, laid out as the products read them, bytes behind the rows' ends
    all ones (NaN)."""
    x = torch.randn(rows, D, generator=gen) * scale * torch.exp(torch.randn(rows, 1, generator=gen))
    v, s = quantized(x)
    return laid_out(v.to(torch.float32).to(torch.float8_e4m3fn), 16), laid_out(s.to(torch.float32).to(torch.float8_e8m0fnu), 4)


def laid_out(t, unit, device="cpu"):
    room = torch.full((*t.shape[:-1], -(-t.shape[-1] // unit) * unit), 255, dtype=torch.uint8, device=device)
    room[..., :t.shape[-1]] = t.view(torch.uint8).to(device)
    return room.view(t.dtype)[..., :t.shape[-1]]


def to_device(pair, dev):
    """A laid-out pair on another device, laid out there as well."""
    return tuple(laid_out(t, n, dev) for t, n in zip(pair, (16, 4)))


def act64(act, z):
    """Value of an activation in 64 bits, and how much an error of z changes it at most."""
    if act is None:
        return z, torch.ones_like(z)
    if act == "relu":
        return z.clamp_min(0), torch.ones_like(z)
    if act in ("silu", "swish"):
        return z * torch.sigmoid(z), torch.full_like(z, 1.1)
    if act == "gelu":
        return z * 0.5 * torch.special.erfc(-z * 0.5 ** 0.5), torch.full_like(z, 1.13)
    v = (2 / torch.pi) ** 0.5 * (z + 0.044715 * z ** 3)
    return z * torch.sigmoid(2 * v), torch.full_like(z, 1.13)


def _fields(v):
    """Exponents of e4m3 numbers as they are held: subnormals at -6; zeros far below."""
    _, e = torch.frexp(v)
    return torch.where(v == 0, torch.full_like(e, -1000), (e - 1).clamp_min(-6)).double()


def cut_off(x, w):
    """[M, N]: what the 8-bit matrix instruction may cut off: of each eight consecutive products the bits below 2^-13 of the
    largest exponent among them, so less than that for each of the eight."""
    (xv, xs), (wv, ws) = ((v.cpu().double(), s.cpu().double()) for v, s in (x, w))
    K = xv.shape[1]
    pad = (0, -K % BLOCK)
    a, b = (torch.nn.functional.pad(_fields(t), pad, value=-1000.0).unflatten(1, (-1, BLOCK // 8, 8)) for t in (xv, wv))
    out = torch.zeros(xv.shape[0], wv.shape[0], dtype=torch.float64)
    for k in range(a.shape[1]):
        most = (a[:, None, k] + b[None, :, k]).amax(-1)          # [M, N, 16]
        out += (8 * torch.exp2(most - 13)).sum(-1) * xs[:, k, None] * ws[None, :, k]
    return out


def linear64(x, w, bias=None, act=None, residual=None, exact=False):
    """fp8_linear in 64 bits on the CPU and how far its fp32 sums and activations may be off, both [M, N].

    Products of two e4m3 are exact in fp32.  exact (an output in fp32): a block's 128 products are added in fp32, then the
    blocks: at most 128 + K / 128 roundings, each 2^-24 of the magnitudes' sum.  Otherwise what the 8-bit instruction cuts
    off, and the fp32 additions of its eights and of the blocks.  A residual rounds once more, an
    activation within 8 roundings of its argument and result (exponential, reciprocal, products; the error function within
    4e-7)."""
    a, b = meant(*x), meant(*w)
    K = a.shape[-1]
    z, size = a @ b.T, a.abs() @ b.abs().T
    if bias is not None:  # the sums begin with it
        z = z + bias.cpu().double()
        size = size + bias.cpu().double().abs()
    err = ((128 if exact else 16) + K / 128) * 2.0 ** -24 * size
    if not exact:
        err = err + cut_off(x, w)
    if act == "swiglu":
        n = z.shape[-1] // 2
        y, slope = act64("silu", z[:, :n])
        err = err[:, :n] * slope * z[:, n:].abs() + err[:, n:] * y.abs() + err[:, :n] * err[:, n:] * 1.1
        y = y * z[:, n:]
        err = err + 8 * 2.0 ** -24 * y.abs() * (1 + z[:, :n].abs())
    else:
        y, slope = act64(act, z)
        err = err * slope
        if act not in (None, "relu"):
            err = err + 8 * 2.0 ** -24 * (z.abs() + y.abs() * (1 + z.abs()))
    if residual is not None:
        y = y + residual.cpu().double()
        err = err + 2.0 ** -24 * (y.abs() + residual.cpu().double().abs())
    return y, err
