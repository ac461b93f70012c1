"""GPU parity of the block norms (``ccq_amd.layer_norm`` / ``rms_norm``) against their formulas in 64 bits.

Tolerances are element by element, from the roundings made: u = eps / 2 of the output's type for its one rounding,
and for the arithmetic in 32 bits C = 64 units of 2^-24 of the magnitudes that enter.  A mean over D <= 8192 is at
most 32 additions in a lane and 10 levels of a tree, so its error is below 42 2^-24 mean|s|; the rest (centring,
square, root, quotient, product) adds a few units.  Sums over rows: at most ceil(rows / 512) + 4 + 32 + 16
additions one after the other.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

D64 = torch.float64
BF, HF, FL = torch.bfloat16, torch.float16, torch.float32
U32, C = 2.0 ** -24, 64


def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda")


def _half_step(t):
    return torch.finfo(t).eps / 2


def formula(layer, x, w, b, r, eps, dy=None, ds=None):
    """Results in 64 bits and, beside each, the magnitude that its 32-bit arithmetic errs by."""
    s = x.to(D64)
    if r is not None:
        s = (s + r.to(D64)).to(x.dtype).to(D64)
    D = s.shape[-1]
    mu = s.mean(-1, keepdim=True) if layer else torch.zeros_like(s[..., :1])
    rho = 1 / torch.sqrt((s - mu).pow(2).mean(-1, keepdim=True) + eps)
    h = (s - mu) * rho
    wd = w.to(D64) if w is not None else torch.ones(D, dtype=D64)
    bd = b.to(D64) if b is not None else torch.zeros(D, dtype=D64)
    off = (s.abs().mean(-1, keepdim=True) * rho if layer else 0) + h.abs()   # error of h, in units
    out = {"y": (h * wd + bd, off * wd.abs() + bd.abs()), "s": (s, 0 * s)}
    if dy is not None:
        d = dy.to(D64)
        a = d * wd
        m1 = (a * h).mean(-1, keepdim=True)
        m0 = a.mean(-1, keepdim=True) if layer else 0
        e = ds.to(D64) if ds is not None else 0
        aa, am = a.abs(), a.abs().mean(-1, keepdim=True)
        m1a = (aa * off).mean(-1, keepdim=True)
        out["dx"] = (rho * (a - m0 - h * m1) + e,
                     rho * (aa + am + 2 * off * m1a) + (ds.to(D64).abs() if ds is not None else 0))
        out["dw"] = ((d * h).sum(0), (d.abs() * off).sum(0))
        out["db"] = (d.sum(0), d.abs().sum(0))
    return out


def close(name, got, want, units=C):
    ref, mag = want
    got = got.detach().to("cpu", D64).reshape(ref.shape)
    bound = _half_step(name[1]) * ref.abs() + units * U32 * mag + torch.finfo(name[1]).tiny
    worst = ((got - ref).abs() / bound).max().item() if ref.numel() else 0.0
    assert torch.isfinite(got).all() and worst <= 1, (name, worst)


def make(layer, rows, D, dtype, wdtype, seed, residual=False, affine=True, pad=0, offset=0.3):
    gen = torch.Generator().manual_seed(seed)

    def rnd(*shape):
        return torch.randn(*shape, generator=gen)

    x = {"x": (rnd(rows, D + pad) * torch.exp(0.5 * rnd(D + pad)) + offset).to(dtype)}
    if affine:
        x["w"] = (1 + 0.1 * rnd(D)).to(wdtype)
        if layer:
            x["b"] = (0.1 * rnd(D)).to(wdtype)
    if residual:
        x["r"] = rnd(rows, D + pad).to(dtype)
        x["ds"] = rnd(rows, D).to(dtype)
    x["dy"] = rnd(rows, D).to(dtype)
    return x


def call(layer, x, D, eps=1e-5, grad=True, pad=0):
    """The operator on the GPU: results by name.  ``pad`` elements of every row lie around the D that are taken."""
    from ccq_amd import layer_norm, rms_norm
    dev = _cuda()
    g = {n: t.to(dev) for n, t in x.items()}
    if grad:
        for n in ("x", "w", "b", "r"):
            if n in g:
                g[n].requires_grad_()
    lo = pad // 2
    cut = {n: (t[:, lo:lo + D] if n in ("x", "r") and pad else t) for n, t in g.items()}
    kw = dict(eps=eps, residual=cut.get("r"))
    got = layer_norm(cut["x"], g.get("w"), g.get("b"), **kw) if layer else rms_norm(cut["x"], g.get("w"), **kw)
    y, s = got if "r" in g else (got, None)
    out = {"y": y}
    if s is not None:
        out["s"] = s
    if grad:
        names = [n for n in ("x", "w", "b", "r") if n in g]
        outs, gs = ([y, s], [g["dy"], g["ds"]]) if s is not None else ([y], [g["dy"]])
        for n, t in zip(names, torch.autograd.grad(outs, [g[n] for n in names], gs)):
            out["d" + n] = t[:, lo:lo + D] if n in ("x", "r") and pad else t
    return out


def check(layer, x, D, dtype, wdtype, eps=1e-5, pad=0):
    lo = pad // 2
    cut = {n: (t[:, lo:lo + D] if n in ("x", "r") and pad else t) for n, t in x.items()}
    want = formula(layer, cut["x"], x.get("w"), x.get("b"), cut.get("r"), eps, x["dy"], x.get("ds"))
    got = call(layer, x, D, eps, True, pad)
    rows = x["x"].shape[0]
    seq = C + -(-rows // 512) + 52
    close(("y", dtype), got["y"], want["y"])
    close(("dx", dtype), got["dx"], want["dx"], 2 * C)
    if "r" in x:
        assert torch.equal(got["s"].cpu().double(), want["s"][0])
        assert torch.equal(got["dr"], got["dx"])
    if "w" in x:
        close(("dw", wdtype), got["dw"], want["dw"], seq)
    if "b" in x:
        close(("db", wdtype), got["db"], want["db"], seq)
    plain = call(layer, x, D, eps, False, pad)   # the call without gradients
    for n in plain:
        assert torch.equal(plain[n], got[n]), n


SIZES = [(1, 1), (1, 1024), (3, 7), (5, 8), (16, 1024), (130, 64), (257, 96), (33, 129), (70, 777), (1200, 256),
         (2100, 1024), (40, 1025), (600, 2048), (21, 2049), (19, 4096), (11, 4100), (9, 8191), (9, 8192)]


@pytest.mark.parametrize("layer", [True, False], ids=["layer", "rms"])
@pytest.mark.parametrize("rows,D", SIZES, ids=str)
def test_norm(layer, rows, D):
    print("test_norm", layer, rows, D, flush=True)
    k = (rows + D) % 4
    dtype, wdtype = [(BF, BF), (BF, FL), (HF, HF), (FL, FL)][k]
    for i, (d, w) in enumerate({(dtype, wdtype), (FL, FL), (BF, BF)}):
        check(layer, make(layer, rows, D, d, w, rows + D + i, residual=i % 2 == 0), D, d, w)


@pytest.mark.parametrize("dtype", [BF, HF, FL], ids=str)
@pytest.mark.parametrize("layer", [True, False], ids=["layer", "rms"])
@pytest.mark.parametrize("D,pad", [(64, 8), (1000, 3), (2048, 1), (4097, 5)])
def test_norm_strided_rows(layer, dtype, D, pad):
    """Rows inside wider ones, at addresses that no 16-byte alignment holds for."""
    print("test_norm_strided_rows", layer, dtype, D, pad, flush=True)
    check(layer, make(layer, 37, D, dtype, FL, 5, residual=True, pad=pad), D, dtype, FL, pad=pad)


@pytest.mark.parametrize("layer", [True, False], ids=["layer", "rms"])
def test_norm_without_weights_and_other_eps(layer):
    check(layer, make(layer, 50, 320, BF, BF, 1, affine=False), 320, BF, BF, eps=1e-3)
    check(layer, make(layer, 50, 320, FL, FL, 2, residual=True, affine=False), 320, FL, FL, eps=0.0)


def test_norm_large_offset_and_constant_rows():
    # a mean far above the deviation: the variance is that of the centred values (an offset of 300 in 32 bits
    # leaves h an error of 300 units, which the bound counts)
    check(True, make(True, 20, 512, FL, FL, 3, offset=300.0), 512, FL, FL)
    x = make(True, 4, 256, BF, BF, 4)
    x["x"][:] = 2.5
    got = call(True, x, 256)
    assert torch.equal(got["y"].cpu(), x["b"].expand(4, 256))
    assert torch.isfinite(got["dx"]).all() and (got["dw"] == 0).all()


def test_norm_bad_values_stay_in_their_row():
    for layer in (True, False):
        x = make(layer, 40, 1024, BF, BF, 6)
        good = call(layer, x, 1024)
        x["x"][7, 5] = float("nan")
        x["x"][30, 1000] = float("inf")
        got = call(layer, x, 1024)
        rows = torch.ones(40, dtype=torch.bool)
        rows[[7, 30]] = False
        for n in ("y", "dx"):
            assert torch.equal(got[n][rows.cuda()], good[n][rows.cuda()])
            assert got[n][7].isnan().all() and got[n][30].isnan().any()


def test_norm_no_rows_and_leading_dimensions():
    from ccq_amd import layer_norm
    dev = _cuda()
    w = torch.ones(96, device=dev, dtype=BF, requires_grad=True)
    b = torch.zeros(96, device=dev, dtype=BF, requires_grad=True)
    x = torch.zeros(0, 5, 96, device=dev, dtype=BF, requires_grad=True)
    y = layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], torch.zeros_like(y))
    assert y.shape == x.shape and dx.shape == x.shape and (dw == 0).all() and (db == 0).all()
    x = torch.randn(2, 3, 4, 96, device=dev).to(BF)
    flat = layer_norm(x.reshape(24, 96), w, b)
    assert torch.equal(layer_norm(x, w, b), flat.view(2, 3, 4, 96))
    t = x.transpose(0, 2)
    assert torch.equal(layer_norm(t, w, b), flat.view(2, 3, 4, 96).transpose(0, 2))
    assert torch.equal(layer_norm(x[0, 0, 0], w, b), flat[0])


def test_norm_broadcast_gradient_and_partial_leaves():
    """A summed output's gradient has stride 0; leaves that need no gradient get none; an unused output has none."""
    from ccq_amd import layer_norm
    dev = _cuda()
    x = make(True, 60, 200, BF, FL, 8, residual=True)
    ref = formula(True, x["x"], x["w"], x["b"], x["r"], 1e-5, torch.ones(60, 200))
    g = {n: t.to(dev) for n, t in x.items()}
    xs = g["x"].requires_grad_()
    y, s = layer_norm(xs, g["w"], g["b"], residual=g["r"])
    y.float().sum().backward()
    close(("dx", BF), xs.grad, ref["dx"], 2 * C)
    w = g["w"].requires_grad_()
    y = layer_norm(g["x"].detach(), w, g["b"])
    y.float().sum().backward()
    ref = formula(True, x["x"], x["w"], x["b"], None, 1e-5, torch.ones(60, 200))
    close(("dw", FL), w.grad, ref["dw"], C + 52)
    xs = x["x"].to(dev).requires_grad_()
    _, s = layer_norm(xs, g["w"].detach(), g["b"], residual=g["r"])
    s.backward(g["ds"])
    assert torch.equal(xs.grad, g["ds"])


def test_norm_against_differences():
    """The gradient of sum(y c) along random directions against central differences of the formula in 64 bits.
    The step h = 1e-4 leaves a truncation of h^2 times the third derivative, about 1e-8 of the sum's scale."""
    for layer in (True, False):
        x = make(layer, 6, 48, FL, FL, 11)
        got = call(layer, x, 48)
        gen = torch.Generator().manual_seed(1)
        for name, grad in (("x", "dx"), ("w", "dw")):
            v = torch.randn(x[name].shape, generator=gen, dtype=D64)

            def loss(t):
                xs = {**x, name: x[name].to(D64) + t * v}
                y = formula(layer, xs["x"], xs["w"], xs.get("b"), None, 1e-5)["y"][0]
                return (y * x["dy"].to(D64)).sum()

            want = (loss(1e-4) - loss(-1e-4)) / 2e-4
            have = (got[grad].cpu().double() * v).sum()
            scale = (got[grad].cpu().double().abs() * v.abs()).sum()
            assert abs(have - want) <= 1e-6 * scale + 1e-6, (layer, name, have.item(), want.item())


def test_norm_same_bits_again_and_other_stream():
    dev = _cuda()
    x = make(True, 1500, 1024, BF, FL, 12, residual=True)
    first = call(True, x, 1024)
    stream = torch.cuda.Stream(dev)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = call(True, x, 1024)
    torch.cuda.current_stream().wait_stream(stream)
    for n in first:
        assert torch.equal(first[n], other[n]), n


def test_norm_captured():
    """Forward and backward in a captured graph, replayed on other inputs with eager work between."""
    from ccq_amd import layer_norm
    dev = _cuda()
    sets = [{n: t.to(dev) for n, t in make(True, 300, 640, BF, FL, 20 + i, residual=True).items()} for i in range(3)]

    def step(g):
        leaves = [g[n].detach().requires_grad_() for n in ("x", "w", "b", "r")]
        y, s = layer_norm(leaves[0], leaves[1], leaves[2], residual=leaves[3])
        return [y, s, *torch.autograd.grad([y, s], leaves, [g["dy"], g["ds"]])]

    want = [[t.clone() for t in step(g)] for g in sets]
    static = {n: t.clone() for n, t in sets[0].items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for k in (0, 1, 2, 1):
        for n in static:
            static[n].copy_(sets[k][n])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want[k]):
            assert torch.equal(a, b)
        step(sets[0])
        torch.cuda.synchronize()


@pytest.mark.parametrize("layer", [False, True], ids=["rms", "layer"])
@pytest.mark.parametrize("rows,D,dtype,residual", [(1100, 8191, FL, True), (600, 8192, FL, False), (1100, 4096, FL, True),
                                                   (1100, 8191, BF, True), (600, 8192, HF, False)], ids=str)
def test_more_wide_rows_than_workgroups(layer, rows, D, dtype, residual):
    """Rows of sixteen waves each, several of them to a workgroup, both ways."""
    check(layer, make(layer, rows, D, dtype, FL, rows + D, residual), D, dtype, FL)
