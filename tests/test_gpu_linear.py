"""GPU parity of the linear map with an epilogue (``ccq_amd.fused_linear``).

Two kinds of inputs.  Small whole numbers: every product and sum is exact in fp32, so the outputs and, without a
curved activation, all gradients have to be the exact results rounded once to their type, bit for bit, whatever the
tile, the tail or the split.  Real numbers: element-by-element bounds from the roundings, u = eps / 2 of the type:
  y:   u |y| + e, e = 2^-24 ((K / 16 + 16) (|x| |W|^T + |b|) + 16 (|z| + 1) + |r|) through the activation (slopes and
       the gate's factor at most 1.2)
  dz:  u (|dz| + |dy| |z|) (its rounding, and z's through a second derivative below 1)
and for dx and dW, whose sums of such errors cancel at random, the relative norm 1.5 u (a rounding's error is below
u / 1.7 in the mean: one of the result, one of dz, one of z); a lost element of the contraction would be 1 / sqrt(4096).
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

D64 = torch.float64
BF, HF, FL = torch.bfloat16, torch.float16, torch.float32
U32 = 2.0 ** -24
ACTS = [None, "relu", "silu", "gelu", "gelu_tanh", "swiglu"]


def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda")


def whole(gen, *shape):
    return torch.randint(-2, 3, shape, generator=gen).float()


def guarded(t, dtype, dev, columns=0):
    """``t`` inside a buffer of NaN: rows above and below, and ``columns`` columns on the right (a view)."""
    rows, cols = t.shape
    big = torch.full((rows + 4, cols + columns), float("nan"), device=dev, dtype=dtype)
    view = big[2:2 + rows, :cols]
    view.copy_(t)
    return view


def run(x, w, b, act, r, dy):
    from ccq_amd import fused_linear
    leaves = [None if t is None else t.detach().requires_grad_() for t in (x, w, b, r)]
    y = fused_linear(leaves[0], leaves[1], leaves[2], act, leaves[3])
    live = [t for t in leaves if t is not None]
    grads = iter(torch.autograd.grad(y, live, dy))
    return y.detach(), [None if t is None else next(grads) for t in leaves]


def formula(x, w, b, act, r, dy):
    """Results in 64 bits: y, z, dz and the four gradients."""
    x, w, b, r, dy = (None if t is None else t.to(D64) for t in (x, w, b, r, dy))
    z = x @ w.T
    if b is not None:
        z = z + b
    z = z.requires_grad_()
    if act == "swiglu":
        g, u = z.chunk(2, -1)
        y = g * torch.sigmoid(g) * u
    else:
        y = {None: lambda t: t * 1.0, "relu": torch.relu, "silu": lambda t: t * torch.sigmoid(t),
             "gelu": lambda t: t * 0.5 * torch.special.erfc(-t / math.sqrt(2)),
             "gelu_tanh": lambda t: 0.5 * t * (1 + torch.tanh(math.sqrt(2 / math.pi) * (t + 0.044715 * t ** 3)))}[act](z)
    dz, = torch.autograd.grad(y, z, dy)
    y = y.detach() if r is None else y.detach() + r
    return y, z.detach(), dz, [dz @ w, dz.T @ x, None if b is None else dz.sum(0), None if r is None else dy]


SIZES = [(1, 1, 1), (1, 1024, 1024), (2, 7, 9), (15, 24, 40), (16, 64, 64), (17, 65, 63), (33, 100, 136), (64, 256, 200),
         (65, 130, 1000), (127, 129, 72), (128, 128, 64), (130, 777, 257), (257, 255, 129), (300, 1000, 128),
         (513, 90, 2051), (1000, 513, 24), (1531, 777, 1000), (4097, 2051, 200), (2300, 2900, 71), (700, 2050, 4104)]


@pytest.mark.parametrize("M,N,K", SIZES, ids=str)
@pytest.mark.parametrize("dtype", [BF, HF], ids=str)
def test_linear_whole_numbers(M, N, K, dtype):
    print("test_linear_whole_numbers", M, N, K, dtype, flush=True)
    dev = _cuda()
    gen = torch.Generator().manual_seed(M + N + K)
    x, w, b, r, dy = whole(gen, M, K), whole(gen, N, K), whole(gen, N), whole(gen, M, N), whole(gen, M, N)
    for act, bias, res in ((None, False, False), (None, True, True), ("relu", True, False)):
        # (the 64-bit sums of whole numbers below 2^24 are those of fp32)
        z = x @ w.T + (b if bias else 0)
        dz = dy if act is None else dy * (z > 0)
        y = (z if act is None else z.relu()) + (r if res else 0)
        xg, wg, rg, dg = (guarded(t, dtype, dev) for t in (x, w, r, dy))
        got, (dx, dw, db, dr) = run(xg, wg, b.to(dev, dtype) if bias else None, act, rg if res else None, dg)
        assert torch.equal(got.cpu(), y.to(dtype)), (act, "y")
        assert torch.equal(dx.cpu(), (dz @ w).to(dtype)), (act, "dx")
        assert torch.equal(dw.cpu(), (dz.T @ x).to(dtype)), (act, "dw")
        if bias:
            assert torch.equal(db.cpu(), dz.sum(0).to(dtype)), (act, "db")
        if res:
            assert torch.equal(dr.cpu(), dy.to(dtype))
        from ccq_amd import fused_linear
        plain = fused_linear(xg, wg, b.to(dev, dtype) if bias else None, act, rg if res else None)
        assert torch.equal(plain, got)


@pytest.mark.parametrize("K", [40, 64, 100, 128, 192, 250, 256, 320, 384, 448, 600], ids=str)
@pytest.mark.parametrize("M,N", [(70, 130), (40000, 48), (2600, 2600)], ids=str)
def test_linear_contraction_lengths(M, N, K):
    """Contractions from part of a step to ten steps, through every number of stages that a tile's operands have in LDS;
    few tiles, many narrow ones and wide ones."""
    print("test_linear_contraction_lengths", M, N, K, flush=True)
    from ccq_amd import fused_linear
    dev = _cuda()
    gen = torch.Generator().manual_seed(M + K)
    x, w, dy = whole(gen, M, K), whole(gen, N, K), whole(gen, M, N)
    xg, wg, dg = (t.to(dev, BF) for t in (x, w, dy))
    got, (dx, dw, _, _) = run(xg, wg, None, None, None, dg)
    assert torch.equal(got.cpu(), (x @ w.T).to(BF))
    assert torch.equal(dx.cpu(), (dy @ w).to(BF))
    assert torch.equal(dw.cpu(), (dy.T @ x).to(BF))
    # the contraction down the rows of both operands, of the same lengths
    a, b = whole(gen, K, 72), whole(gen, K, 136)
    _, (_, dw, _, _) = run(b.to(dev, BF), whole(gen, 72, 136).to(dev, BF), None, None, None, a.to(dev, BF))
    assert torch.equal(dw.cpu(), (a.T @ b).to(BF))
    z = x[:5] @ w.T
    g, u = z.double().chunk(2, -1)
    y = fused_linear(xg[:5], wg, activation="swiglu").cpu().double()
    want = g * torch.sigmoid(g) * u
    # one rounding, and a few units of fp32 of |g| <= 4 K in the exponential
    assert ((y - want).abs() <= torch.finfo(BF).eps / 2 * want.abs() + U32 * 16 * (g.abs() + 1) * (g * u).abs() + 1e-30).all()


@pytest.mark.parametrize("columns", [8, 3], ids=["aligned", "odd"])
@pytest.mark.parametrize("M,N,K", [(40, 96, 64), (200, 131, 72), (2100, 2048, 136)], ids=str)
def test_linear_strided_operands(M, N, K, columns):
    """Views into wider buffers of NaN: nothing of what lies beside the rows comes into a result."""
    print("test_linear_strided_operands", M, N, K, columns, flush=True)
    dev = _cuda()
    gen = torch.Generator().manual_seed(7)
    x, w, r, dy = whole(gen, M, K), whole(gen, N, K), whole(gen, M, N), whole(gen, M, N)
    got, (dx, dw, _, dr) = run(*(guarded(t, BF, dev, columns) for t in (x, w)), None, None, guarded(r, BF, dev, columns),
                               guarded(dy, BF, dev, columns))
    assert torch.equal(got.cpu(), (x @ w.T + r).bfloat16())
    assert torch.equal(dx.cpu(), (dy @ w).bfloat16()) and torch.equal(dw.cpu(), (dy.T @ x).bfloat16())
    assert torch.equal(dr.cpu(), dy.bfloat16())


@pytest.mark.parametrize("M,N,K", [(3, 5, 7), (16, 176, 64), (77, 131, 300), (700, 90, 1000), (1531, 776, 264),
                                   (3000, 1500, 520)], ids=str)
@pytest.mark.parametrize("act", ACTS, ids=str)
def test_linear_activations(M, N, K, act):
    print("test_linear_activations", M, N, K, act, flush=True)
    dev = _cuda()
    outs = 2 * N if act == "swiglu" else N
    for dtype, bdtype in ((BF, BF), (HF, FL)):
        gen = torch.Generator().manual_seed(M + N)
        x, w = torch.randn(M, K, generator=gen).to(dtype), (torch.randn(outs, K, generator=gen) / math.sqrt(K)).to(dtype)
        b, r = torch.randn(outs, generator=gen).to(bdtype), torch.randn(M, N, generator=gen).to(dtype)
        dy = torch.randn(M, N, generator=gen).to(dtype)
        y, z, dz, grads = formula(x, w, b, act, r, dy)
        got, have = run(x.to(dev), w.to(dev), b.to(dev), act, r.to(dev), dy.to(dev))
        u = torch.finfo(dtype).eps / 2
        e = U32 * ((K / 16 + 16) * (x.to(D64).abs() @ w.to(D64).abs().T + b.to(D64).abs()) + 16 * (z.abs() + 1))
        if act == "swiglu":
            gate, up = z.chunk(2, -1)
            e = 1.2 * (e[:, :N] * up.abs() + e[:, N:] * gate.abs())
        bound = u * y.abs() * (1 + u) + 1.2 * e + U32 * r.to(D64).abs() + torch.finfo(dtype).tiny
        off = (got.cpu().double() - y).abs()
        assert (off <= bound).all(), (dtype, (off / bound).max())
        for name, a, want in zip(("dx", "dw", "db", "dr"), have, grads):
            rel = ((a.cpu().double() - want).norm() / want.norm()).item()
            assert rel <= 1.5 * u, (dtype, name, rel)
        # db, in 32 bits: its sum's own error and the roundings of z that its terms carry
        if bdtype == FL:
            term = u * (dy.to(D64).abs().repeat(1, outs // N) * z.abs() * (1 + z.abs().roll(N, 1) if act == "swiglu" else 1))
            bound = term.sum(0) + (M / 16 + 64) * U32 * dz.abs().sum(0) + 1e-6
            assert ((have[2].cpu().double() - grads[2]).abs() <= bound).all()


@pytest.mark.parametrize("M,N,K", [(5, 44, 4200), (20, 130, 8200)], ids=str)
@pytest.mark.parametrize("act", ACTS, ids=str)
def test_linear_few_outputs_of_many_parts(M, N, K, act):
    """Long contractions of few outputs: the forward adds ten parts and more before its epilogue."""
    test_linear_activations(M, N, K, act)


def test_linear_against_differences():
    """Central differences of the 64-bit formula along random directions; whole numbers and fp16, whose dz rounds by
    2^-11 (the bound), truncation h^2 = 1e-8."""
    dev = _cuda()
    gen = torch.Generator().manual_seed(3)
    for act in ACTS:
        outs = 48 if act == "swiglu" else 24
        x, w = torch.randn(10, 16, generator=gen).half(), torch.randn(outs, 16, generator=gen).half() / 4
        b, dy = torch.randn(outs, generator=gen).half(), torch.randn(10, 24, generator=gen).half()
        _, have = run(x.to(dev), w.to(dev), b.to(dev), act, None, dy.to(dev))
        for k, (t, g) in enumerate(zip((x, w, b), have)):
            v = torch.randn(t.shape, generator=gen, dtype=D64)

            def loss(h):
                args = [x.to(D64), w.to(D64), b.to(D64)]
                args[k] = args[k] + h * v
                return (formula(*args, act, None, dy)[0] * dy.to(D64)).sum()

            want = (loss(1e-4) - loss(-1e-4)) / 2e-4
            terms = (g.cpu().double() * v).abs().sum()
            assert abs((g.cpu().double() * v).sum() - want) <= 4 * 2.0 ** -11 * terms, (act, k)


def test_linear_bad_values_stay_in_their_row():
    from ccq_amd import fused_linear
    dev = _cuda()
    gen = torch.Generator().manual_seed(5)
    for M in (20, 300):
        x, w = torch.randn(M, 200, generator=gen).bfloat16(), torch.randn(96, 200, generator=gen).bfloat16()
        good = fused_linear(x.to(dev), w.to(dev), activation="silu")
        x[M - 1, 3] = float("nan")
        x[2, 199] = float("inf")
        got = fused_linear(x.to(dev), w.to(dev), activation="silu")
        rows = [i for i in range(M) if i not in (2, M - 1)]
        assert torch.equal(got[rows], good[rows]) and got[M - 1].isnan().all() and not torch.isfinite(got[2]).all()


def test_linear_extreme_logits():
    """Activations far out: the limits, no NaN from an exponential that overflows."""
    dev = _cuda()
    x = torch.tensor([[1.0, 0.0], [0.0, 1.0], [-1.0, 0.0], [0.0, -1.0]], device=dev).bfloat16()
    w = torch.tensor([[1e4, 80.0], [-300.0, 1e30]], device=dev).bfloat16()
    for act in ("silu", "gelu", "gelu_tanh", "relu", "swiglu"):
        N = 1 if act == "swiglu" else 2
        dy = torch.ones(4, N, device=dev, dtype=BF)
        y, grads = run(x, w, None, act, None, dy)
        want, _, dz, ref = formula(x.cpu(), w.cpu(), None, act, None, dy.cpu())
        assert torch.isfinite(y).all()
        assert torch.allclose(y.cpu().double(), want, rtol=2.0 ** -8, atol=1e-30), act
        assert all(torch.isfinite(g).all() for g in grads if g is not None), act


def test_linear_shapes_and_partial_leaves():
    from ccq_amd import fused_linear
    dev = _cuda()
    gen = torch.Generator().manual_seed(6)
    x, w, b = whole(gen, 24, 40).to(dev, BF), whole(gen, 32, 40).to(dev, BF), whole(gen, 32).to(dev)
    flat = fused_linear(x, w, b)
    assert torch.equal(fused_linear(x.view(2, 3, 4, 40), w, b), flat.view(2, 3, 4, 32))
    assert torch.equal(fused_linear(x[0], w, b), flat[0])
    t = x.view(4, 6, 40).transpose(0, 1)
    assert torch.equal(fused_linear(t, w, b), flat.view(4, 6, 32).transpose(0, 1))
    assert torch.equal(fused_linear(x, w.t().contiguous().t(), b), flat)      # a weight stored the other way
    # no rows
    e = torch.zeros(0, 40, device=dev, dtype=BF)
    y, (dx, dw, db, _) = run(e, w, b, "silu", None, torch.zeros(0, 32, device=dev, dtype=BF))
    assert y.shape == (0, 32) and dx.shape == (0, 40) and (dw == 0).all() and (db == 0).all() and db.dtype == FL
    # one leaf at a time, and the broadcast gradient of a sum
    dz = torch.ones(24, 32)
    for k, want in enumerate((dz @ w.cpu().float(), dz.T @ x.cpu().float(), dz.sum(0), dz)):
        leaves = [x, w, b, torch.zeros(24, 32, device=dev, dtype=BF)]
        leaves[k] = leaves[k].detach().requires_grad_()
        fused_linear(leaves[0], leaves[1], leaves[2], None, leaves[3]).sum().backward()
        assert torch.equal(leaves[k].grad.cpu().float(), want.to(leaves[k].dtype).float()), k


def test_linear_same_bits_again_and_other_stream():
    dev = _cuda()
    gen = torch.Generator().manual_seed(9)
    x, w = torch.randn(900, 600, generator=gen).bfloat16().to(dev), torch.randn(512, 600, generator=gen).bfloat16().to(dev)
    dy = torch.randn(900, 256, generator=gen).bfloat16().to(dev)
    first = run(x, w, None, "swiglu", None, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run(x, w, None, "swiglu", None, dy)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first[0], other[0]) and all(torch.equal(a, b) for a, b in zip(first[1][:2], other[1][:2]))


def test_linear_captured():
    """Forward and backward in two graphs, each with its own workspace, replayed in turn with eager work between."""
    dev = _cuda()

    def inputs(seed, M):
        gen = torch.Generator().manual_seed(seed)
        return [t.to(dev, BF) for t in (torch.randn(M, 264, generator=gen), torch.randn(200, 264, generator=gen) / 16,
                                        torch.randn(200, generator=gen), torch.randn(M, 100, generator=gen))]

    def step(x, w, b, dy):
        y, grads = run(x, w, b, "swiglu", None, dy)
        return [y, *grads[:3]]

    graphs = []
    for M in (24, 700):
        sets = [inputs(i, M) for i in range(3)]
        want = [[t.clone() for t in step(*s)] for s in sets]
        static = [t.clone() for t in sets[0]]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*static)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*static)
        graphs.append((sets, want, static, graph, out))
    for k in (0, 1, 2, 1):
        for sets, want, static, graph, out in graphs:
            for s, t in zip(static, sets[k]):
                s.copy_(t)
            graph.replay()
        torch.cuda.synchronize()
        for sets, want, static, graph, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want[k]))
            step(*sets[0])
        torch.cuda.synchronize()
