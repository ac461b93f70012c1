"""The ways in which ``ccq_amd.fp8_linear`` runs - a few rows in parts of the contraction, tiles of 64, 128 and 256, outputs
in 8 bits written at once and through fp32 - at odd ends, and the operators as serving runs them: one after another,
captured and replayed, on two streams, on rows that lie past 32-bit offsets.  Which way a size takes is asked of the library
and asserted, so that a change of the rule names the cases that it takes out.

Whole numbers in blocks of different scales: every product and sum is a multiple of 1/4 below 2^22, so exact in fp32 in any
order, and no eight products are so far apart that the matrix instruction cuts bits off.  Outputs have to be equal bit for
bit.  swiglu's gates get a bias that leaves them at 32 and more, where the sigmoid is 1 in fp32 (1 + e^-32 rounds to 1).
"""

import ctypes

import pytest
import torch

from _fp8 import check_rounded, laid_out, linear64, random_rows, to_device

pytestmark = pytest.mark.gpu

BF, HF, FL = torch.bfloat16, torch.float16, torch.float32
DTYPES = {BF: 0, HF: 1, FL: 2}
ACTS = {None: 0, "relu": 1, "swiglu": 5}


def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda", 0)


def plan(M, N, K, act, dtype, into8):
    from ccq_amd import _lib
    side, parts, through = ctypes.c_int(), ctypes.c_int(), ctypes.c_int()
    assert _lib.load().ccq_fp8_linear_plan(M, N, K, ACTS[act], DTYPES[dtype], into8, ctypes.byref(side),
                                           ctypes.byref(parts), ctypes.byref(through)) == 0
    return (str(side.value) if side.value else f"0/{parts.value}") + "t" * through.value


def whole(gen, rows, K, dev):
    """Whole numbers times 1/2, 1 or 2, block by block, as 8-bit rows laid out with NaN behind their ends."""
    from ccq_amd import Fp8Rows
    v = torch.randint(-2, 3, (rows, K), generator=gen).to(torch.float8_e4m3fn)
    s = torch.exp2(torch.randint(-1, 2, (rows, -(-K // 128)), generator=gen).float()).to(torch.float8_e8m0fnu)
    return Fp8Rows(laid_out(v, 16, dev), laid_out(s, 4, dev))


KINDS = [(None, BF, 0), ("relu", BF, 0), ("swiglu", BF, 0), (None, FL, 0), (None, BF, 1), ("relu", BF, 1), ("swiglu", BF, 1)]
#         M, N, K             how the KINDS run
CASES = [((3, 37, 1000), "0/8 0/8 0/8 0/8 0/1 0/1 0/1"),
         ((5, 300, 1030), "0/8 0/8 0/8 0/8 0/1 0/1 0/1"),
         ((30, 1030, 513), "64 0/4 64 0/4 0/1 0/1 0/1"),
         ((33, 4100, 2000), "0/2 0/2 64 0/2 0/1 0/1 0/1"),
         ((900, 300, 600), "64 64 64 0/1 0/1 0/1 0/1"),
         ((250, 530, 300), "64 64 64 0/2 0/1 0/1 0/1"),
         ((600, 1100, 700), "64 64 64 64 128 0/1 64t"),
         ((1, 129, 4100), "0/8 0/8 0/8 0/8 0/8t 0/8t 0/8t"),
         ((1100, 520, 90), "64 64 64 64 128 128 64t"),
         ((3001, 2101, 250), "128 64 128 64 128 128 256"),
         ((4363, 2188, 959), "128 64 128 64 128 128 256"),
         ((4500, 8300, 128), "128 128 128 64 128 128 256"),
         ((5000, 4100, 256), "128 64 128 64 128 128 256"),
         ((2561, 6150, 385), "128 64 128 64 128 128 256"),
         ((16300, 2040, 2100), "256 128 256 64 256 128 256"),
         ((16301, 2047, 4100), "256 256 256 64 256 256 256"),
         ((16384, 2048, 2176), "256 256 256 64 256 256 256"),
         ((8190, 4097, 1100), "128 128 128 64 128 128 256"),
         ((16384, 4096, 1040), "256 128 256 64 256 128 256"),
         ((8192, 4096, 300), "128 128 128 64 128 128 256")]


@pytest.mark.parametrize("size,ways", CASES, ids=lambda c: "x".join(map(str, c)) if isinstance(c, tuple) else "")
def test_ways(size, ways):
    from ccq_amd import fp8_linear, quantize_fp8
    M, N, K = size
    print("test_ways", size, flush=True)
    assert " ".join(plan(M, N, K, *k) for k in KINDS) == ways
    dev = _cuda()
    gen = torch.Generator().manual_seed(M + N + K)
    x, w = whole(gen, M, K, dev), whole(gen, 2 * N, K, dev)
    bias = torch.randint(-3, 4, (2 * N,), generator=gen).float()
    gates = bias.clone()
    gates[:N] += 16 * K + 32
    bias, gates = bias.to(dev), gates.to(dev)
    res = torch.randint(-9, 10, (M, N), generator=gen).float().to(dev)
    z = x.dequantize() @ w.dequantize().T
    one = type(w)(w.values[:N], w.scales[:N])
    for act, dtype, into8 in KINDS:
        print(" ", act, dtype, into8, flush=True)
        b = gates if act == "swiglu" else bias[:N]
        want = z + gates if act == "swiglu" else z[:, :N] + b
        want = want[:, :N] * want[:, N:] if act == "swiglu" else want.relu() if act else want
        if into8:
            y, want = fp8_linear(x, w if act == "swiglu" else one, b, act, quantize=True), quantize_fp8(want)
            assert torch.equal(y.values.view(torch.uint8), want.values.view(torch.uint8)), (act, "values")
            assert torch.equal(y.scales.view(torch.uint8), want.scales.view(torch.uint8)), (act, "scales")
            continue
        for t in {dtype, HF if dtype == BF and act != "swiglu" else dtype}:
            if act != "swiglu":  # (its products are rounded, or taken into the sum unrounded)
                assert torch.equal(fp8_linear(x, one, b, act, res.to(t), t), (want + res).to(t)), (act, t)
            y = fp8_linear(x, w if act == "swiglu" else one, b, act, dtype=t)
            assert torch.equal(y, want.to(t)), (act, t, "no residual")


@pytest.mark.parametrize("M,N,K", [(3, 37, 1000), (33, 523, 300), (300, 260, 200), (1100, 520, 90), (3001, 2101, 250),
                                   (4363, 1100, 513)], ids=str)
@pytest.mark.parametrize("act", ["none", "swiglu"])
def test_nothing_else_is_written(M, N, K, act):
    """What lies around y and, beyond a row's 16 (scales: 4) bytes, between its rows."""
    from ccq_amd import _lib
    print("test_nothing_else_is_written", M, N, K, act, flush=True)
    dev, lib = _cuda(), _lib.load()
    gen = torch.Generator().manual_seed(M + K)
    outs, code = (2 * N, 5) if act == "swiglu" else (N, 0)
    x, w = whole(gen, M, K, dev), whole(gen, outs, K, dev)
    st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)

    def call(y, ldy, ys, ldys, dtype, into8):
        room = lib.ccq_fp8_linear_workspace_bytes(M, N, K, code, dtype, into8)
        ws = torch.empty(max(room, 16), dtype=torch.uint8, device=dev)
        args = [v for t in (*x, *w) for v in (t.data_ptr(), t.stride(0))]
        assert lib.ccq_fp8_linear(*args, None, 0, None, 0, y, ldy, ys, ldys, ws.data_ptr(), M, N, K, code, dtype, st) == 0
        torch.cuda.synchronize()

    for dtype, size in ((0, 2), (2, 4)):
        big = torch.full((M * N * size + 512,), 0xA5, dtype=torch.uint8, device=dev)
        call(big.data_ptr() + 256, N, None, 0, dtype, 0)
        assert bool((big[:256] == 0xA5).all()) and bool((big[256 + M * N * size:] == 0xA5).all())
    n16, blocks = -(-N // 16) * 16, -(-N // 128)
    n4 = -(-blocks // 4) * 4
    big = torch.full((M + 2, n16 + 48), 0xA5, dtype=torch.uint8, device=dev)
    scales = torch.full((M + 2, n4 + 4), 0xA5, dtype=torch.uint8, device=dev)
    call(big[1].data_ptr() + 16, n16 + 48, scales[1].data_ptr(), n4 + 4, 0, 1)
    assert bool((big[[0, -1]] == 0xA5).all()) and bool((big[1:-1, :16] == 0xA5).all())
    assert bool((big[1:-1, 16 + n16:] == 0xA5).all())
    assert bool((scales[[0, -1]] == 0xA5).all()) and bool((scales[1:-1, n4:] == 0xA5).all())


def _mlp(x, weight, up, down, residual):
    from ccq_amd import fp8_linear, rms_norm_fp8
    h, s = rms_norm_fp8(x, weight, 1e-6, residual)
    a = fp8_linear(h, up, activation="swiglu", quantize=True)
    return fp8_linear(a, down, residual=s), h, s, a


def _mlp_inputs(gen, M, D, H, dev):
    from ccq_amd import Fp8Rows
    x, r = (torch.randn(M, D, generator=gen).to(BF) for _ in range(2))
    weight = (1 + 0.1 * torch.randn(D, generator=gen)).to(BF)
    up, down = random_rows(gen, 2 * H, D, D ** -0.5), random_rows(gen, D, H, H ** -0.5)
    return x, r, weight, up, down, [t.to(dev) for t in (x, r, weight)], Fp8Rows(*to_device(up, dev)), Fp8Rows(*to_device(down, dev))


@pytest.mark.parametrize("M,D,H", [(1, 256, 700), (7, 200, 333), (65, 256, 384), (1100, 130, 260)], ids=str)
def test_a_layer(M, D, H):
    """Norm of the stream, up with swiglu, down with the stream added: each step in 64 bits of what the last one left."""
    print("test_a_layer", M, D, H, flush=True)
    dev = _cuda()
    gen = torch.Generator().manual_seed(M + D)
    x, r, weight, up, down, (xd, rd, wd), upd, downd = _mlp_inputs(gen, M, D, H, dev)
    y, h, s, a = _mlp(xd, wd, upd, downd, rd)
    assert torch.equal(s.cpu(), (x.float() + r.float()).to(BF))
    # fp32: a sum of D squares within (D + 2) 2^-24 of itself, its root half of that, and four roundings behind
    n = s.cpu().double()
    n = n / torch.sqrt(n.square().mean(-1, keepdim=True) + 1e-6) * weight.double()
    check_rounded(h.values, h.scales, n, ((D + 2) / 2 + 6) * 2.0 ** -24 * n.abs())
    want, err = linear64(tuple(t.cpu() for t in h), up, None, "swiglu")
    check_rounded(a.values, a.scales, want, err)
    want, err = linear64(tuple(t.cpu() for t in a), down, None, None, s.cpu())
    assert bool(((y.cpu().double() - want).abs() <= err + 2.0 ** -8 * (want.abs() + err)).all())


@pytest.mark.parametrize("sizes", [((4, 256, 700), (2, 200, 1400)), ((300, 512, 700), (700, 400, 690))], ids=str)
def test_captured_and_replayed(sizes):
    """Two captured layers replayed in turn, new inputs in their tensors and eager work of the same kind between."""
    print("test_captured_and_replayed", sizes, flush=True)
    dev = _cuda()
    gen = torch.Generator().manual_seed(5)
    graphs = []
    for M, D, H in sizes:
        *_, (x, r, weight), up, down = _mlp_inputs(gen, M, D, H, dev)
        sets = [[torch.randn(M, D, generator=gen).to(BF).to(dev) for _ in range(2)] for _ in range(3)]
        _mlp(x, weight, up, down, r)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _mlp(x, weight, up, down, r)[0]
        graphs.append((sets, x, r, weight, up, down, graph, out))
    for k in range(3):
        for sets, x, r, weight, up, down, graph, out in graphs:
            x.copy_(sets[k][0])
            r.copy_(sets[k][1])
            graph.replay()
        for sets, x, r, weight, up, down, graph, out in graphs:
            want = _mlp(sets[k][0], weight, up, down, sets[k][1])[0]
            torch.cuda.synchronize()
            assert torch.equal(out, want), k


@pytest.mark.parametrize("M,D,H", [(4, 256, 700), (700, 400, 690)], ids=str)
def test_two_streams(M, D, H):
    """The same layer on two other streams at once leaves on each what it leaves alone."""
    print("test_two_streams", M, D, H, flush=True)
    dev = _cuda()
    gen = torch.Generator().manual_seed(6)
    *_, (x, r, weight), up, down = _mlp_inputs(gen, M, D, H, dev)
    want = [_mlp(a, weight, up, down, b)[0] for a, b in ((x, r), (r, x))]
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[k].append(_mlp(*((x, weight, up, down, r) if k == 0 else (r, weight, up, down, x)))[0])
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(y, want[k]) for y in outs[k])


def test_rows_past_32_bits():
    """Rows of x, of the weight and of the outputs whose bytes lie past 2^31 and 2^32: as the same rows alone."""
    from ccq_amd import Fp8Rows, fp8_linear, quantize_fp8, rms_norm_fp8
    print("test_rows_past_32_bits", flush=True)
    dev = _cuda()
    M, K, step = 70001, 256, 65536                             # 4.6 GB of values
    gen = torch.Generator().manual_seed(7)
    few = whole(gen, 97, K, dev)
    big = torch.zeros(M, step, dtype=torch.uint8, device=dev)
    scales = torch.full((M, 4), 255, dtype=torch.uint8, device=dev)
    at = torch.cat([torch.arange(64), torch.arange(M - 33, M)]).to(dev)
    scales[:, :2] = 127
    big[at, :K] = few.values.view(torch.uint8)
    scales[at, :2] = few.scales.view(torch.uint8)
    far = Fp8Rows(big.view(torch.float8_e4m3fn)[:, :K], scales.view(torch.float8_e8m0fnu)[:, :2])
    w = whole(gen, 40, K, dev)
    assert torch.equal(fp8_linear(far, w, dtype=FL)[at], fp8_linear(few, w, dtype=FL))
    assert torch.equal(fp8_linear(far, w)[at], fp8_linear(few, w))
    q, want = fp8_linear(far, w, quantize=True), fp8_linear(few, w, quantize=True)
    assert torch.equal(q.values.view(torch.uint8)[at], want.values.view(torch.uint8))
    # as a weight: of few rows and of many
    for rows in (3, 300):
        x = whole(gen, rows, K, dev)
        assert torch.equal(fp8_linear(x, far)[:, at], fp8_linear(x, few))
    # an output of 4.6 GB
    w = whole(gen, 33000, K, dev)
    y = fp8_linear(far, w)
    assert y.numel() * 2 > 2 ** 32 and torch.equal(y[at], fp8_linear(few, w))
    del y, big, far
    # rows to quantise and to norm, columns of a wide buffer
    rows = torch.zeros(M, 33000, dtype=BF, device=dev)
    some = torch.randn(97, 300, generator=gen).to(BF).to(dev)
    rows[at, 32700:] = some
    view = rows[:, 32700:]
    q, n = quantize_fp8(view), rms_norm_fp8(view)
    for got, want in ((q, quantize_fp8(some)), (n, rms_norm_fp8(some))):
        assert torch.equal(got.values.view(torch.uint8)[at], want.values.view(torch.uint8))
        assert torch.equal(got.scales.view(torch.uint8)[at], want.scales.view(torch.uint8))
