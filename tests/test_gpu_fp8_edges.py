"""``ccq_fp8_linear`` at the edges of each way that it runs: strides of outputs, scales far from one, numbers that are not
finite, channels far above the others; norms into 8 bits of more wide rows than workgroups.  Which way a size takes is asserted, as in
``test_gpu_fp8_paths.py``, whose whole numbers these are: outputs have to be equal bit for bit."""

import ctypes

import pytest
import torch

import test_gpu_fp8
from _fp8 import check_rounded, laid_out, linear64, quantized, random_rows, to_device
from test_gpu_fp8_paths import ACTS, BF, CASES, DTYPES, FL, HF, KINDS, _cuda, plan, whole

pytestmark = pytest.mark.gpu


close64 = test_gpu_fp8._close


def _bytes(t):
    return t.contiguous().view(torch.uint8)


def rows8(x):
    """Rows on the CPU in 8 bits, by the definition in 64 bits, laid out with NaN behind their ends."""
    v, s = quantized(x)
    return laid_out(v.float().to(torch.float8_e4m3fn), 16), laid_out(s.float().to(torch.float8_e8m0fnu), 4)


#        M, N, K            act, dtype, way
ROWS = [((5, 300, 1030), None, BF, "0/8"), ((5, 300, 1030), "swiglu", HF, "0/8"), ((33, 4100, 2000), "relu", FL, "0/2"),
        ((900, 300, 600), None, BF, "64"), ((600, 1100, 700), "relu", FL, "64"), ((1100, 520, 90), "swiglu", HF, "64"),
        ((8192, 4096, 300), None, BF, "128"), ((3001, 2101, 250), "swiglu", BF, "128"), ((4500, 8300, 128), "relu", HF, "128"),
        ((16300, 2040, 2100), None, BF, "256"), ((16301, 2047, 4100), "relu", BF, "256"),
        ((16300, 2040, 2100), "swiglu", HF, "256")]


@pytest.mark.parametrize("size,act,dtype,way", ROWS, ids=str)
def test_output_rows_apart(size, act, dtype, way):
    """Rows of y at a stride of their own are those of a contiguous y, and nothing is written between them."""
    from ccq_amd import _lib
    M, N, K = size
    print("test_output_rows_apart", size, act, dtype, flush=True)
    assert plan(M, N, K, act, dtype, 0) == way
    dev, lib = _cuda(), _lib.load()
    gen = torch.Generator().manual_seed(M + N + K)
    x, w = whole(gen, M, K, dev), whole(gen, 2 * N if act == "swiglu" else N, K, dev)
    res = torch.randint(-9, 10, (M, N), generator=gen).to(dtype).to(dev)
    st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)

    def call(y, ldy):
        args = [v for t in (*x, *w) for v in (t.data_ptr(), t.stride(0))]
        assert lib.ccq_fp8_linear(*args, None, 0, res.data_ptr(), N, y.data_ptr(), ldy, None, 0, None, M, N, K, ACTS[act],
                                  DTYPES[dtype], st) == 0

    want = torch.empty(M, N, dtype=dtype, device=dev)
    call(want, N)
    for ldy in (0, N + 1, N + 24):
        big = torch.full((M * max(ldy, N) + 64,), -77.0, dtype=dtype, device=dev)
        call(big, ldy)
        torch.cuda.synchronize()
        rows = big[:M * max(ldy, N)].view(M, -1)
        assert torch.equal(_bytes(rows[:, :N]), _bytes(want)), ldy
        assert bool((rows[:, N:] == -77).all()) and bool((big[M * max(ldy, N):] == -77).all()), ldy


NOT_FINITE = [(1, 129, 4100), (5, 300, 1030), (33, 4100, 2000), (900, 300, 600), (600, 1100, 700), (1100, 520, 90),
              (3001, 2101, 250), (4500, 8300, 128), (16300, 2040, 2100), (16301, 2047, 4100), (16384, 2048, 2176)]


@pytest.mark.parametrize("size", NOT_FINITE, ids=lambda s: "x".join(map(str, s)))
def test_not_finite(size):
    """NaN values and NaN scales of x and of the weight, in first, inner and last tiles and blocks, reach their own row or
    column (of an output in 8 bits: their blocks of it), and every other output keeps its bits."""
    from ccq_amd import fp8_linear
    M, N, K = size
    print("test_not_finite", size, flush=True)
    assert " ".join(plan(M, N, K, *k) for k in KINDS) == dict(CASES)[size]
    dev = _cuda()
    gen = torch.Generator().manual_seed(M + N + K)
    x, w = whole(gen, M, K, dev), whole(gen, 2 * N, K, dev)
    one = type(w)(w.values[:N], w.scales[:N])
    bias = torch.randint(-3, 4, (2 * N,), generator=gen).float()
    gates = bias.clone()
    gates[:N] += 16 * K + 32
    bias, gates = bias.to(dev), gates.to(dev)

    def outputs():
        for act, dtype, into8 in KINDS:
            b, rows = (gates, w) if act == "swiglu" else (bias[:N], one)
            yield (act, into8), fp8_linear(x, rows, b, act, dtype=dtype, quantize=bool(into8))

    clean = list(outputs())
    last = -(-K // 128) - 1
    bad_rows = torch.zeros(M, dtype=torch.bool, device=dev)
    if M > 1:
        for m, k in ((1, K - 1), (M // 2, 0)):
            x.values.view(torch.uint8)[m, k] = 0x7F
            bad_rows[m] = True
        for m, k in ((3, 0), (M - 2, last)):
            x.scales.view(torch.uint8)[m, k] = 255
            bad_rows[m] = True
    bad = torch.zeros(2 * N, dtype=torch.bool, device=dev)
    for n, k in ((7, 0), (N // 2, K - 1), (N + 11, K // 2)):
        w.values.view(torch.uint8)[n, k] = 0xFF
        bad[n] = True
    for n, k in ((N - 1, last), (N // 3, 0), (N + N // 4, last)):
        w.scales.view(torch.uint8)[n, k] = 255
        bad[n] = True
    for (way, was), (_, y) in zip(clean, outputs()):
        print(" ", way, flush=True)
        act, into8 = way
        mask = bad_rows[:, None] | (bad[:N] | bad[N:] if act == "swiglu" else bad[:N])
        if not into8:
            assert torch.equal(torch.isnan(y), mask), way
            assert torch.equal(y[~mask], was[~mask]), way
            continue
        blocks = torch.nn.functional.pad(mask, (0, -N % 128)).unflatten(1, (-1, 128)).any(-1)
        assert torch.equal(_bytes(y.scales) == 255, blocks), way
        assert torch.equal(_bytes(y.scales)[~blocks], _bytes(was.scales)[~blocks]), way
        wide = blocks.repeat_interleave(128, 1)[:, :N]
        assert bool((_bytes(y.values)[wide] == 0x7F).all()), way
        assert torch.equal(_bytes(y.values)[~wide], _bytes(was.values)[~wide]), way


FAR = [((5, 300, 1030), "0/8 0/8 0/8 0/8 0/1 0/1 0/1"), ((1, 129, 4100), "0/8 0/8 0/8 0/8 0/8t 0/8t 0/8t"),
       ((600, 1100, 700), "64 64 64 64 128 0/1 64t"), ((1100, 520, 1300), "64 64 64 64 128 64t 64t"),
       ((2500, 1030, 1152), "64 64 64 64 128 128 64t"), ((3001, 2101, 250), "128 64 128 64 128 128 256"),
       ((16301, 2047, 4100), "256 256 256 64 256 256 256")]


@pytest.mark.parametrize("size,ways", FAR, ids=lambda c: "x".join(map(str, c)) if isinstance(c, tuple) else "")
def test_scales_far_from_one(size, ways):
    """Scales of 2^-55 .. 2^55 on either side, different for every row, column and block, beside blocks of nothing (2^-126,
    as padded rows have them): a row of x has one block that is not zero, so that every output is one block's sum, a whole
    number times a power of two, exact in fp32.  swiglu's gates are their bias, 32 .. 40, where the sigmoid is 1."""
    from ccq_amd import Fp8Rows, fp8_linear, quantize_fp8
    M, N, K = size
    print("test_scales_far_from_one", size, flush=True)
    assert " ".join(plan(M, N, K, *k) for k in KINDS) == ways
    dev = _cuda()
    gen = torch.Generator().manual_seed(M + N + K)
    n = -(-K // 128)

    def powers(rows):
        return torch.randint(127 - 55, 127 + 56, (rows, n), generator=gen).to(torch.uint8)

    own = torch.arange(M) % n
    v = torch.randint(-2, 3, (M, K), generator=gen).float()
    v[(torch.arange(K) // 128)[None] != own[:, None]] = 0
    s = powers(M)
    s[torch.arange(n)[None] != own[:, None]] = 1
    x = Fp8Rows(laid_out(v.to(torch.float8_e4m3fn), 16, dev), laid_out(s.view(torch.float8_e8m0fnu), 4, dev))
    v, s = torch.randint(-2, 3, (2 * N, K), generator=gen).float(), powers(2 * N)
    one = Fp8Rows(laid_out(v[:N].to(torch.float8_e4m3fn), 16, dev), laid_out(s[:N].view(torch.float8_e8m0fnu), 4, dev))
    v[:N], s[:N] = 0, 1
    w = Fp8Rows(laid_out(v.to(torch.float8_e4m3fn), 16, dev), laid_out(s.view(torch.float8_e8m0fnu), 4, dev))
    gates = torch.cat([torch.randint(32, 41, (N,), generator=gen).float(), torch.zeros(N)]).to(dev)
    plain = x.dequantize() @ one.dequantize().T
    gated = gates[:N] * (x.dequantize() @ w.dequantize()[N:].T)
    for act, dtype, into8 in KINDS:
        print(" ", act, dtype, into8, flush=True)
        want = gated if act == "swiglu" else plain.relu() if act else plain
        args = (x, w, gates, act) if act == "swiglu" else (x, one, None, act)
        if not into8:
            assert torch.equal(fp8_linear(*args, dtype=dtype), want.to(dtype)), (act, dtype)
            continue
        y, want = fp8_linear(*args, quantize=True), quantize_fp8(want)
        assert torch.equal(y.dequantize(), want.dequantize()), act   # (-0 and 0 are one number)
        assert torch.equal(_bytes(y.scales), _bytes(want.scales)), act


@pytest.mark.parametrize("size,way", [((5, 300, 1030), "0/8"), ((1100, 520, 1300), "64"), ((2500, 1030, 1152), "64")], ids=str)
def test_exact_sums_of_mixed_scales(size, way):
    """fp32: steps whose scales all lie near one beside steps where a row or a column has one far from it, and blocks of
    nothing, in the same sums."""
    from ccq_amd import Fp8Rows, fp8_linear
    M, N, K = size
    print("test_exact_sums_of_mixed_scales", size, flush=True)
    assert plan(M, N, K, None, FL, 0) == way
    dev = _cuda()
    gen = torch.Generator().manual_seed(M + N + K)
    x, w = random_rows(gen, M, K), random_rows(gen, N, K, K ** -0.5)
    n = -(-K // 128)
    for t, rows in ((x, M), (w, N)):                       # one block of every eighth row: nothing
        m = torch.arange(0, rows, 8)
        k = m // 8 % n
        t[1].view(torch.uint8)[m, k] = 1
        for a, b in zip(m.tolist(), k.tolist()):
            t[0].view(torch.uint8)[a, 128 * b:128 * b + 128] = 0
    m = torch.arange(3, M, 200)                            # some blocks of x large, the weight's there small
    x[1].view(torch.uint8)[m, 2] += 70
    w[1].view(torch.uint8)[torch.arange(0, N, 3), 2] -= 60
    rows = torch.cat([torch.randperm(M, generator=gen)[:150], m])
    want, err = linear64(tuple(t[rows] for t in x), w, exact=True)
    y = fp8_linear(Fp8Rows(*to_device(x, dev)), Fp8Rows(*to_device(w, dev)), dtype=FL)
    close64(y[rows.to(dev)], want, err)


@pytest.mark.parametrize("M,N,K", [(70, 96, 520), (1300, 520, 520)], ids=str)
@pytest.mark.parametrize("how", ["one channel", "two that cancel"])
def test_outlying_channels(M, N, K, how):
    """Channels a thousand times the others: 16-bit outputs within what the 8-bit instruction cuts off, and the sums in fp32,
    from which a caller rounds to 16 or 8 bits by itself, within fp32's additions."""
    from ccq_amd import Fp8Rows, fp8_linear, quantize_fp8
    print("test_outlying_channels", M, N, K, how, flush=True)
    dev = _cuda()
    gen = torch.Generator().manual_seed(M + N + K)
    x = torch.randn(M, K, generator=gen)
    w = torch.randn(N, K, generator=gen) * K ** -0.5
    x[:, 5] *= 1000
    if how == "two that cancel":
        x[:, 70], w[:, 70] = x[:, 5], -w[:, 5]
    x, w = rows8(x), rows8(w)
    xd, wd = Fp8Rows(*to_device(x, dev)), Fp8Rows(*to_device(w, dev))
    res = torch.randn(M, N, generator=gen)
    rows = torch.arange(0, M, max(1, M // 150))
    some = tuple(t[rows] for t in x)
    for dtype in (BF, HF):
        r = res.to(dtype)
        want, err = linear64(some, w, None, None, r[rows])
        close64(fp8_linear(xd, wd, residual=r.to(dev), dtype=dtype)[rows.to(dev)], want, err)
        want, err = linear64(some, w, None, None, r[rows], exact=True)
        y = fp8_linear(xd, wd, residual=r.float().to(dev), dtype=FL)
        close64(y[rows.to(dev)], want, err)
        close64(y.to(dtype)[rows.to(dev)], want, err)
    want, err = linear64(some, w, exact=True)
    q = quantize_fp8(fp8_linear(xd, wd, dtype=FL))
    check_rounded(q.values.cpu()[rows], q.scales.cpu()[rows], want, err)


@pytest.mark.parametrize("residual", [False, True], ids=["", "residual"])
@pytest.mark.parametrize("dtype,rows,D", [(FL, 1100, 5003), (FL, 1100, 8192), (FL, 520, 4100), (BF, 2500, 8191)], ids=str)
def test_more_wide_rows_than_workgroups(dtype, rows, D, residual):
    """Norms into 8 bits of sixteen waves a row (fp32 above 4096 columns) and of four with four pieces a lane, each workgroup
    over several rows."""
    test_gpu_fp8.test_norm(rows, D, dtype, FL, residual)
