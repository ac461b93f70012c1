"""quantize_fp8, rms_norm_fp8 and fp8_linear against their definitions in 64 bits."""

import pytest
import torch

from _fp8 import check_rounded, laid_out, linear64, meant, quantized, random_rows, to_device

pytestmark = pytest.mark.gpu

BF, HF, FL = torch.bfloat16, torch.float16, torch.float32
NAN8, NAN_SCALE = 0x7F, 255


def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda")


def _bytes(t):
    return t.cpu().contiguous().view(torch.uint8)


# ---- quantize_fp8 ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF, HF, FL], ids=str)
@pytest.mark.parametrize("rows,D", [(1, 1), (3, 7), (5, 128), (4, 129), (17, 300), (9, 512), (2, 777), (3, 4100), (130, 64)],
                         ids=str)
def test_quantize(rows, D, dtype):
    from ccq_amd import quantize_fp8
    dev = _cuda()
    gen = torch.Generator().manual_seed(rows * 10000 + D)
    x = (torch.randn(rows, D, generator=gen) * torch.exp(2 * torch.randn(rows, 1, generator=gen))).to(dtype)
    x[0, : D // 2] = 0
    q = quantize_fp8(x.to(dev))
    assert q.values.shape == x.shape and q.scales.shape == (rows, -(-D // 128))
    v, s = quantized(x)
    assert torch.equal(q.values.cpu().double(), v) and torch.equal(q.scales.cpu().double(), s)
    assert torch.equal(q.dequantize().cpu().double(), v * s.repeat_interleave(128, -1)[:, :D])


def test_quantize_borders():
    """Largest magnitudes at the borders of scales, ties between values, the smallest and largest numbers."""
    from ccq_amd import quantize_fp8
    dev = _cuda()
    up = torch.nextafter(torch.tensor(448.0), torch.tensor(1e9)).item()
    most = [448.0, up, 447.9, 1.75, 3.5, 3.4e38, 1e-38, 2.0 ** -126, 1e-45, 448 * 2.0 ** -126, 1.0, 0.0]
    x = torch.zeros(len(most), 256)
    x[:, 3] = torch.tensor(most)
    x[:, 128] = -torch.tensor(most)
    ties = torch.arange(1, 120).float()  # of e4m3 values and halfway between them, in a block that 448 leads
    x = torch.cat([x, torch.zeros(2, 256)])
    x[-1, :119], x[-1, 127] = ties + 0.5, -448
    x[-2, :119], x[-2, 127] = ties * 2.0 ** -10, 448
    q = quantize_fp8(x.to(dev))
    v, s = quantized(x)
    assert torch.equal(q.values.cpu().double(), v) and torch.equal(q.scales.cpu().double(), s)


def test_quantize_strides_and_shapes():
    from ccq_amd import quantize_fp8
    dev = _cuda()
    gen = torch.Generator().manual_seed(5)
    wide = torch.randn(2, 6, 500, generator=gen).to(BF).to(dev)
    for x in (wide[:, :, 1:302], wide[:, ::2, :200], wide.transpose(0, 1), wide[1, 2], wide[:, :0], wide[..., ::2]):
        q, want = quantize_fp8(x), quantize_fp8(x.contiguous())
        assert q.values.shape == x.shape and q.scales.shape == (*x.shape[:-1], -(-x.shape[-1] // 128))
        assert torch.equal(_bytes(q.values), _bytes(want.values)) and torch.equal(_bytes(q.scales), _bytes(want.scales))
        if x.numel():
            v, s = quantized(x.cpu())
            assert torch.equal(q.values.cpu().double(), v) and torch.equal(q.scales.cpu().double(), s)


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")], ids=str)
@pytest.mark.parametrize("dtype", [BF, HF, FL], ids=str)
def test_quantize_not_finite(dtype, bad):
    from ccq_amd import quantize_fp8
    dev = _cuda()
    x = torch.ones(3, 400).to(dtype)
    x[1, 200] = bad
    x[2, 399] = bad
    q = quantize_fp8(x.to(dev))
    v, s = _bytes(q.values), _bytes(q.scales)
    at = torch.zeros(3, 400, dtype=torch.bool)
    at[1, 128:256] = at[2, 384:] = True
    assert bool((v[at] == NAN8).all()) and bool((v[~at] != NAN8).all())
    assert s.eq(NAN_SCALE).tolist() == [[False] * 4, [False, True, False, False], [False, False, False, True]]


# ---- rms_norm_fp8 ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("residual", [False, True], ids=["", "residual"])
@pytest.mark.parametrize("dtype,wdtype", [(BF, BF), (BF, FL), (HF, HF), (FL, FL)], ids=str)
@pytest.mark.parametrize("rows,D", [(1, 1), (3, 5), (7, 48), (33, 128), (5, 130), (9, 511), (4, 777), (17, 1024), (3, 2048),
                                    (2, 4100), (3, 8192)], ids=str)
def test_norm(rows, D, dtype, wdtype, residual):
    """fp32: a sum of D squares within (D + 2) 2^-24 of itself, its root half of that, and four roundings behind."""
    from ccq_amd import rms_norm_fp8
    dev = _cuda()
    gen = torch.Generator().manual_seed(rows * 10000 + D)
    x = (torch.randn(rows, D, generator=gen) * torch.exp(torch.randn(D, generator=gen))).to(dtype)
    w = (1 + 0.3 * torch.randn(D, generator=gen)).to(wdtype)
    r = torch.randn(rows, D, generator=gen).to(dtype) if residual else None
    got = rms_norm_fp8(x.to(dev), w.to(dev), residual=None if r is None else r.to(dev))
    s = x
    if residual:
        got, stream = got
        s = (x.float() + r.float()).to(dtype)
        assert torch.equal(stream.cpu(), s)
    y = s.double() / torch.sqrt(s.double().square().mean(-1, keepdim=True) + 1e-5) * w.double()
    check_rounded(got.values, got.scales, y, ((D + 2) / 2 + 6) * 2.0 ** -24 * y.abs())


@pytest.mark.parametrize("residual", [False, True], ids=["", "residual"])
@pytest.mark.parametrize("dtype,rows,D", [(BF, 5, 4104), (HF, 3, 7271), (FL, 3, 2052), (FL, 2, 4096), (FL, 2, 5003), (BF, 1500, 5000)],
                         ids=str)
def test_norm_wide(dtype, rows, D, residual):
    """Rows of more than two pieces a lane, and more of them than workgroups."""
    test_norm(rows, D, dtype, FL, residual)


def test_norm_without_weight_strides_and_other_shapes():
    from ccq_amd import quantize_fp8, rms_norm, rms_norm_fp8
    dev = _cuda()
    gen = torch.Generator().manual_seed(6)
    wide = torch.randn(2, 6, 500, generator=gen).to(dev)
    for x in (wide[:, :, 1:302], wide[:, ::2, :200], wide.transpose(0, 1), wide[1, 2], wide[:, :0]):
        q = rms_norm_fp8(x)
        want = quantize_fp8(rms_norm(x))  # (rows in fp32: the norm's result as it is)
        assert q.values.shape == x.shape and torch.equal(_bytes(q.values), _bytes(want.values))
        assert torch.equal(_bytes(q.scales), _bytes(want.scales))


def test_norm_of_nothing_and_not_finite():
    from ccq_amd import rms_norm_fp8
    dev = _cuda()
    x = torch.randn(4, 300, generator=torch.Generator().manual_seed(7)).to(BF)
    x[1] = 0
    x[2, 7] = float("nan")
    q = rms_norm_fp8(x.to(dev))
    v, s = _bytes(q.values), _bytes(q.scales)
    assert bool((v[1] == 0).all()) and bool((s[1] == 1).all())        # 2^-126: the least scale
    assert bool((v[2] == NAN8).all()) and bool((s[2] == NAN_SCALE).all())
    assert bool((s[[0, 3]] != NAN_SCALE).all())


# ---- fp8_linear ------------------------------------------------------------------------------------------------

def _close(y, want, err):
    half = torch.finfo(y.dtype).eps / 2
    off = (y.cpu().double() - want).abs()
    room = err + half * (want.abs() + err) + torch.finfo(y.dtype).tiny
    bad = off > room
    assert not bool(bad.any()), (int(bad.sum()), float((off / room).max()), torch.nonzero(bad)[:4].tolist())


SIZES = [(1, 1, 1), (1, 16, 128), (3, 5, 15), (16, 77, 16), (17, 64, 129), (5, 128, 640), (64, 65, 300), (65, 200, 100),
         (130, 131, 513), (16, 320, 1024), (33, 48, 2000), (300, 257, 384), (1, 1000, 777), (128, 128, 4096)]


@pytest.mark.parametrize("M,N,K", SIZES, ids=str)
def test_linear(M, N, K):
    from ccq_amd import Fp8Rows, fp8_linear
    print("test_linear", M, N, K, flush=True)
    dev = _cuda()
    gen = torch.Generator().manual_seed(M * 1000000 + N * 1000 + K)
    x, w = random_rows(gen, M, K), random_rows(gen, N, K, K ** -0.5)
    xd, wd = Fp8Rows(*to_device(x, dev)), Fp8Rows(*to_device(w, dev))
    for dtype in (FL, BF, HF):
        want, err = linear64(x, w, exact=dtype == FL)
        y = fp8_linear(xd, wd, dtype=dtype)
        assert y.shape == (M, N) and y.dtype == dtype
        _close(y, want, err)


@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu", "gelu_tanh", "swiglu"])
@pytest.mark.parametrize("M,N,K", [(5, 24, 200), (16, 130, 128), (70, 96, 333), (200, 300, 64)], ids=str)
def test_linear_epilogue(M, N, K, act):
    from ccq_amd import Fp8Rows, fp8_linear
    print("test_linear_epilogue", M, N, K, act, flush=True)
    dev = _cuda()
    gen = torch.Generator().manual_seed(M * 1000000 + N * 1000 + K)
    outs = 2 * N if act == "swiglu" else N
    x, w = random_rows(gen, M, K), random_rows(gen, outs, K, K ** -0.5)
    xd, wd = Fp8Rows(*to_device(x, dev)), Fp8Rows(*to_device(w, dev))
    for dtype, btype in ((FL, FL), (BF, BF), (HF, FL)):
        bias = torch.randn(outs, generator=gen).to(btype)
        res = torch.randn(M, N, generator=gen).to(dtype)
        for b, r in ((bias, None), (None, res), (bias, res)):
            want, err = linear64(x, w, b, act, r, exact=dtype == FL)
            y = fp8_linear(xd, wd, None if b is None else b.to(dev), act, None if r is None else r.to(dev), dtype)
            _close(y, want, err)


@pytest.mark.parametrize("act", [None, "relu", "gelu", "swiglu"])
@pytest.mark.parametrize("M,N,K", [(1, 1, 100), (4, 100, 200), (16, 128, 256), (40, 300, 130), (300, 700, 640)], ids=str)
def test_linear_into_8_bits(M, N, K, act):
    from ccq_amd import Fp8Rows, fp8_linear
    print("test_linear_into_8_bits", M, N, K, act, flush=True)
    dev = _cuda()
    gen = torch.Generator().manual_seed(M * 1000000 + N * 1000 + K)
    outs = 2 * N if act == "swiglu" else N
    x, w = random_rows(gen, M, K), random_rows(gen, outs, K, K ** -0.5)
    bias = torch.randn(outs, generator=gen)
    y = fp8_linear(Fp8Rows(*to_device(x, dev)), Fp8Rows(*to_device(w, dev)), bias.to(dev), act, quantize=True)
    assert y.values.shape == (M, N) and y.scales.shape == (M, -(-N // 128))
    want, err = linear64(x, w, bias, act)
    check_rounded(y.values, y.scales, want, err)


@pytest.mark.parametrize("act", [None, "silu", "swiglu"])
@pytest.mark.parametrize("M,N,K", [(2051, 4097, 300), (4100, 1030, 1000)], ids=str)
def test_linear_of_many_tiles(M, N, K, act):
    """As many tiles as large calls have; rows and columns sampled for the definition."""
    from ccq_amd import Fp8Rows, fp8_linear
    print("test_linear_of_many_tiles", M, N, K, act, flush=True)
    dev = _cuda()
    gen = torch.Generator().manual_seed(M + K)
    outs = 2 * N if act == "swiglu" else N
    x, w = random_rows(gen, M, K), random_rows(gen, outs, K, K ** -0.5)
    rows = torch.cat([torch.randperm(M, generator=gen)[:10], torch.tensor([0, M - 1])])
    res = torch.randn(M, N, generator=gen).to(BF)
    xd, wd = Fp8Rows(*to_device(x, dev)), Fp8Rows(*to_device(w, dev))
    for dtype in (BF, FL):
        want, err = linear64(tuple(t[rows] for t in x), w, None, act, res[rows], exact=dtype == FL)
        y = fp8_linear(xd, wd, activation=act, residual=res.to(dev, dtype), dtype=dtype)
        _close(y[rows.to(dev)], want, err)
    q = fp8_linear(xd, wd, activation=act, quantize=True)
    want, err = linear64(tuple(t[rows] for t in x), w, None, act)
    check_rounded(q.values.cpu()[rows], q.scales.cpu()[rows], want, err)


def test_linear_scales_apart():
    """Scales over the whole range where their product is one fp32 holds: e4m3 ones stand for 2^a and 2^b."""
    from ccq_amd import Fp8Rows, fp8_linear
    dev = _cuda()
    K = 1100
    one = torch.ones(254, K).to(torch.float8_e4m3fn)
    scales = torch.arange(1, 255, dtype=torch.uint8)[:, None].expand(254, 9).contiguous().view(torch.float8_e8m0fnu)
    want = K * torch.exp2(torch.arange(1, 255).double() - 127)[:, None] * torch.exp2(torch.arange(1, 255).double() - 127)
    fits = (want >= 2.0 ** -126 * K) & (want < 2.0 ** 128)
    rows = Fp8Rows(one.to(dev), scales.to(dev))
    for dtype in (FL, BF):
        y = fp8_linear(rows, rows, dtype=dtype).cpu().double()
        assert torch.equal(y[fits], want.to(dtype)[fits].double())
        assert bool(torch.isinf(y[want >= 2.0 ** 128]).all())
        assert bool((y[want < 2.0 ** -126] <= 2.0 ** -126 * K).all())


def test_linear_block_by_block():
    """Every block's scales count for that block alone: one block of x not zero at a time, scales all different."""
    from ccq_amd import Fp8Rows, fp8_linear
    dev = _cuda()
    K, M, N = 1000, 20, 70
    n = -(-K // 128)
    gen = torch.Generator().manual_seed(8)
    w = random_rows(gen, N, K)
    v = torch.zeros(n * M, K)
    for b in range(n):
        part = v[b * M:(b + 1) * M, b * 128:(b + 1) * 128]
        part += torch.randint(-8, 9, part.shape, generator=gen)
    e = torch.randint(-20, 21, (n * M, n), generator=gen)
    x = (laid_out(v.to(torch.float8_e4m3fn), 16), laid_out(torch.exp2(e.float()).to(torch.float8_e8m0fnu), 4))
    for dtype in (FL, BF):
        want, err = linear64(x, w, exact=dtype == FL)
        _close(fp8_linear(Fp8Rows(*to_device(x, dev)), Fp8Rows(*to_device(w, dev)), dtype=dtype), want, err)


def test_linear_not_finite():
    """A NaN value and a NaN scale reach their own row (x) or column (weight), nothing else."""
    from ccq_amd import Fp8Rows, fp8_linear
    dev = _cuda()
    gen = torch.Generator().manual_seed(9)
    for M, N, K in ((5, 40, 300), (300, 130, 520)):
        x, w = random_rows(gen, M, K), random_rows(gen, N, K)
        x[0].view(torch.uint8)[1, K - 1] = NAN8
        x[1].view(torch.uint8)[3, 0] = NAN_SCALE
        w[0].view(torch.uint8)[7, 0] = 0xFF
        w[1].view(torch.uint8)[N - 1, K // 128] = NAN_SCALE
        bad = torch.zeros(M, N, dtype=torch.bool)
        bad[[1, 3]] = True
        bad[:, [7, N - 1]] = True
        for dtype in (FL, HF):
            y = fp8_linear(Fp8Rows(*to_device(x, dev)), Fp8Rows(*to_device(w, dev)), dtype=dtype)
            assert torch.equal(torch.isnan(y.cpu()), bad)
        q = fp8_linear(Fp8Rows(*to_device(x, dev)), Fp8Rows(*to_device(w, dev)), quantize=True)
        blocks = torch.nn.functional.pad(bad, (0, -N % 128)).unflatten(1, (-1, 128)).any(-1)
        assert torch.equal(_bytes(q.scales) == NAN_SCALE, blocks)


def test_linear_layouts():
    """Views of wider rows with NaN behind them, rows apart, leading dimensions, single rows, tensors from anywhere: the same
    numbers, the same bits."""
    from ccq_amd import Fp8Rows, fp8_linear
    dev = _cuda()
    gen = torch.Generator().manual_seed(10)
    M, N, K = 24, 40, 203
    x, w = random_rows(gen, M, K), random_rows(gen, N, K)
    want, err = linear64(x, w, exact=True)
    xd, wd = Fp8Rows(*to_device(x, dev)), Fp8Rows(*to_device(w, dev))
    y = fp8_linear(xd, wd, dtype=FL)
    _close(y, want, err)

    def put(t, room, at, step):
        big = torch.full((t.shape[0] * step + 3, room), 255, dtype=torch.uint8, device=dev)
        view = big[1:1 + t.shape[0] * step:step, at:at + t.shape[1]]
        view.copy_(t.view(torch.uint8))
        return view.view(t.dtype)

    for room, at, step in ((256, 32, 1), (256, 32, 2), (240, 0, 3), (230, 3, 1), (203, 0, 1)):
        a = Fp8Rows(put(x[0], room, at, step), put(x[1], 8, at % 8, step))
        b = Fp8Rows(put(w[0], room, at, step), put(w[1], 5, at % 4, step))
        assert torch.equal(fp8_linear(a, b, dtype=FL), y)
    tight = Fp8Rows(x[0].contiguous().to(dev), x[1].contiguous().to(dev))
    assert torch.equal(fp8_linear(tight, Fp8Rows(w[0].contiguous().to(dev), w[1].contiguous().to(dev)), dtype=FL), y)
    lead = Fp8Rows(xd.values.unflatten(0, (2, 3, 4)), xd.scales.unflatten(0, (2, 3, 4)))
    assert torch.equal(fp8_linear(lead, wd, dtype=FL), y.unflatten(0, (2, 3, 4)))
    part = Fp8Rows(lead.values[:, 1], lead.scales[:, 1])
    assert torch.equal(fp8_linear(part, wd, dtype=FL), y.unflatten(0, (2, 3, 4))[:, 1])
    assert torch.equal(fp8_linear(Fp8Rows(xd.values[3], xd.scales[3]), wd, dtype=FL), y[3])
    none = fp8_linear(Fp8Rows(xd.values[:0], xd.scales[:0]), wd)
    assert none.shape == (0, N)
    res = torch.randn(M, 3 * N, generator=gen).to(dev)[:, N:2 * N]
    assert torch.equal(fp8_linear(xd, wd, residual=res, dtype=FL), fp8_linear(xd, wd, residual=res.contiguous(), dtype=FL))
