"""Refusals of the operators of serving in 8 bits that need no GPU, in the Python entry points and at the C ABI, and the
tests' own 64-bit definition of the format against torch's conversions."""

import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from _fp8 import exponent, quantized, to_e4m3
from ccq_amd import Fp8Rows, _lib, fp8_linear, quantize_fp8, rms_norm_fp8

SHAPE, NULL, ALIGN = -1, -2, -3
P = ctypes.c_void_p(0x1000)     # never dereferenced: the checks fail first
ODD = ctypes.c_void_p(0x1001)
BF = torch.bfloat16


def _rows(rows, K, lead=()):
    return Fp8Rows(torch.zeros(*lead, rows, K).to(torch.float8_e4m3fn),
                   torch.ones(*lead, rows, -(-K // 128)).to(torch.float8_e8m0fnu))


def test_definition():
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    every = every[torch.isfinite(every)]
    assert torch.equal(to_e4m3(every), every)
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(4000, generator=gen) * torch.exp(3 * torch.randn(4000, generator=gen))
    x = x.clamp(-448, 448)
    assert torch.equal(to_e4m3(x.double()).float(), x.to(torch.float8_e4m3fn).float())
    ties = (every.sort().values[1:] + every.sort().values[:-1]) / 2
    assert torch.equal(to_e4m3(ties).float(), ties.float().to(torch.float8_e4m3fn).float())
    m = torch.tensor([0.0, 448.0, 448.0001, 896.0, 1.0, 1.75, 1.7500001, 2.0 ** -140], dtype=torch.float64)
    assert exponent(m).tolist() == [-126, 0, 1, 1, -8, -8, -7, -126]
    v, s = quantized(torch.randn(3, 300, generator=gen))
    assert v.shape == (3, 300) and s.shape == (3, 3) and float(v.abs().max()) <= 448


def test_quantize_refusals():
    x = torch.zeros(4, 64, dtype=BF)
    with pytest.raises(RuntimeError, match="GPU"):
        quantize_fp8(x)
    with pytest.raises(TypeError, match="bf16, fp16 or fp32"):
        quantize_fp8(x.double())
    with pytest.raises(TypeError, match="bf16, fp16 or fp32"):
        quantize_fp8(x.to(torch.float8_e4m3fn))
    with pytest.raises(ValueError, match="last dimension"):
        quantize_fp8(x[:, :0])
    with pytest.raises(ValueError, match="last dimension"):
        quantize_fp8(torch.zeros((), dtype=BF))
    with pytest.raises(ValueError, match="last dimension"):
        quantize_fp8(torch.zeros(1, dtype=BF).expand((1 << 22) + 1))
    with pytest.raises(RuntimeError, match="no gradients"):
        quantize_fp8(x.float().requires_grad_())


def test_norm_refusals():
    x, w = torch.zeros(4, 64, dtype=BF), torch.ones(64, dtype=BF)
    with pytest.raises(RuntimeError, match="GPU"):
        rms_norm_fp8(x, w)
    with pytest.raises(TypeError, match="bf16, fp16 or fp32"):
        rms_norm_fp8(x.double(), w)
    with pytest.raises(ValueError, match="last dimension"):
        rms_norm_fp8(torch.zeros(2, 8193, dtype=BF))
    with pytest.raises(ValueError, match="weight"):
        rms_norm_fp8(x, w[:32])
    with pytest.raises(TypeError, match="weight"):
        rms_norm_fp8(x, w.half())
    with pytest.raises(ValueError, match="residual"):
        rms_norm_fp8(x, w, residual=x[:1])
    with pytest.raises(ValueError, match="eps"):
        rms_norm_fp8(x, w, eps=-1.0)
    for call in (lambda: rms_norm_fp8(x.clone().requires_grad_(), w), lambda: rms_norm_fp8(x, w.clone().requires_grad_()),
                 lambda: rms_norm_fp8(x, w, residual=x.clone().requires_grad_())):
        with pytest.raises(RuntimeError, match="no gradients"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):
            call()
    with fwAD.dual_level(), torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
        rms_norm_fp8(fwAD.make_dual(x.float(), torch.ones(4, 64)))


def test_linear_refusals():
    x, w = _rows(4, 200), _rows(32, 200)
    with pytest.raises(RuntimeError, match="GPU"):
        fp8_linear(x, w)
    with pytest.raises(ValueError, match="activation"):
        fp8_linear(x, w, activation="tanh")
    with pytest.raises(TypeError, match="float8_e4m3fn"):
        fp8_linear((x.values.float(), x.scales), w)
    with pytest.raises(TypeError, match="float8_e8m0fnu"):
        fp8_linear(x, (w.values, w.scales.float()))
    with pytest.raises(ValueError, match="x scales"):
        fp8_linear((x.values, x.scales[:, :1]), w)
    with pytest.raises(ValueError, match="weight scales"):
        fp8_linear(x, (w.values, w.scales[:31]))
    with pytest.raises(ValueError, match="weight"):
        fp8_linear(x, _rows(32, 201))
    with pytest.raises(ValueError, match="weight"):
        fp8_linear(x, _rows(32, 200, (2,)))
    with pytest.raises(ValueError, match="at least one"):
        fp8_linear(x, _rows(0, 200))
    with pytest.raises(ValueError, match="last dimension"):
        fp8_linear(_rows(4, 0), w)
    with pytest.raises(ValueError, match="up rows"):
        fp8_linear(x, _rows(31, 200), activation="swiglu")
    with pytest.raises(TypeError, match="dtype"):
        fp8_linear(x, w, dtype=torch.float64)
    with pytest.raises(ValueError, match="bias"):
        fp8_linear(x, w, torch.zeros(31))
    with pytest.raises(TypeError, match="bias"):
        fp8_linear(x, w, torch.zeros(32, dtype=torch.float64))
    with pytest.raises(ValueError, match="residual"):
        fp8_linear(x, w, residual=torch.zeros(1, 32, dtype=BF))
    with pytest.raises(ValueError, match="residual"):
        fp8_linear(x, w, residual=torch.zeros(4, 32))
    with pytest.raises(ValueError, match="residual"):
        fp8_linear(x, w, residual=torch.zeros(4, 32, dtype=BF), quantize=True)
    with pytest.raises(RuntimeError, match="no gradients"):
        fp8_linear(x, w, torch.zeros(32, requires_grad=True))
    with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):
        fp8_linear(x, w, torch.zeros(32, requires_grad=True))


def test_abi_refusals():
    lib = _lib.load()

    def quant(x=P, ldx=200, v=P, ldv=208, s=P, lds=4, rows=4, D=200, dtype=0):
        return lib.ccq_quantize_fp8(x, ldx, v, ldv, s, lds, rows, D, dtype, None)

    assert quant(D=0) == SHAPE and quant(ldx=199) == SHAPE and quant(dtype=3) == SHAPE and quant(rows=-1) == SHAPE
    assert quant(ldv=200) == SHAPE and quant(ldv=192) == SHAPE and quant(lds=2) == SHAPE and quant(lds=6) == SHAPE
    assert quant(D=600, ldx=600, ldv=608) == SHAPE      # five scales a row need 8 bytes
    assert quant(D=(1 << 22) + 1, ldx=1 << 23, ldv=1 << 23) == SHAPE and quant(ldv=(1 << 22) + 16) == SHAPE
    assert quant(x=None) == NULL and quant(v=None) == NULL and quant(s=None) == NULL
    assert quant(x=ODD) == ALIGN and quant(v=ctypes.c_void_p(0x1008)) == ALIGN and quant(s=ctypes.c_void_p(0x1002)) == ALIGN
    assert quant(rows=0) == 0

    def norm(x=P, ldx=200, r=None, ldr=0, w=P, v=P, ldv=208, s=P, lds=4, stream=None, D=200, dtype=0, wdtype=0):
        return lib.ccq_norm_fp8_fwd(x, ldx, r, ldr, w, v, ldv, s, lds, stream, 4, D, dtype, wdtype, 1e-5, None)

    assert norm(D=0) == SHAPE and norm(D=8193, ldx=9000, ldv=9008, lds=80) == SHAPE and norm(ldx=199) == SHAPE
    assert norm(wdtype=1) == SHAPE and norm(r=P, ldr=199, stream=P) == SHAPE and norm(ldv=200) == SHAPE
    assert norm(x=None) == NULL and norm(v=None) == NULL and norm(s=None) == NULL and norm(r=P, ldr=200) == NULL
    assert norm(x=ODD) == ALIGN and norm(v=ODD) == ALIGN and norm(w=ODD) == ALIGN

    def linear(x=P, ldx=208, xs=P, ldxs=4, w=P, ldw=208, ws=P, ldws=4, b=None, bd=0, r=None, ldr=0, y=P, ldy=32, ys=None,
               ldys=0, work=P, M=4, N=32, K=200, act=0, dt=0):
        return lib.ccq_fp8_linear(x, ldx, xs, ldxs, w, ldw, ws, ldws, b, bd, r, ldr, y, ldy, ys, ldys, work, M, N, K, act, dt, None)

    assert linear(M=-1) == SHAPE and linear(N=0) == SHAPE and linear(K=0) == SHAPE and linear(act=6) == SHAPE
    assert linear(dt=3) == SHAPE and linear(bd=3) == SHAPE and linear(r=P, ldr=31) == SHAPE
    assert linear(ldx=200) == SHAPE and linear(ldw=192) == SHAPE and linear(ldxs=3) == SHAPE and linear(ldws=0) == SHAPE
    assert linear(ys=P, ldys=4, ldy=24) == SHAPE and linear(ys=P, ldys=2) == SHAPE
    assert linear(ys=P, ldys=4, r=P, ldr=32) == SHAPE
    assert linear(M=1 << 18, N=1 << 18) == SHAPE    # 2^24 tiles of 64: 2^32 work items, one more than a launch holds
    assert linear(M=1 << 30, N=1 << 22) == SHAPE and linear(N=(1 << 21) + 1, act=5) == SHAPE
    assert linear(x=None) == NULL and linear(xs=None) == NULL and linear(w=None) == NULL and linear(ws=None) == NULL
    assert linear(y=None) == NULL
    assert linear(x=ctypes.c_void_p(0x1008)) == ALIGN and linear(xs=ODD) == ALIGN and linear(ws=ODD) == ALIGN
    assert linear(y=ODD) == ALIGN and linear(b=ODD) == ALIGN and linear(r=ODD, ldr=32) == ALIGN
    # few rows, long: through fp32 (which sizes go that way is the plan's, and asked first)
    K = 16384
    assert lib.ccq_fp8_linear_workspace_bytes(4, 32, K, 0, 0, 1) > 0
    assert linear(ys=P, ldys=4, K=K, ldx=K, ldw=K, ldxs=K // 128, ldws=K // 128, work=None) == NULL
    assert linear(work=ODD) == ALIGN
    assert linear(M=0) == 0
    size = lib.ccq_fp8_linear_workspace_bytes
    assert size(4, 32, K, 0, 0, 1) == 4 * 32 * 4 and size(4, 32, K, 0, 0, 0) == 0 and size(0, 32, K, 0, 0, 1) == 0
    assert size(32768, 4096, 4096, 0, 0, 1) == 0


def test_plan_refusals():
    lib = _lib.load()
    a, b, c = (ctypes.byref(ctypes.c_int()) for _ in range(3))
    for size in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (1 << 31, 1, 1)):
        assert lib.ccq_fp8_linear_plan(*size, 0, 0, 0, a, b, c) == -1
    assert lib.ccq_fp8_linear_plan(1, 1, 1, 9, 0, 0, a, b, c) == -1
    assert lib.ccq_fp8_linear_plan(1, 1, 1, 0, 9, 0, a, b, c) == -1
    assert lib.ccq_fp8_linear_plan(1, 1, 1, 0, 0, 0, a, b, None) == -2
    assert lib.ccq_fp8_linear_plan(1, 1, 1, 0, 9, 1, a, b, c) == 0


def test_plan_and_workspace_agree():
    """An output goes through the workspace where the plan says so, and only one in 8 bits does."""
    lib = _lib.load()
    seen = set()
    for M in (1, 5, 16, 64, 300, 1000, 1100, 5000, 70000):
        for N in (1, 129, 700, 4096, 40000):
            for K in (1, 130, 1000, 8192):
                for act in (0, 3, 5):
                    for dtype, into8 in ((0, 0), (2, 0), (0, 1)):
                        a, b, c = (ctypes.c_int() for _ in range(3))
                        assert lib.ccq_fp8_linear_plan(M, N, K, act, dtype, into8, *map(ctypes.byref, (a, b, c))) == 0
                        room = lib.ccq_fp8_linear_workspace_bytes(M, N, K, act, dtype, into8)
                        assert room == (4 * M * N if c.value else 0) and (into8 or not c.value)
                        assert a.value in (0, 64, 128, 256) and (b.value == 1 or a.value == 0 and b.value in (2, 4, 8))
                        assert a.value or M <= 1024
                        seen.add((a.value, dtype, into8, c.value))
    assert {s[0] for s in seen} == {0, 64, 128, 256} and {s[3] for s in seen} == {0, 1}


def test_abi_stride_of_16_bit_outputs():
    """y in 16 or 32 bits has a row stride as the other rows have: 0 (contiguous) or N and more."""
    lib = _lib.load()

    def linear(ldy, M=4, dt=0):
        return lib.ccq_fp8_linear(P, 208, P, 4, P, 208, P, 4, None, 0, None, 0, P, ldy, None, 0, P, M, 32, 200, 0, dt, None)

    for dt in (0, 1, 2):
        assert linear(31, dt=dt) == SHAPE and linear(-32, dt=dt) == SHAPE and linear(1, dt=dt) == SHAPE
        assert linear(0, M=0, dt=dt) == 0 and linear(32, M=0, dt=dt) == 0 and linear(40, M=0, dt=dt) == 0


def test_plan_offers_what_is_compiled():
    """Tiles of 256 write 16 and 8 bits, those of 64 16 and 32; a gated output in 8 bits needs 128 columns, so tiles of 256 or a
    wave's sixteen."""
    lib = _lib.load()
    sizes = [int(1.7 ** i) + i % 3 for i in range(2, 24)]
    for M in sizes:
        for N in sizes:
            for K in sizes[::3]:
                for act in (0, 1, 5):
                    for dtype, into8 in ((0, 0), (2, 0), (0, 1)):
                        side, parts, through = (ctypes.c_int() for _ in range(3))
                        assert lib.ccq_fp8_linear_plan(M, N, K, act, dtype, into8, *map(ctypes.byref, (side, parts, through))) == 0
                        side, parts, through = side.value, parts.value, through.value
                        if into8 and not through:
                            assert side in ((0, 256) if act == 5 else (0, 128, 256)) and parts == 1
                        elif into8:
                            assert side in (0, 64, 128)
                        elif dtype == 2:
                            assert side in (0, 64)
