"""Refusals of the operators around the mixers that need no GPU: arguments are checked before anything is launched,
in the Python entry points and at the C ABI."""

import ctypes

import pytest
import torch

from ccq_amd import _lib, layer_norm, rms_norm, token_logprobs

SHAPE, NULL, ALIGN = -1, -2, -3
P = ctypes.c_void_p(0x1000)     # never dereferenced: the checks fail first
ODD = ctypes.c_void_p(0x1001)


@pytest.mark.parametrize("norm", [layer_norm, rms_norm])
def test_norm_refusals(norm):
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    w = torch.ones(64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="GPU"):
        norm(x, w)
    with pytest.raises(TypeError, match="bf16, fp16 or fp32"):
        norm(x.double(), w)
    with pytest.raises(ValueError, match="last dimension"):
        norm(torch.zeros(2, 8193, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="last dimension"):
        norm(torch.zeros(2, 0, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="last dimension"):
        norm(torch.zeros((), dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="weight"):
        norm(x, w[:32])
    with pytest.raises(TypeError, match="weight"):
        norm(x, w.half())
    with pytest.raises(ValueError, match="residual"):
        norm(x, w, residual=x[:1])
    with pytest.raises(ValueError, match="residual"):
        norm(x, w, residual=x.float())
    with pytest.raises(ValueError, match="eps"):
        norm(x, w, eps=-1.0)
    with pytest.raises(ValueError, match="eps"):
        norm(x, w, eps=float("nan"))


def test_layer_norm_bias_type():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="one type"):
        layer_norm(x, torch.ones(64), torch.zeros(64, dtype=torch.bfloat16))


def test_norm_abi_refusals():
    lib = _lib.load()

    def fwd(x=P, ldx=64, r=None, ldr=0, w=P, b=None, y=P, s=None, mean=None, rstd=None, D=64, dtype=0, wdtype=0,
            layer=1):
        return lib.ccq_norm_fwd(x, ldx, r, ldr, w, b, y, s, mean, rstd, 4, D, dtype, wdtype, layer, 1e-5, None)

    assert fwd(D=0) == SHAPE and fwd(D=8193, ldx=9000) == SHAPE and fwd(ldx=63) == SHAPE
    assert fwd(dtype=3) == SHAPE and fwd(wdtype=1) == SHAPE and fwd(b=P, layer=0) == SHAPE
    assert fwd(r=P, s=P, ldr=63) == SHAPE
    assert fwd(x=None) == NULL and fwd(y=None) == NULL and fwd(r=P, ldr=64) == NULL and fwd(rstd=P) == NULL
    assert fwd(x=ODD) == ALIGN and fwd(w=ODD) == ALIGN

    def bwd(x=P, ldy=64, mean=P, rstd=P, dy=P, dx=P, dw=P, db=P, ws=P, layer=1):
        return lib.ccq_norm_bwd(x, 64, P, mean, rstd, dy, ldy, None, 0, dx, dw, db, ws, 4, 64, 0, 0, layer, None)

    assert bwd(ldy=10) == SHAPE and bwd(layer=0) == SHAPE
    assert bwd(x=None) == NULL and bwd(mean=None) == NULL and bwd(rstd=None) == NULL and bwd(ws=None) == NULL
    assert bwd(ws=ctypes.c_void_p(0x1008)) == ALIGN and bwd(dx=ODD) == ALIGN
    # partial rows of dw and db: one for each workgroup, at most 512 (1024 where a lane holds one piece of a row)
    assert lib.ccq_norm_bwd_workspace_bytes(100000, 1024, 0) == 2 * 512 * 1024 * 4
    assert lib.ccq_norm_bwd_workspace_bytes(8, 1024, 0) == 2 * 2 * 1024 * 4
    assert lib.ccq_norm_bwd_workspace_bytes(100000, 2048, 0) == 2 * 1024 * 2048 * 4


def test_token_logprobs_refusals():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    ids = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="GPU"):
        token_logprobs(x, ids)
    with pytest.raises(TypeError, match="logits"):
        token_logprobs(x.double(), ids)
    with pytest.raises(TypeError, match="ids"):
        token_logprobs(x, ids.float())
    with pytest.raises(ValueError, match="ids"):
        token_logprobs(x, ids[:3])
    with pytest.raises(ValueError, match="ids"):
        token_logprobs(torch.zeros(4, 0, dtype=torch.bfloat16), ids)
    with pytest.raises(ValueError, match="top_k"):
        token_logprobs(x, ids, top_k=65)
    with pytest.raises(ValueError, match="top_k"):
        token_logprobs(x[:, :8], ids, top_k=9)
    with pytest.raises(ValueError, match="top_k"):
        token_logprobs(x, ids, top_k=-1)


def test_token_logprobs_abi_refusals():
    lib = _lib.load()

    def fwd(x=P, ldx=64, ids=P, logp=P, ent=P, top=P, top_ids=P, V=64, k=4, dtype=0):
        return lib.ccq_token_logprobs_fwd(x, ldx, ids, logp, ent, None, top, top_ids, 4, V, k, -100, dtype, None)

    assert fwd(V=0) == SHAPE and fwd(ldx=63) == SHAPE and fwd(dtype=7) == SHAPE
    assert fwd(k=65, V=100, ldx=100) == SHAPE and fwd(k=5, V=4) == SHAPE and fwd(k=-1) == SHAPE
    assert fwd(x=None) == NULL and fwd(ids=None) == NULL and fwd(logp=None) == NULL and fwd(top=None) == NULL
    assert fwd(x=ODD) == ALIGN

    def bwd(x=P, ids=P, ent=P, stats=P, dx=P, V=64):
        return lib.ccq_token_logprobs_bwd(x, 64, ids, ent, stats, P, P, dx, 4, V, -100, 0, None)

    assert bwd(V=65) == SHAPE and bwd(ent=None) == NULL and bwd(stats=None) == NULL and bwd(dx=None) == NULL
    assert bwd(dx=ODD) == ALIGN


def test_fused_linear_refusals():
    from ccq_amd import fused_linear
    bf = torch.bfloat16
    x, w = torch.zeros(4, 64, dtype=bf), torch.zeros(32, 64, dtype=bf)
    with pytest.raises(RuntimeError, match="GPU"):
        fused_linear(x, w)
    with pytest.raises(TypeError, match="one type"):
        fused_linear(x.float(), w.float())
    with pytest.raises(TypeError, match="one type"):
        fused_linear(x, w.half())
    with pytest.raises(ValueError, match="activation"):
        fused_linear(x, w, activation="tanh")
    with pytest.raises(ValueError, match="weight"):
        fused_linear(x, w[:, :32])
    with pytest.raises(ValueError, match="weight"):
        fused_linear(x, w[0])
    with pytest.raises(ValueError, match="at least 1"):
        fused_linear(x, w[:0])
    with pytest.raises(ValueError, match="at least 1"):
        fused_linear(x[:, :0], w[:, :0])
    with pytest.raises(ValueError, match="up rows"):
        fused_linear(x, w[:31], activation="swiglu")
    with pytest.raises(ValueError, match="bias"):
        fused_linear(x, w, torch.zeros(31, dtype=bf))
    with pytest.raises(TypeError, match="bias"):
        fused_linear(x, w, torch.zeros(32, dtype=torch.float16))
    with pytest.raises(ValueError, match="residual"):
        fused_linear(x, w, residual=torch.zeros(4, 16, dtype=bf))
    with pytest.raises(ValueError, match="residual"):
        fused_linear(x, w, residual=torch.zeros(1, 32, dtype=bf))
    with pytest.raises(ValueError, match="residual"):
        fused_linear(x, w, residual=torch.zeros(4, 32))


def test_linear_abi_refusals():
    lib = _lib.load()

    def fwd(x=P, ldx=64, w=P, ldw=64, b=None, bd=0, r=None, ldr=32, y=P, z=None, ws=P, M=4, N=32, K=64, act=0, dt=0):
        return lib.ccq_linear_fwd(x, ldx, w, ldw, b, bd, r, ldr, y, z, ws, M, N, K, act, dt, None)

    assert fwd(N=0) == SHAPE and fwd(K=0) == SHAPE and fwd(M=-1) == SHAPE and fwd(ldx=60) == SHAPE
    assert fwd(ldw=63) == SHAPE and fwd(ldx=68) == SHAPE and fwd(act=6) == SHAPE and fwd(dt=2) == SHAPE
    assert fwd(bd=1) == SHAPE and fwd(r=P, ldr=31) == SHAPE and fwd(K=65) == SHAPE   # (rows of 65 need 72)
    assert fwd(ldx=(1 << 22) + 8) == SHAPE
    assert fwd(x=None) == NULL and fwd(w=None) == NULL and fwd(y=None) == NULL
    assert fwd(x=ctypes.c_void_p(0x1008)) == ALIGN and fwd(y=ODD) == ALIGN and fwd(z=ODD) == ALIGN

    def bwd(x=P, w=P, z=P, dy=P, ldy=32, dx=P, dw=P, db=None, ws=P, act=2):
        return lib.ccq_linear_bwd(x, 64, w, 64, z, dy, ldy, dx, dw, db, 0, ws, 4, 32, 64, act, 0, None)

    assert bwd(ldy=31) == SHAPE and bwd(ws=None) == NULL and bwd(z=None) == NULL and bwd(dy=None) == NULL
    assert bwd(x=None) == NULL and bwd(w=None) == NULL and bwd(dx=ODD) == ALIGN and bwd(dy=ODD) == ALIGN
    assert bwd(ws=ctypes.c_void_p(0x1008)) == ALIGN
    assert lib.ccq_pad_rows(P, 5, P, 7, 3, 5, None) == SHAPE and lib.ccq_pad_rows(P, 5, P, 8, 3, 6, None) == SHAPE
    assert lib.ccq_pad_rows(P, 5, ODD, 8, 3, 5, None) == ALIGN and lib.ccq_pad_rows(None, 5, P, 8, 3, 5, None) == NULL
    # sizes of nothing: no rows, one output
    assert lib.ccq_linear_workspace_bytes(0, 32, 64, 0) == 0
    assert lib.ccq_linear_bwd_workspace_bytes(0, 32, 64, 0) >= 0 and lib.ccq_linear_bwd_workspace_bytes(1, 1, 1, 5) > 0


def test_linear_abi_sizes_refused():
    """Products of more tiles than a launch holds; the longest and widest that fit pass on to the pointers' checks."""
    lib = _lib.load()

    def fwd(M, N, K):
        k8 = (K + 7) // 8 * 8
        return lib.ccq_linear_fwd(None, k8, P, k8, None, 0, None, 0, P, None, P, M, N, K, 0, 0, None)

    assert fwd(1 << 30, 1 << 22, 8) == SHAPE and fwd(1 << 30, 8, 1 << 22) == SHAPE and fwd((1 << 30) + 1, 8, 8) == SHAPE
    assert fwd(8, (1 << 22) + 1, 8) == SHAPE and fwd(8, 8, (1 << 22) + 1) == SHAPE
    assert fwd(1 << 30, 1, 1) == NULL and fwd(1, 1 << 22, 8) == NULL and fwd(1, 8, 1 << 22) == NULL
