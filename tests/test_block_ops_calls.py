"""Calls of the operators around the mixers that are refused on any device: derivatives that the kernels do not have,
sizes that they cannot count."""

import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from ccq_amd import _lib, fused_linear, layer_norm, rms_norm, token_logprobs

BF = torch.bfloat16


def _calls():
    """Every operator with one of its inputs given, the others fixed."""
    x, w, v, ids = torch.ones(4, 64), torch.ones(64, 64, dtype=BF), torch.ones(64), torch.zeros(4, dtype=torch.int64)
    return {
        "layer_norm x": (x, lambda t: layer_norm(t, v, v)), "layer_norm weight": (v, lambda t: layer_norm(x, t, v)),
        "layer_norm bias": (v, lambda t: layer_norm(x, v, t)),
        "layer_norm residual": (x, lambda t: layer_norm(x, v, v, residual=t)),
        "rms_norm x": (x, lambda t: rms_norm(t, v)), "rms_norm weight": (v, lambda t: rms_norm(x, t)),
        "fused_linear x": (x.to(BF), lambda t: fused_linear(t, w)), "fused_linear weight": (w, lambda t: fused_linear(x.to(BF), t)),
        "fused_linear bias": (v, lambda t: fused_linear(x.to(BF), w, t)),
        "fused_linear residual": (x.to(BF), lambda t: fused_linear(x.to(BF), w, None, "silu", t)),
        "token_logprobs logits": (x, lambda t: token_logprobs(t, ids)),
    }


@pytest.mark.parametrize("name", list(_calls()))
@pytest.mark.parametrize("leaf", [False, True], ids=["plain", "leaf"])
def test_forward_mode_is_refused(name, leaf):
    """An input with a tangent raises: outputs without one would be a derivative of zero."""
    t, call = _calls()[name]
    t = t.clone().requires_grad_(leaf)
    with fwAD.dual_level():
        dual = fwAD.make_dual(t, torch.ones_like(t))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(dual)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            call(dual)
        with fwAD._set_fwd_grad_enabled(False), pytest.raises(RuntimeError, match="GPU only"):
            call(dual)
        with pytest.raises(RuntimeError, match="GPU only"):     # its value alone
            call(fwAD.unpack_dual(dual).primal)


@pytest.mark.parametrize("V", [(1 << 30) + 1, (1 << 32) + 8, 1 << 40])
def test_vocabularies_that_a_row_cannot_count_are_refused(V):
    """Above 2^30 tokens, which the kernels' columns count to; a size that 32 bits would cut to a small one among them."""
    x = torch.zeros(1, 1, dtype=BF).expand(2, V)
    with pytest.raises(ValueError, match="last dimension"):
        token_logprobs(x, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="GPU only"):
        token_logprobs(x[:, :1 << 30], torch.zeros(2, dtype=torch.int64))


def test_linear_plan_refusals():
    lib = _lib.load()
    a, b = ctypes.c_int(), ctypes.c_int()
    for size in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (1 << 31, 1, 1)):
        assert lib.ccq_linear_plan(*size, ctypes.byref(a), ctypes.byref(b)) == -1
    assert lib.ccq_linear_plan(1, 1, 1, None, ctypes.byref(b)) == -2


def test_linear_backward_workspace_of_a_call():
    """dz has no place where dy is read itself, the bias's partial sums none without its gradient."""
    lib = _lib.load()

    def need(M, N, K, act=0, dy=0x1000, ldy=None, dx=1, dw=1, db=0):
        return lib.ccq_linear_bwd_call_workspace_bytes(M, N, K, act, ctypes.c_void_p(dy), N if ldy is None else ldy, dx, dw, db)

    parts = max(lib.ccq_linear_workspace_bytes(16384, 1024, 32000, 0), lib.ccq_linear_workspace_bytes(32000, 1024, 16384, 0))
    dz = 16384 * 32000 * 2
    assert need(16384, 32000, 1024) <= parts + 256
    for case in (dict(dy=0x1008), dict(ldy=32004), dict(ldy=(1 << 22) + 8), dict(act=2)):
        assert dz <= need(16384, 32000, 1024, **case) <= dz + parts + 512, case
    assert need(16384, 32000, 1024, act=2, dx=0, dw=0, db=1) < dz    # (db alone: no product reads dz)
    assert need(16384, 31999, 1024) >= dz - 16384 * 2
    assert 0 < need(64, 64, 64, db=1) <= lib.ccq_linear_bwd_workspace_bytes(64, 64, 64, 0)
    assert need(64, 64, 64) == 0 and need(0, 64, 64, act=2) == 0 and need(-1, 64, 64) == 0
    for act in range(6):
        for M, N, K in ((1, 1, 1), (16384, 2816, 1024), (37, 4200, 24), (128, 128, 262144)):
            assert need(M, N, K, act, dy=0x1002, db=1) <= lib.ccq_linear_bwd_workspace_bytes(M, N, K, act)
