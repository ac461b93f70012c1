"""Calls of the operators around the mixers that are refused on any device: derivatives that the kernels do not have,
sizes that they cannot count."""

import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from ccq_amd import fused_linear, layer_norm, rms_norm, token_logprobs

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
    from ccq_amd import _lib
    lib = _lib.load()
    a, b = ctypes.c_int(), ctypes.c_int()
    for size in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (1 << 31, 1, 1)):
        assert lib.ccq_linear_plan(*size, ctypes.byref(a), ctypes.byref(b)) == -1
    assert lib.ccq_linear_plan(1, 1, 1, None, ctypes.byref(b)) == -2
