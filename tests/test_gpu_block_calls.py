"""Calls of the operators around the mixers beside the ordinary ones: forward-mode derivatives, workspaces, buffers."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD

pytestmark = pytest.mark.gpu

BF, HF, FL = torch.bfloat16, torch.float16, torch.float32


def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda")


@pytest.mark.parametrize("name", ["layer_norm", "rms_norm", "fused_linear", "logprobs", "entropy"])
def test_forward_mode_through_a_gradient_is_refused(name):
    """A gradient that arrives with a tangent raises; its value alone, and an input's value alone, are taken as ever."""
    from ccq_amd import fused_linear, layer_norm, rms_norm, token_logprobs
    dev = _cuda()
    gen = torch.Generator(dev).manual_seed(3)
    x = torch.randn(6, 64, device=dev, generator=gen).to(BF).requires_grad_()
    w, v = torch.randn(64, 64, device=dev, generator=gen).to(BF), torch.ones(64, device=dev)
    ids = torch.arange(6, device=dev)
    call = {"layer_norm": lambda t: layer_norm(t, v, v), "rms_norm": lambda t: rms_norm(t, v),
            "fused_linear": lambda t: fused_linear(t, w, activation="silu"),
            "logprobs": lambda t: token_logprobs(t, ids).logprobs, "entropy": lambda t: token_logprobs(t, ids).entropy}[name]
    y = call(x)
    dy = torch.randn(y.shape, device=dev, generator=gen).to(y.dtype)
    want, = torch.autograd.grad(y, x, dy, retain_graph=True)
    with fwAD.dual_level():
        dual = fwAD.make_dual(dy, torch.ones_like(dy))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(y, x, dual, retain_graph=True)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(fwAD.make_dual(x.detach(), torch.ones_like(x)))
        got, = torch.autograd.grad(y, x, fwAD.unpack_dual(dual).primal, retain_graph=True)
        assert torch.equal(got, want) and torch.equal(call(x.detach()), y)
