"""The products of ``ccq_amd.fused_linear`` as large training calls run them: tiles of 256 and 128 whose tile rows begin
their contraction at different steps and come round to the first ones, and contractions in parts of such tiles, each
with odd ends.  Which tiles and parts a size takes is asked of the library and asserted, so that a change of the rule
names the cases that it takes out.

Whole numbers: every product and sum is exact in fp32, in the library's products that they are compared with too, so the
outputs have to be equal bit for bit.  Swiglu on real numbers: the bounds of ``test_gpu_linear``, u = eps / 2 of the type.
"""

import ctypes
import math

import pytest
import torch

from test_gpu_linear import BF, D64, HF, U32, _cuda, formula, guarded, run

pytestmark = pytest.mark.gpu


def plan(M, N, K):
    """Side of the tiles, parts of the contraction and steps of 64 in each part."""
    from ccq_amd import _lib
    lib = _lib.load()
    side, parts = ctypes.c_int(), ctypes.c_int()
    assert lib.ccq_linear_plan(M, N, K, ctypes.byref(side), ctypes.byref(parts)) == 0
    return side.value, parts.value, -(-(-(-K // 64)) // parts.value)


#        M, N, K               forward        dx             dW
CASES = [((9001, 1100, 2100), (256, 1, 33), (128, 1, 18), (128, 3, 47)),     # forward: 32 whole steps and a tail, turned
         ((9001, 1100, 2176), (256, 1, 34), (128, 1, 18), (128, 3, 47)),     # no tail
         ((4097, 4099, 2123), (128, 1, 34), (256, 1, 65), (256, 1, 65)),     # dx, dW turned: ends of 3 and of 1
         ((12001, 2900, 1030), (128, 1, 17), (256, 1, 46), (256, 4, 47)),    # dW of 256 in turned parts, the last shorter
         ((16400, 2050, 520), (128, 1, 9), (256, 1, 33), (128, 6, 43)),      # dx: 32 whole steps and a tail of 2
         ((20000, 1030, 1500), (128, 1, 24), (256, 1, 17), (256, 8, 40)),    # dW: 8 turned parts
         ((1030, 1020, 16390), (128, 7, 37), (128, 1, 16), (128, 1, 17))]    # forward in parts of 128


@pytest.mark.parametrize("dtype", [BF, HF], ids=str)
@pytest.mark.parametrize("size,fwd,dx_,dw_", CASES, ids=lambda c: "x".join(map(str, c)))
def test_large_products_of_whole_numbers(size, fwd, dx_, dw_, dtype):
    print("test_large_products_of_whole_numbers", size, dtype, flush=True)
    M, N, K = size
    assert (plan(M, N, K), plan(M, K, N), plan(N, K, M)) == (fwd, dx_, dw_)
    dev = _cuda()
    gen = torch.Generator(dev).manual_seed(M + N + K)

    def whole(*shape):
        return torch.randint(-2, 3, shape, generator=gen, device=dev).float()

    x, w, r, dy, b = whole(M, K), whole(N, K), whole(M, N), whole(M, N), whole(N)
    xg, wg, rg, dg = (guarded(t, dtype, dev) for t in (x, w, r, dy))
    got, (dx, dw, db, dr) = run(xg, wg, b.to(dtype), None, rg, dg)
    assert torch.equal(got, (x @ w.T + b + r).to(dtype)), "y"
    assert torch.equal(dx, (dy @ w).to(dtype)), "dx"
    assert torch.equal(dw, (dy.T @ x).to(dtype)), "dw"
    assert torch.equal(db, dy.sum(0).to(dtype)) and torch.equal(dr, dy.to(dtype))
    # an activation whose slopes are 0 and 1
    got, (dx, dw, _, _) = run(xg, wg, None, "relu", None, dg)
    z = x @ w.T
    dz = dy * (z > 0)
    assert torch.equal(got, z.relu().to(dtype)) and torch.equal(dx, (dz @ w).to(dtype)) and torch.equal(dw, (dz.T @ x).to(dtype))


@pytest.mark.parametrize("M,N,K,side", [(4200, 1025, 2120, 256), (1030, 510, 16390, 128)], ids=str)
def test_large_swiglu(M, N, K, side):
    """Gates and ups of tiles that begin at different steps, and of joined parts."""
    print("test_large_swiglu", M, N, K, flush=True)
    assert plan(M, 2 * N, K)[0] == side
    dev = _cuda()
    gen = torch.Generator(dev).manual_seed(M)
    x, w = (torch.randn(*s, generator=gen, device=dev) for s in ((M, K), (2 * N, K)))
    x, w, dy = x.to(BF), (w / math.sqrt(K)).to(BF), torch.randn(M, N, generator=gen, device=dev).to(BF)
    y, z, _, grads = formula(x, w, None, "swiglu", None, dy)
    got, have = run(x, w, None, "swiglu", None, dy)
    u = torch.finfo(BF).eps / 2
    e = U32 * ((K / 16 + 16) * (x.to(D64).abs() @ w.to(D64).abs().T) + 16 * (z.abs() + 1))
    gate, up = z.chunk(2, -1)
    e = 1.2 * 1.2 * (e[:, :N] * up.abs() + e[:, N:] * gate.abs())
    assert ((got.double() - y).abs() <= u * y.abs() * (1 + u) + e + torch.finfo(BF).tiny).all()
    for name, a, want in zip(("dx", "dw"), have, grads):
        assert ((a.double() - want).norm() / want.norm()).item() <= 1.5 * u, name
