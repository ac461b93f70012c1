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


def kept_z(x, w, act, bias=None):
    """What a training forward keeps of x W^T + b (b fp32) for the activation's backward: 16 bits, then 8, of every value."""
    from ccq_amd import _lib
    lib = _lib.load()
    M, K, outs = x.shape[0], x.shape[1], w.shape[0]
    N, ld = outs // 2 if act == 5 else outs, (outs + 7) // 8 * 8
    y = torch.empty(M, N, device=x.device, dtype=x.dtype)
    z = torch.zeros(3 * M * ld, device=x.device, dtype=torch.uint8)
    ws = torch.empty(max(16, lib.ccq_linear_workspace_bytes(M, N, K, act)), device=x.device, dtype=torch.uint8)
    status = lib.ccq_linear_fwd(x.data_ptr(), K, w.data_ptr(), K, None if bias is None else bias.data_ptr(), 2, None, 0,
                                y.data_ptr(), z.data_ptr(), ws.data_ptr(), M, N, K, act, 0,
                                torch.cuda.current_stream().cuda_stream)
    assert status == 0, lib.ccq_last_error()
    z = z.cpu()
    hi = z[:2 * M * ld].view(torch.int16).view(M, ld)[:, :outs].int()
    lo = z[2 * M * ld:].view(M, ld)[:, :outs].int()
    return (hi << 16 | lo << 8).view(torch.float32)


@pytest.mark.parametrize("act", [2, 5], ids=["silu", "swiglu"])
@pytest.mark.parametrize("M,N,K", [(40, 70, 8), (700, 301, 64), (3000, 1500, 128), (6, 44, 4200)], ids=str)
def test_kept_values_round_to_nearest(M, N, K, act):
    """Whole numbers of 24 bits: at most half a step of 16 bits, and the 4 units of 2^-24 that the products may err by
    (4 / 256 of a step).  (6 x 44 over 4200 adds parts of the contraction.)"""
    print("test_kept_values_round_to_nearest", M, N, K, act, flush=True)
    dev = _cuda()
    gen = torch.Generator().manual_seed(M + K)
    outs = 2 * N if act == 5 else N
    x = torch.zeros(M, K)
    x[:, 0], x[:, 1], x[:, K - 1] = 65536, 256, 1
    x *= torch.randint(0, 2, (M, 1), generator=gen) * 2 - 1
    w = torch.zeros(outs, K)
    w[:, [0, 1, K - 1]] = torch.randint(0, 256, (outs, 3), generator=gen).float()
    z = x.double() @ w.double().T
    kept = kept_z(x.to(dev, BF), w.to(dev, BF), act).double()
    step = torch.exp2(torch.floor(torch.log2(z.abs().clamp_min(1))) - 15)
    worst = ((kept - z).abs() / step).max().item()
    assert worst <= 0.5 + 4 / 256, worst


def test_kept_values_at_the_ends():
    """The largest finite value stays finite, infinities and NaN stay, zeros keep their sign."""
    dev = _cuda()
    x = torch.zeros(8, 8, device=dev, dtype=BF)
    x[:, :3] = torch.tensor([torch.finfo(BF).max, 255 * 2.0 ** 112, 255 * 2.0 ** 104], dtype=BF)
    x[1] = -x[1]
    x[2, 1:] = 0
    x[3] = float("inf")
    x[4] = -float("inf")
    x[5, 0] = float("nan")
    x[6] = 0
    x[7] = 2.0 ** -120
    w = torch.ones(16, 8, device=dev, dtype=BF)
    kept = kept_z(x, w, 2)
    big = torch.finfo(FL).max
    assert torch.isfinite(kept[:3]).all() and torch.isfinite(kept[6:]).all()
    assert ((kept[0] - big).abs() <= big * 2.0 ** -15).all() and ((kept[1] + big).abs() <= big * 2.0 ** -15).all()
    assert (kept[2] == torch.finfo(BF).max).all()
    assert (kept[3] == float("inf")).all() and (kept[4] == -float("inf")).all() and kept[5].isnan().all()
    assert (kept[6] == 0).all() and (kept[7] == 2.0 ** -117).all()
    # NaN of any payload: of the lowest bit alone, of all of them, of either sign
    bits = torch.tensor([0x7f800001, 0x7fffffff, 0x800001 - 2 ** 31 + 0x7f000000, -1] * 4, dtype=torch.int32)
    assert bits.view(FL).isnan().all()
    assert kept_z(x[6:], w, 2, bits.to(dev).view(FL)).isnan().all()


@pytest.mark.parametrize("bias", [False, True], ids=["plain", "bias"])
def test_linear_backward_memory_of_a_head(bias):
    """A head's backward reads the logits' gradient where it lies: beside the gradients it allocates the products' and
    the bias's partial sums, nothing of the logits' size."""
    from ccq_amd import _lib, fused_linear
    dev, lib = _cuda(), _lib.load()
    M, N, K = 4096, 32000, 256
    gen = torch.Generator(dev).manual_seed(4)
    x = torch.randint(-2, 3, (M, K), generator=gen, device=dev).to(BF).requires_grad_()
    w = torch.randint(-2, 3, (N, K), generator=gen, device=dev).to(BF).requires_grad_()
    leaves = [x, w] + ([torch.zeros(N, device=dev, requires_grad=True)] if bias else [])
    y = fused_linear(*leaves)
    dy = torch.randint(-2, 3, (M, N), generator=gen, device=dev).to(BF)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    grads = torch.autograd.grad(y, leaves, dy)
    peak = torch.cuda.max_memory_allocated() - before
    most = lib.ccq_linear_bwd_call_workspace_bytes(M, N, K, 0, dy.data_ptr(), N, 1, 1, int(bias))
    assert peak <= sum(2 * g.numel() for g in grads[:2]) + 4 * N + most + (8 << 20), peak    # (blocks of whole MiB)
    assert bias or most < M * N
    assert torch.equal(grads[0], (dy.float() @ w.detach().float()).to(BF))
    assert torch.equal(grads[1], (dy.float().T @ x.detach().float()).to(BF))
    if bias:
        assert torch.equal(grads[2], dy.float().sum(0))


@pytest.mark.parametrize("act", [None, "silu", "swiglu"])
@pytest.mark.parametrize("wanted", range(1, 8))
def test_linear_gradients_one_by_one(act, wanted):
    """Any set of the gradients of x, weight and bias: each call's own workspace, the same bits as of all together; from
    rows of dy that are read in place, padded ones and ones inside wider rows."""
    from ccq_amd import fused_linear
    dev = _cuda()
    gen = torch.Generator(dev).manual_seed(5)
    for M, N, K, pad in ((300, 136, 200, 0), (300, 136, 200, 8), (300, 131, 72, 0), (70, 44, 4200, 0), (2100, 64, 64, 1)):
        outs = 2 * N if act == "swiglu" else N
        x, w, b = (torch.randn(*s, generator=gen, device=dev).to(BF) for s in ((M, K), (outs, K), (outs,)))
        dy = torch.randn(M, N + pad, generator=gen, device=dev).to(BF)[:, :N]

        def grads(which):
            leaves = [t.detach().requires_grad_(bool(which >> i & 1)) for i, t in enumerate((x, w / K ** 0.5, b))]
            return torch.autograd.grad(fused_linear(*leaves, activation=act), [t for t in leaves if t.requires_grad], dy)

        want = [g for i, g in enumerate(grads(7)) if wanted >> i & 1]
        assert all(torch.equal(s, t) for s, t in zip(grads(wanted), want))


def test_more_than_2_31_elements():
    """Rows whose offsets pass 32 bits, forward and backward: the last rows as in a call of them alone (600 rows and more
    take the same workgroups), whole numbers for the linear map."""
    from ccq_amd import fused_linear, rms_norm, token_logprobs
    dev = _cuda()
    gen = torch.Generator(dev).manual_seed(6)
    tail = slice(-700, None)

    def norm(x, r, dy):
        x = x.detach().requires_grad_()
        y, s = rms_norm(x, None, residual=r)
        return [y, s, torch.autograd.grad(y, x, dy)[0]]

    def score(x, ids):
        x = x.detach().requires_grad_()
        got = token_logprobs(x, ids, 3)
        return [*got, torch.autograd.grad(got.logprobs.sum(), x)[0]]

    rows = 2 ** 31 // 8192 + 1000
    x, dy = (torch.empty(rows, 8192, device=dev, dtype=BF).normal_(generator=gen) for _ in range(2))
    print("norm", flush=True)
    for a, b in zip(norm(x, dy, dy), norm(x[tail], dy[tail], dy[tail])):
        assert torch.equal(a[tail], b)
    del x, dy, a, b
    rows = 2 ** 31 // 32000 + 1000
    x = torch.empty(rows, 32000, device=dev, dtype=BF).normal_(generator=gen)
    ids = torch.randint(0, 32000, (rows,), generator=gen, device=dev)
    print("logprobs", flush=True)
    for a, b in zip(score(x, ids), score(x[tail], ids[tail])):
        assert torch.equal(a[tail], b)
    del x, ids, a, b
    M, N, K = 2 ** 31 // 4096 + 1000, 4096, 64
    x, w, dy = (torch.randint(-2, 3, s, generator=gen, device=dev, dtype=torch.int8).to(BF) for s in ((M, K), (N, K), (M, N)))
    x.requires_grad_(), w.requires_grad_()
    print("linear", flush=True)
    y = fused_linear(x, w, activation="relu")
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    z = x[tail].detach().float() @ w.detach().float().T
    dz = dy[tail].float() * (z > 0)
    assert torch.equal(y[tail], z.relu().to(BF)) and torch.equal(dx[tail], (dz @ w.detach().float()).to(BF))
    want = torch.zeros(N, K, device=dev)
    for part in range(0, M, 65536):     # (sums of whole numbers below 2^24)
        p, q = x[part:part + 65536].detach().float(), dy[part:part + 65536].float()
        want += (q * (p @ w.detach().float().T > 0)).T @ p
    assert torch.equal(dw, want.to(BF))
