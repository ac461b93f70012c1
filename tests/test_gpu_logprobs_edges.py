"""Rows at the edges of ``ccq_amd.token_logprobs``: infinities and NaN where the alternatives' list begins, rows of
nothing but -inf with each of the two gradients alone.  Orders and NaN are exact; values beside them keep their bits."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, HF, FL = torch.bfloat16, torch.float16, torch.float32


def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda")


@pytest.mark.parametrize("dtype", [BF, HF, FL], ids=str)
@pytest.mark.parametrize("rows", [12, 600], ids=str)      # both workgroup sizes
@pytest.mark.parametrize("V", [9, 1003, 40000], ids=str)
def test_top_with_positive_infinities(V, rows, dtype):
    """+inf from the first piece to the last one, alone and in every place: such rows are NaN, their alternatives in the
    logits' order, and the other rows as they are without them."""
    print("test_top_with_positive_infinities", V, rows, dtype, flush=True)
    from ccq_amd import token_logprobs
    dev = _cuda()
    gen = torch.Generator().manual_seed(V + rows)
    x = torch.randn(rows, V, generator=gen).to(dtype)
    ids = torch.randint(0, V, (rows,), generator=gen).to(dev)
    k = min(V, 7)
    good = token_logprobs(x.to(dev), ids, k)
    x[0, 0] = x[1, 8] = x[2, V - 1] = x[3, V // 2] = math.inf
    x[4] = math.inf
    x[5, ::2] = math.inf
    x[6, ::2], x[6, 1::2] = math.inf, -math.inf
    got = token_logprobs(x.to(dev), ids, k)
    order = torch.sort(x.double(), dim=-1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(got.top_ids.cpu(), order)
    assert got.logprobs[:7].isnan().all() and got.entropy[:7].isnan().all() and got.top_logprobs[:7].isnan().all()
    for a, b in zip(got, good):
        assert torch.equal(a[7:], b[7:])


@pytest.mark.parametrize("dtype", [BF, HF, FL], ids=str)
@pytest.mark.parametrize("rows", [6, 600], ids=str)
@pytest.mark.parametrize("V", [1, 2, 64, 1003], ids=str)
def test_top_with_nan_logits(V, rows, dtype):
    """A NaN stands before every number, the lowest index first: at token 0, at the last one, all over the row, beside
    +inf; with as many alternatives as tokens each of them once."""
    print("test_top_with_nan_logits", V, rows, dtype, flush=True)
    from ccq_amd import token_logprobs
    dev = _cuda()
    gen = torch.Generator().manual_seed(V + rows)
    x = torch.randn(rows, V, generator=gen).to(dtype)
    x[0, 0] = x[1, V - 1] = math.nan
    x[2] = math.nan
    x[3, 0], x[3, V // 2] = math.inf, math.nan
    x[4, 0], x[4, V // 2] = math.nan, math.inf
    ids = torch.randint(0, V, (rows,), generator=gen).to(dev)
    key = torch.where(x.isnan(), math.inf, x.double()) + 0.0
    # NaN first: a stable sort by the number, then one by being a NaN
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    nan = x.isnan().gather(1, order).int()
    order = order.gather(1, torch.sort(nan, dim=-1, descending=True, stable=True).indices)
    for k in sorted({1, min(V, 5), min(V, 64)}):
        got = token_logprobs(x.to(dev), ids, k)
        assert torch.equal(got.top_ids.cpu(), order[:, :k]), k
        assert got.top_logprobs[:5].isnan().all() and got.logprobs[:5].isnan().all()
        assert torch.isfinite(got.top_logprobs[5:]).all()


@pytest.mark.parametrize("dtype", [BF, HF, FL], ids=str)
@pytest.mark.parametrize("rows", [9, 600], ids=str)
def test_gradient_of_rows_without_a_logit(rows, dtype):
    """Nothing but -inf, a NaN, +inf, a token outside: NaN gradients whichever of the two results they come from, the
    entropy's alone only where the entropy is NaN; the other rows as they are without them."""
    print("test_gradient_of_rows_without_a_logit", rows, dtype, flush=True)
    from ccq_amd import token_logprobs
    dev = _cuda()
    gen = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, 777, generator=gen).to(dtype)
    ids = torch.randint(0, 777, (rows,), generator=gen)
    good_ids = ids.clone()
    bad = x.clone()
    bad[0] = -math.inf
    bad[1] = -math.inf
    bad[2, 5], bad[3, 700] = math.nan, math.inf
    bad[4] = -math.inf
    ids[0], ids[4], ids[5] = 0, -100, 777
    one, some, none = torch.ones(rows), torch.randn(rows, generator=gen), torch.zeros(rows)

    def grad(x, ids, dlogp, dent):
        leaf = x.to(dev).requires_grad_()
        got = token_logprobs(leaf, ids.to(dev))
        outs = [(o, g.to(dev)) for o, g in ((got.logprobs, dlogp), (got.entropy, dent)) if g is not None]
        return torch.autograd.grad([o for o, _ in outs], leaf, [g for _, g in outs])[0]

    for dlogp, dent in ((one, None), (one, none), (none, None), (None, some), (some, some), (None, none)):
        dx, want = grad(bad, ids, dlogp, dent), grad(x, good_ids, dlogp, dent)
        assert dx[:4].isnan().all(), (dlogp is None, dent is None)
        assert dx[5].isnan().all()
        assert (dx[4] == 0).all()
        assert torch.equal(dx[6:], want[6:])
