"""GPU parity of the log probabilities of given tokens (``ccq_amd.token_logprobs``) against log softmax in 64 bits.

Tolerances, absolute and element by element, from 32-bit arithmetic in units of 2^-24: a sum over the vocabulary is
at most V / 256 additions in a thread and 16 merges of a few operations each, and an exponential's argument x - m is
off by half a unit of itself, so log Z and the entropy's two sums carry at most n = V / 256 + 64 units of their size
(the exponential's error, |x - m| units, is weighted by e^(x - m) |x - m| <= 0.37).  logp adds the roundings of
x - m and of the difference; gradients are products of p, whose relative error is n units and the roundings of
x - m, log Z and their difference, and round once to the logits' type.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

D64 = torch.float64
BF, HF, FL = torch.bfloat16, torch.float16, torch.float32
U32 = 2.0 ** -24


def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda")


def make(rows, V, dtype, seed, ignored=0.2, scale=3.0):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, V, generator=gen) * scale).to(dtype)
    ids = torch.randint(0, V, (rows,), generator=gen)
    if rows > 2:
        ids[torch.rand(rows, generator=gen) < ignored] = -100
    return x, ids, torch.randn(rows, generator=gen), torch.randn(rows, generator=gen)


def formula(x, ids, dlogp=None, dent=None):
    z = x.to(D64)
    keep = ids != -100
    u = z - z.amax(-1, keepdim=True)     # (apart from the maximum: beside -3e38 even 64 bits lose log Z)
    logz = u.exp().sum(-1).log()
    lp = u - logz[:, None]
    p = lp.exp()
    plp = torch.where(p > 0, p * lp, 0.0)
    ent = -plp.sum(-1)
    at = ids.clamp_min(0)[:, None]
    out = {"logz": logz, "logp": torch.where(keep, lp.gather(1, at)[:, 0], 0.0),
           "ent": torch.where(keep, ent, 0.0), "lp": lp, "keep": keep}
    if dlogp is not None:
        a, b = (torch.where(keep, t.to(D64), 0.0)[:, None] for t in (dlogp, dent))
        dx = -p * a - b * (plp + p * ent[:, None])
        mag = p * a.abs() + b.abs() * (plp.abs() + p * ent[:, None].abs())
        one = torch.zeros_like(dx).scatter_(1, at, a)
        out["dx"], out["mag"], out["one"] = dx + one, mag, one.abs()
    return out


def call(x, ids, k=0, dlogp=None, dent=None, **kw):
    from ccq_amd import token_logprobs
    dev = _cuda()
    xg = (x if x.is_cuda else x.to(dev)).detach()
    if dlogp is None and dent is None:
        return token_logprobs(xg, ids.to(dev), top_k=k, **kw), None
    xg.requires_grad_()
    got = token_logprobs(xg, ids.to(dev), top_k=k, **kw)
    outs = [(o, g.to(dev)) for o, g in ((got.logprobs, dlogp), (got.entropy, dent)) if g is not None]
    return got, torch.autograd.grad([o for o, _ in outs], xg, [g for _, g in outs])[0]


def check_values(got, want, V):
    n = (V / 256 + 64) * U32
    off = (got.logprobs.cpu().double() - want["logp"]).abs()
    assert (off <= n + 4 * U32 * (want["logp"].abs() + want["logz"])).all(), off.max()
    off = (got.entropy.cpu().double() - want["ent"]).abs()
    assert (off <= n * (1 + 2 * want["ent"])).all(), off.max()


def check_top(got, x, want, k):
    """The stable order of the logits, largest first: ties to the lowest index."""
    order = torch.sort(x.to(D64), dim=-1, descending=True, stable=True).indices[:, :k]
    keep = want["keep"][:, None]
    assert torch.equal(got.top_ids.cpu(), torch.where(keep, order, -1))
    top = torch.where(keep, want["lp"].gather(1, order), 0.0)
    have = got.top_logprobs.cpu().double()
    far = top == -math.inf
    assert torch.equal(have == -math.inf, far)
    n = (x.shape[1] / 256 + 64) * U32 + 4 * U32 * (top.abs() + want["logz"][:, None])
    assert ((have - top).abs()[~far] <= n[~far]).all()


def check_grad(dx, want, dtype, V):
    ref = want["dx"]
    fin = torch.finfo(dtype)
    n = (V / 256 + 64) + 4 * (want["logz"][:, None] + want["lp"].abs().clamp_max(1e4))
    bound = fin.eps / 2 * ref.abs() + U32 * (n * want["mag"] + 2 * want["one"]) * (1 + fin.eps) \
        + fin.tiny * fin.eps + 1e-37
    worst = ((dx.cpu().double() - ref).abs() / bound).max().item()
    assert worst <= 1, worst


SIZES = [(1, 1), (3, 2), (5, 7), (4, 64), (9, 65), (33, 1000), (600, 1023), (520, 2500), (16, 32000), (7, 32007),
         (3, 70001), (2, 160000)]


@pytest.mark.parametrize("dtype", [BF, HF, FL], ids=str)
@pytest.mark.parametrize("rows,V", SIZES, ids=str)
def test_logprobs(rows, V, dtype):
    print("test_logprobs", rows, V, dtype, flush=True)
    x, ids, a, b = make(rows, V, dtype, rows + V)
    want = formula(x, ids, a, b)
    k = min(V, 20)
    got, dx = call(x, ids, k, a, b)
    check_values(got, want, V)
    check_top(got, x, want, k)
    check_grad(dx, want, dtype, V)
    plain, _ = call(x, ids, 0)
    assert torch.equal(plain.logprobs, got.logprobs) and torch.equal(plain.entropy, got.entropy)
    assert plain.top_ids is None and plain.top_logprobs is None


@pytest.mark.parametrize("k", [1, 2, 5, 32, 63, 64])
def test_top_many_ties(k):
    """Few distinct values, so that far more logits reach the k-th largest than any list holds, and one row whose
    candidates are exactly the list's length or one more."""
    print("test_top_many_ties", k, flush=True)
    gen = torch.Generator().manual_seed(k)
    V = 5000
    x = torch.randint(-2, 2, (600, V), generator=gen).to(BF)
    x[1] = 0.0
    x[2] = 0.0
    x[2, ::2] = -0.0            # equal to 0
    x[3] = -math.inf
    x[3, 100] = 1.0             # one token left
    for i, n in ((4, 1023), (5, 1024), (6, 1025)):
        x[i] = -1.0
        x[i, torch.randperm(V, generator=gen)[:n]] = 3.0
    x[7] = torch.finfo(BF).min  # a mask of the type's lowest value over the whole row: uniform
    ids = torch.randint(0, V, (600,), generator=gen)
    ids[3] = 100
    want = formula(x, ids)
    for rows in (600, 40):      # both workgroup sizes
        w = {n: t[:rows] for n, t in want.items()}
        got, _ = call(x[:rows], ids[:rows], k)
        check_values(got, w, V)
        check_top(got, x[:rows], w, k)


@pytest.mark.parametrize("dtype", [BF, HF, FL], ids=str)
def test_logprobs_masks(dtype):
    """Masked vocabularies: -inf and the type's lowest value, whole parts of the row, and one token left."""
    x, ids, a, b = make(12, 3001, dtype, 3, ignored=0.0)
    low = torch.finfo(dtype).min
    x[0, 1500:] = -math.inf
    x[1, :2999] = -math.inf
    x[2, ::2] = low
    x[3, 1:] = low
    x[4, 1:] = -math.inf
    x[5] = low
    x[6] += 100.0
    x[7, 5] = 1000.0
    ids[:8] = torch.tensor([3, 3000, 1, 0, 0, 77, 9, 5])
    want = formula(x, ids, a, b)
    got, dx = call(x, ids, 4, a, b)
    check_values(got, want, 3001)
    check_top(got, x, want, 4)
    check_grad(dx, want, dtype, 3001)
    ids[0] = 2000               # a masked token: probability 0
    got, dx = call(x, ids, 0, a, b)
    assert got.logprobs[0].item() == -math.inf and torch.isfinite(dx[1:]).all()


@pytest.mark.parametrize("rows", [10, 700])
def test_logprobs_bad_rows(rows):
    """NaN, +inf, nothing but -inf, tokens outside the vocabulary: NaN in that row alone; skipped rows are not read."""
    x, ids, a, b = make(rows, 500, FL, 4, ignored=0.0)
    want = formula(x, ids, a, b)
    good, gdx = call(x, ids, 3, a, b)
    x[0, 17] = math.nan
    x[1, 400] = math.inf
    x[2] = -math.inf
    ids[3], ids[4], ids[5] = 500, -1, 1 << 40
    x[6] = math.nan
    ids[6] = -100
    got, dx = call(x, ids, 3, a, b)
    assert got.logprobs[:6].isnan().all() and got.entropy[:3].isnan().all()
    assert got.top_logprobs[:3].isnan().all()
    assert got.top_ids[0, 0].item() == 17 and got.top_ids[1, 0].item() == 400 and got.top_ids[2].tolist() == [0, 1, 2]
    assert dx[:6].isnan().all()
    assert got.logprobs[6].item() == 0 and got.entropy[6].item() == 0 and (dx[6] == 0).all()
    assert (got.top_ids[6] == -1).all() and (got.top_logprobs[6] == 0).all()
    assert torch.equal(got.entropy[3:6], good.entropy[3:6])
    for s, t in ((got.logprobs, good.logprobs), (got.entropy, good.entropy), (dx, gdx), (got.top_ids, good.top_ids)):
        assert torch.equal(s[7:], t[7:])
    check_values(good, want, 500)


def test_logprobs_other_ignore_and_id_types_and_shapes():
    from ccq_amd import token_logprobs
    dev = _cuda()
    x, ids, _, _ = make(24, 333, BF, 5)
    want = formula(x, ids)
    flat, _ = call(x, ids, 2)
    ids0 = torch.where(ids == -100, 7, ids)
    got = token_logprobs(x.to(dev).view(2, 3, 4, 333), torch.where(ids0 == 7, -1, ids0).to(dev).int().view(2, 3, 4), 2, -1)
    same = (ids0 != 7).view(2, 3, 4).to(dev)
    assert got.logprobs.shape == (2, 3, 4) and got.top_ids.shape == (2, 3, 4, 2)
    assert torch.equal(got.logprobs[same], flat.logprobs.view(2, 3, 4)[same])
    assert (got.logprobs[~same] == 0).all()
    one = token_logprobs(x[0].to(dev), torch.tensor(5, device=dev))
    assert one.logprobs.shape == () and abs(one.logprobs.item() - want["lp"][0, 5].item()) < 1e-5
    none = token_logprobs(x[:0].to(dev).requires_grad_(), ids[:0].to(dev), 2)
    assert none.logprobs.shape == (0,) and none.top_ids.shape == (0, 2)


@pytest.mark.parametrize("dtype", [BF, FL], ids=str)
def test_logprobs_strided_logits(dtype):
    """Rows inside wider ones, at any element's address; positions taken out of [B, T, V] (the shifted loss)."""
    dev = _cuda()
    x, ids, a, b = make(30, 1003, dtype, 6)
    want = formula(x[:, 1:-1], torch.where(ids == -100, -100, ids % 1001), a, b)
    ids = torch.where(ids == -100, -100, ids % 1001)
    got, dx = call(x.to(dev)[:, 1:-1], ids, 5, a, b)
    check_values(got, want, 1001)
    check_top(got, x[:, 1:-1], want, 5)
    check_grad(dx, want, dtype, 1001)
    y, jds, a, b = make(40, 1001, dtype, 7)
    want = formula(y.view(4, 10, 1001)[:, :-1].reshape(36, 1001), jds[:36], a[:36], b[:36])
    got, dx = call(y.to(dev).view(4, 10, 1001)[:, :-1], jds[:36].view(4, 9), 0, a[:36].view(4, 9), b[:36].view(4, 9))
    assert dx.shape == (4, 9, 1001)
    check_grad(dx.reshape(36, 1001), want, dtype, 1001)


def test_logprobs_single_gradients_and_broadcast():
    x, ids, a, b = make(50, 700, BF, 8)
    zero = torch.zeros(50)
    check_grad(call(x, ids, 0, a, None)[1], formula(x, ids, a, zero), BF, 700)
    check_grad(call(x, ids, 0, None, b)[1], formula(x, ids, zero, b), BF, 700)
    one = torch.ones(()).expand(50)     # the gradient of a sum: stride 0
    check_grad(call(x, ids, 3, one, None)[1], formula(x, ids, torch.ones(50), zero), BF, 700)


def test_logprobs_against_differences():
    """Central differences of the 64-bit formula along random directions (truncation h^2 = 1e-8 of the scale)."""
    x, ids, a, b = make(5, 40, FL, 9, ignored=0.0)
    _, dx = call(x, ids, 0, a, b)
    v = torch.randn(5, 40, generator=torch.Generator().manual_seed(2), dtype=D64)

    def loss(t):
        f = formula(x.to(D64) + t * v, ids)
        return (f["logp"] * a.to(D64)).sum() + (f["ent"] * b.to(D64)).sum()

    want = (loss(1e-4) - loss(-1e-4)) / 2e-4
    have = (dx.cpu().double() * v).sum()
    assert abs(have - want) <= 1e-6 * (dx.cpu().double().abs() * v.abs()).sum() + 1e-6


def test_logprobs_captured_and_other_stream():
    from ccq_amd import token_logprobs
    dev = _cuda()
    sets = [[t.to(dev) for t in make(40, 5003, BF, 30 + i)] for i in range(3)]

    def step(x, ids, a, b):
        leaf = x.detach().requires_grad_()
        got = token_logprobs(leaf, ids, top_k=6)
        return [*got, torch.autograd.grad([got.logprobs, got.entropy], leaf, [a, b])[0]]

    want = [[t.clone() for t in step(*s)] for s in sets]
    static = [t.clone() for t in sets[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(*static)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(s, t) for s, t in zip(other, want[0]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*static)
    for k in (0, 1, 2, 1):
        for s, t in zip(static, sets[k]):
            s.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(s, t) for s, t in zip(out, want[k]))
        step(*sets[0])
        torch.cuda.synchronize()


def test_logprobs_more_rows_than_a_launch_is_wide():
    """2^24 + 3 rows of two logits: workgroups of every row would pass 32 bits of work items in one dimension."""
    from ccq_amd import token_logprobs
    dev = _cuda()
    rows = 2 ** 24 + 3
    x = torch.randn(rows, 2, device=dev, generator=torch.Generator(dev).manual_seed(3)).half().requires_grad_()
    ids = torch.randint(0, 2, (rows,), device=dev, generator=torch.Generator(dev).manual_seed(4))
    got = token_logprobs(x, ids)
    dx = torch.autograd.grad(got.logprobs.sum(), x)[0]
    d = (x.detach()[:, 1].double() - x.detach()[:, 0].double()) * (2 * ids - 1)    # log odds of the given token
    want = -torch.log1p(torch.exp(-d))
    assert ((got.logprobs.double() - want).abs() <= (2 / 256 + 64) * U32 + 4 * U32 * (want.abs() + math.log(2))).all()
    other = torch.sigmoid(-d)
    sign = torch.stack([1.0 - 2 * ids, 2 * ids - 1.0], -1)
    # one rounding to the logits' type (half a step, or half the smallest one), and the relative error of p
    n = torch.finfo(HF).eps / 2 + (2 / 256 + 64 + 16) * U32
    assert ((dx.double() - sign * other[:, None]).abs() <= n * other[:, None] + 2.0 ** -25).all()


@pytest.mark.parametrize("dtype", [BF, HF, FL], ids=str)
@pytest.mark.parametrize("rows", [8, 600], ids=str)      # both workgroup sizes
def test_top_sorted_rows(rows, dtype):
    """Rows in rising order, whose every later piece reaches the bound of the first ones, and in falling order; runs of
    equal logits, and the likeliest tokens all in one piece."""
    V = 40000
    x = torch.zeros(rows, V)
    rise = torch.linspace(-20.0, 8.0, V)
    x[0::8], x[1::8] = rise, rise.flip(0)
    x[2::8] = rise.round()
    x[3::8] = rise.round().flip(0)
    x[4::8, 39990:] = torch.arange(10.0)
    x[5::8, 20000:20064] = 3.0
    x[6::8] = -rise.abs()
    x[7::8, :2000] = 5.0
    x = x.to(dtype)
    ids = torch.arange(rows) * 61 % V
    want = formula(x, ids)
    for k in (1, 7, 64):
        got, _ = call(x, ids, k)
        check_values(got, want, V)
        check_top(got, x, want, k)
