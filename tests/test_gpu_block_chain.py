"""The operators around the mixers one after the other, as a block's MLP and a model's head run them: norm with the
residual stream, swiglu up projection, down projection onto the stream, final norm, LM head, log probabilities; its
training step against 64 bits, the step of a few rows in a captured graph, and two of them at once.

Tolerance of the chain, relative norm: about ten tensors round on the way forward and as many gradients on the way
back, each by u / 1.7 in the mean and independently, and the swiglu and the norms pass an error on by at most about 2:
2 sqrt(20) u / 1.7 = 5.3 u, u = 2^-8 (bf16) or 2^-11 (fp16).
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

D64 = torch.float64
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch.device("cuda")


def make(B, T, D, inter, V, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)

    def rnd(*shape, scale=1.0):
        return torch.randn(*shape, generator=gen) * scale

    p = dict(x=rnd(B, T, D), o=rnd(B, T, D, scale=0.5), w1=1 + rnd(D, scale=0.1), gate_up=rnd(2 * inter, D, scale=D ** -0.5),
             down=rnd(D, inter, scale=inter ** -0.5), w2=1 + rnd(D, scale=0.1), b2=rnd(D, scale=0.1),
             head=rnd(V, D, scale=2 * D ** -0.5))
    ids = torch.randint(0, V, (B, T), generator=gen)
    ids[torch.rand(B, T, generator=gen) < 0.2] = -100
    return {n: t.to(dtype) for n, t in p.items()}, ids


def ours(p, ids, top_k=0):
    from ccq_amd import fused_linear, layer_norm, rms_norm, token_logprobs
    h, s = rms_norm(p["o"], p["w1"], residual=p["x"])
    s = fused_linear(fused_linear(h, p["gate_up"], activation="swiglu"), p["down"], residual=s)
    logits = fused_linear(layer_norm(s, p["w2"], p["b2"]), p["head"])
    return logits, token_logprobs(logits, ids, top_k=top_k)


def formula(p, ids):
    s = p["x"] + p["o"]
    h = s / torch.sqrt(s.pow(2).mean(-1, keepdim=True) + 1e-5) * p["w1"]
    g, u = (h @ p["gate_up"].T).chunk(2, -1)
    s = s + (g * torch.sigmoid(g) * u) @ p["down"].T
    c = s - s.mean(-1, keepdim=True)
    logits = (c / torch.sqrt(c.pow(2).mean(-1, keepdim=True) + 1e-5) * p["w2"] + p["b2"]) @ p["head"].T
    lp = torch.log_softmax(logits, -1)
    keep = ids != -100
    logp = torch.where(keep, lp.gather(-1, ids.clamp_min(0)[..., None])[..., 0], 0.0)
    ent = torch.where(keep, -(lp.exp() * lp).sum(-1), 0.0)
    return logits, logp, ent


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("shape", [(2, 150, 256, 320, 1000), (3, 37, 200, 136, 501), (1, 1, 64, 96, 33)], ids=str)
def test_block_training_step(shape, dtype):
    print("test_block_training_step", shape, dtype, flush=True)
    dev = _cuda()
    p, ids = make(*shape, dtype)
    ids[0, 0] = 7
    ref = {n: t.to(D64).requires_grad_() for n, t in p.items()}
    _, logp, ent = formula(ref, ids)
    n = (ids != -100).sum()
    (-(logp.sum()) / n - 0.01 * ent.sum() / n).backward()
    got = {n: t.to(dev).requires_grad_() for n, t in p.items()}
    _, r = ours(got, ids.to(dev))
    (-(r.logprobs.sum()) / n - 0.01 * r.entropy.sum() / n).backward()
    tol = 5.3 * U[dtype]
    assert ((r.logprobs.detach().cpu().double() - logp.detach()).norm() / logp.detach().norm()).item() <= tol
    for name, t in ref.items():
        rel = ((got[name].grad.cpu().double() - t.grad).norm() / t.grad.norm()).item()
        assert rel <= tol, (name, rel)


def test_block_step_captured_twice():
    """A decode step's rows in two graphs over the same weights, replayed in turn: each has its own buffers."""
    dev = _cuda()
    p, _ = make(4, 1, 256, 320, 1000, torch.bfloat16)
    p = {n: t.to(dev) for n, t in p.items()}
    ids = torch.tensor([[1], [999], [5], [17]], device=dev)
    inputs = [[torch.randn(4, 1, 256, device=dev, generator=torch.Generator(dev).manual_seed(2 * i + k)).bfloat16()
               for k in range(2)] for i in range(3)]

    def step(x, o):
        logits, r = ours({**p, "x": x, "o": o}, ids, top_k=5)
        return [logits, *r]

    want = [[t.clone() for t in step(*i)] for i in inputs]
    graphs = []
    for _ in range(2):
        x, o = (t.clone() for t in inputs[0])
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(x, o)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(x, o)
        graphs.append((x, o, g, out))
    for k in (0, 1, 2, 1):
        for j, (x, o, g, out) in enumerate(graphs):
            for s, t in zip((x, o), inputs[(k + j) % 3]):
                s.copy_(t)
            g.replay()
        torch.cuda.synchronize()
        for j, (x, o, g, out) in enumerate(graphs):
            assert all(torch.equal(a, b) for a, b in zip(out, want[(k + j) % 3]))
        step(*inputs[0])


def test_two_streams_at_once():
    dev = _cuda()
    p, ids = make(2, 150, 256, 320, 1000, torch.bfloat16)
    p, ids = {n: t.to(dev) for n, t in p.items()}, ids.to(dev)
    q = {**p, "x": p["x"].flip(0).contiguous()}
    want = [[t.clone() for t in (lambda r: [r[0], r[1].logprobs, r[1].entropy])(ours(v, ids))] for v in (p, q)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    out = [[], []]
    for _ in range(5):
        for k, v in enumerate((p, q)):
            with torch.cuda.stream(streams[k]):
                logits, r = ours(v, ids)
                out[k].append([logits, r.logprobs, r.entropy])
    torch.cuda.synchronize()
    for k in range(2):
        for got in out[k]:
            assert all(torch.equal(a, b) for a, b in zip(got, want[k]))


def each_operator(dev):
    """Every differentiable operator as a function of one leaf."""
    import ccq_amd
    gen = torch.Generator(dev).manual_seed(11)
    w = torch.randn(64, 64, device=dev, generator=gen).bfloat16()
    v = torch.ones(64, device=dev)
    ids = torch.arange(6, device=dev)
    return {"rms_norm": lambda x: ccq_amd.rms_norm(x, v), "layer_norm": lambda x: ccq_amd.layer_norm(x, v, v),
            "fused_linear": lambda x: ccq_amd.fused_linear(x, w, activation="silu"),
            "token_logprobs": lambda x: ccq_amd.token_logprobs(x, ids).logprobs}


@pytest.mark.parametrize("name", ["rms_norm", "layer_norm", "fused_linear", "token_logprobs"])
def test_second_derivative_raises(name):
    dev = _cuda()
    x = torch.randn(6, 64, device=dev, generator=torch.Generator(dev).manual_seed(1)).bfloat16().requires_grad_()
    dx, = torch.autograd.grad(each_operator(dev)[name](x).float().square().sum(), x, create_graph=True)
    assert torch.isfinite(dx).all()
    with pytest.raises(RuntimeError, match="twice"):
        dx.float().square().sum().backward()


@pytest.mark.parametrize("name", ["rms_norm", "layer_norm", "fused_linear", "token_logprobs"])
def test_captured_backward_beside_an_eager_graph_of_its_leaf(name):
    """Refused where the eager graph is of another stream (autograd would wait for it and end the process); captured and
    replayed once that graph is gone."""
    dev = _cuda()
    f = each_operator(dev)[name]
    x = torch.randn(6, 64, device=dev, generator=torch.Generator(dev).manual_seed(1)).bfloat16().requires_grad_()
    y = f(x)
    dy = torch.randn(y.shape, device=dev, generator=torch.Generator(dev).manual_seed(2)).to(y.dtype)
    want, = torch.autograd.grad(y, x, dy, retain_graph=True)
    torch.cuda.synchronize()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(RuntimeError, match="alive"):
            f(x).backward(dy)
    del y
    assert x.grad is None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, = torch.autograd.grad(f(x), x, dy)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        got.zero_()
        f(x.detach())
        torch.cuda.synchronize()
