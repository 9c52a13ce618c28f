"""embed, layer_norm, linear, their gradients and AdamW as one layer in front of the softmax loss: the example's adapter (needs the GPU)."""
import math
import os

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def example(monkeypatch):
    monkeypatch.syspath_prepend(os.path.join(ROOT, "allan-poe_amd", "examples"))
    import query_adapter
    return query_adapter


def world(dtype, m=70, dim=64, hidden=104, vocab=90, n=300):
    import torch
    g = torch.Generator().manual_seed(1)
    counts = torch.randint(0, 9, (m,), generator=g)
    off = torch.zeros(m + 1, dtype=torch.int32)
    off[1:] = counts.cumsum(0)
    total = int(off[-1])
    terms = off.cuda(), torch.randint(0, vocab, (total,), generator=g, dtype=torch.int32).cuda(), torch.rand(total, generator=g).cuda()
    unit = lambda t: t / t.norm(dim=1, keepdim=True)  # noqa: E731
    x, rows = (unit(torch.randn(k, dim, generator=g)).to(dtype).cuda() for k in (m, n))
    t_off = torch.arange(m + 1, dtype=torch.int32, device="cuda")
    t_idx = torch.randint(0, n, (m,), generator=g, dtype=torch.int32).cuda()
    return x, terms, rows, t_off, t_idx


def adapter_of(example, ctx, dtype, bits=32, dim=64, hidden=104, vocab=90):
    import torch
    a = example.MlpAdapter(ctx, dim=dim, hidden=hidden, vocab=vocab, dtype=dtype, bits=bits)
    g = torch.Generator().manual_seed(2)
    a.params["E"].copy_(0.3 * torch.randn(vocab, dim, generator=g))  # a table that has learned something
    a.params["W2"].mul_(20)
    for k, c in a.copies.items():
        c.copy_(a.params[k])
    return a


def formula(a, x, terms, rows, t_idx, temperature):
    """Loss and gradients of the whole layer in 64 bits, by automatic differentiation."""
    import torch
    p = {k: (a._matrix(k) if k in a.copies else v).detach().cpu().double().requires_grad_() for k, v in a.params.items()}
    off, idx, val = (t.cpu() for t in terms)
    x, rows = x.cpu().double(), rows.cpu().double()
    row = torch.repeat_interleave(torch.arange(len(x)), (off[1:] - off[:-1]).long())
    e = x + a.SCALE * torch.zeros_like(x).index_add(0, row, p["E"][idx.long()] * val.double()[:, None])
    c = e - e.mean(1, keepdim=True)
    n = c / torch.sqrt((c * c).mean(1, keepdim=True) + 1e-5) * p["w"] + p["b"]
    z = n @ p["W1"].T + p["b1"]
    y = e + (z * 0.5 * torch.erfc(-z / math.sqrt(2.0))) @ p["W2"].T + p["b2"]
    s = (y / y.norm(dim=1, keepdim=True)) @ rows.T / temperature
    loss = torch.logsumexp(s, 1) - s.gather(1, t_idx.cpu().long()[:, None])[:, 0]
    grads = torch.autograd.grad(loss.mean() * a.LOSS_SCALE, list(p.values()))
    return loss.detach(), dict(zip(p, grads))


@pytest.mark.parametrize("dtype,off", [("float32", 1e-5), ("float16", 1e-2)])
def test_gradients_of_the_whole_layer(gpu_ctx, example, dtype, off):
    """Against the formula, relative to each gradient's norm. float32: some 200 operations between the loss and the table, each off by a few 2^-24 of terms that are
    a few times the result: 1e-5. float16: a rounding is off by up to 2^-11 (0.3 of that in the mean), some ten lie in the way of each gradient, and logits of up
    to 20 turn the queries' roundings of 2^-11 into 1 % of the exponentials at most: 1e-2."""
    import torch
    a = adapter_of(example, gpu_ctx, getattr(torch, dtype))
    x, terms, rows, t_off, t_idx = world(getattr(torch, dtype))
    loss, grads = a.gradients(x, terms, rows, t_off, t_idx, 0.05)
    want, want_grads = formula(a, x, terms, rows, t_idx, 0.05)
    assert float((loss.cpu().double() - want).abs().max()) <= 20 * off
    assert set(grads) == set(a.params)
    for k, w in want_grads.items():
        assert grads[k].shape == w.shape
        err = float((grads[k].cpu().double() - w).norm() / w.norm())
        assert err <= off, (k, err)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_training_step(example, bits):
    """A whole step, from the terms to the parameters, captured and replayed against the same steps without a graph: bit for bit, but for the rate and the step's
    number, which the graph reads on the GPU (rounded once more)."""
    import torch
    import apoe
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    ctx = apoe.Context(0, stream=stream)
    with torch.cuda.stream(stream):
        x, terms, rows, t_off, t_idx = world(torch.float16)
        graphed, eager = (adapter_of(example, ctx, torch.float16, bits) for _ in range(2))
        t, lr = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.full((1,), 1e-3, device="cuda")
        graphed.gradients(x, terms, rows, t_off, t_idx, 0.05)  # the workspace grows
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        loss, grads = graphed.gradients(x, terms, rows, t_off, t_idx, 0.05)
        t.add_(1)
        graphed.opt.step([grads[k] for k in graphed.params], lr, grad_scale=1 / graphed.LOSS_SCALE, t=t)
    for k in range(4):
        with torch.cuda.stream(stream):
            graph.replay()
            same = eager.step(x, terms, rows, t_off, t_idx, 0.05, 1e-3)
            torch.randn(1000, device="cuda").sum()
        stream.synchronize()
        if k == 0:
            assert bool((loss == same).all())
        for name, p in graphed.params.items():
            d = (p - eager.params[name]).abs().max()
            assert float(d) <= 2e-3 * 1e-3 * (k + 1), (name, float(d))  # steps of 1e-3, whose gradients differ once a half-precision copy is rounded the other way
    assert int(t) == 4
    del graph
    ctx.close()


@pytest.mark.parametrize("bits", ["32", "8"])
def test_the_example_runs(example, bits):
    import torch
    out = example.main(["--docs", "3000", "--train", "2048", "--held-out", "64", "--steps", "12", "--batch", "129", "--block", "mlp", "--bits", bits])
    assert out["block"] == "mlp" and out["steps"] == 12
    assert all(math.isfinite(v) for v in out.values() if not isinstance(v, str))
    assert 0.0 <= out["recall_at_10_after"] <= 1.0
