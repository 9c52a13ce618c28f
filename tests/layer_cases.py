"""What the tests of embed, layer_norm, linear and AdamW share: matrices with something between their rows, and comparisons."""
U = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}    # half a step, relative
SMALL = {"float32": 2.0 ** -149, "float16": 2.0 ** -24, "bfloat16": 2.0 ** -133}  # the smallest number: a rounding below it
E = 2.0 ** -24
TYPES = ["float16", "bfloat16", "float32"]


def matrix(g, n, d, dtype, scale=1.0, pad=0, shift=0):
    """A random matrix on the GPU whose rows are `pad` elements apart and begin `shift` elements behind the allocation; between them NaN."""
    import torch
    dt = getattr(torch, dtype)
    store = torch.full((n * (d + pad) + shift,), float("nan"), dtype=dt, device="cuda")
    v = store[shift:].view(n, d + pad)[:, :d] if n else torch.empty(0, d, dtype=dt, device="cuda")
    v.copy_((scale * torch.randn(n, d, generator=g)).to(dt))
    return v


def room(n, d, dtype, pad=3):
    """(a matrix to write to, a check that nothing around it was written): NaN before, between and behind its rows."""
    import torch
    store = torch.full((n + 2, d + pad), float("nan"), dtype=getattr(torch, dtype), device="cuda")
    inner = store[1:n + 1, :d]

    def untouched():
        outside = store.clone()
        outside[1:n + 1, :d] = float("nan")
        return bool(outside.isnan().all())
    return inner, untouched


def close(got, want, tol, name=""):
    """|got - want| <= tol everywhere; what is not finite agrees."""
    import torch
    got, want = got.detach().cpu().double(), want.detach().cpu().double()
    tol = tol.detach().cpu().double() if isinstance(tol, torch.Tensor) else torch.full_like(want, tol)
    assert got.shape == want.shape, (name, got.shape, want.shape)
    odd = ~torch.isfinite(want)
    assert bool((torch.isfinite(got) == ~odd).all()), (name, "not finite", int((torch.isfinite(got) != ~odd).sum()))
    assert bool((got.isnan() == want.isnan()).all()), name
    d = torch.where(odd, torch.zeros_like(got), (got - want).abs())
    bad = ~(d <= torch.where(odd, torch.ones_like(tol), tol))
    assert not bool(bad.any()), (name, float((d / (tol + 1e-300)).nan_to_num(0).max()), int(bad.sum()), [tuple(x.tolist()) for x in bad.nonzero()[:4]])


def captured(ctx_of, call, times=3):
    """Runs `call(ctx)` on a stream of its own, captures it, and replays it with other work in between; yields what each replay left. The
    outputs of the capture are the graph's own."""
    import torch
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    ctx = ctx_of(stream)
    with torch.cuda.stream(stream):
        call(ctx)  # the workspace grows
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = call(ctx)
    for i in range(times):
        with torch.cuda.stream(stream):
            for t in out.values():
                t.fill_(float("nan") if t.is_floating_point() else 1)
            torch.randn(1000, device="cuda").sum()
            graph.replay()
        stream.synchronize()
        yield {k: t.clone() for k, t in out.items()}
    ctx.close()
