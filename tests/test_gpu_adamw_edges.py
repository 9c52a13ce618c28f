"""What an AdamW step refuses to read, and what its object tells of captured steps (needs the GPU)."""
import pytest

pytestmark = pytest.mark.gpu


def test_gradients_in_what_a_step_writes_are_refused(gpu_ctx):
    """Another parameter's values, moments or copy, an own array at another place or with values of another size, and the rate or the step's number among them."""
    import torch
    import apoe
    store = torch.arange(4000, dtype=torch.float32, device="cuda")
    p, copies = [store[:1000], store[1000:2000]], [torch.zeros(1000, dtype=torch.float16, device="cuda"), None]
    opt = apoe.AdamW(gpu_ctx, p, copies=copies)
    free, state, kept = store[2000:3000], opt.state(), store.clone()
    m, v = state["m"], state["v"]
    at = opt.offsets[1]
    for grads in ([p[1], free], [free, p[0]], [store[500:1500], None], [store[1:1001], None], [store[1500:2500], None], [None, copies[0]], [None, copies[0].view(torch.bfloat16)],
                  [m[at:at + 1000], None], [None, v[:1000]], [p[0].view(torch.float16)[:1000], None]):
        with pytest.raises(apoe.ApoeError, match="the same memory"):
            opt.step(grads, 0.1)
    with pytest.raises(apoe.ApoeError, match="the same memory"):
        opt.step([free, None], p[1][5])
    with pytest.raises(apoe.ApoeError, match="the same memory"):
        opt.step([free, None], 0.1, t=m[at:at + 1].view(torch.int32))
    assert bool((store == kept).all()) and not bool(m.any()) and not bool(v.any()) and opt.t == 0
    opt.close()


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_beside_or_in_their_own_parameter(gpu_ctx, bits):
    """A gradient that is the parameter itself, or its copy (each value is read before it is written), and one that begins where another array ends."""
    import torch
    import apoe
    g = torch.Generator().manual_seed(1)
    store = torch.randn(2400, generator=g).cuda()
    half = torch.randn(700, generator=g).half().cuda()

    def run(own):
        buf, copy = store.clone(), half.clone()
        a, b = buf[:1100], buf[1100:1800]
        opt = apoe.AdamW(gpu_ctx, [a, b], copies=[None, copy], bits=bits, seed=3)
        for _ in range(2):
            opt.step([a if own else a.clone(), copy if own else copy.clone()], 0.1)
        opt.step([None, buf[1800:2400].repeat(2)[:700]], 0.1)
        out = [buf, copy, *opt.moments()]
        opt.close()
        return out
    for x, y in zip(run(True), run(False)):
        assert bool((x == y).all())


@pytest.mark.parametrize("after", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
def test_the_number_of_captured_steps(bits, after):
    """Steps whose number is a tensor are counted as the GPU takes them, whether the program counts up before or behind each: an object that goes on from the state, and the
    object itself without a graph, take the next one."""
    import torch
    import apoe
    g = torch.Generator().manual_seed(4)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    ctx = apoe.Context(0, stream=stream)
    with torch.cuda.stream(stream):
        first, grad = torch.randn(1000, generator=g).cuda(), [(0.01 * torch.randn(1000, generator=g)).cuda()]
        eager, graphed = first.clone(), first.clone()
        want, opt = (apoe.AdamW(ctx, [p], bits=bits, seed=5) for p in (eager, graphed))
        for o in (want, opt):
            o.step(grad, 0.1)
        t, lr = torch.full((1,), 2 if after else 1, dtype=torch.int32, device="cuda"), torch.full((1,), 0.1, device="cuda")
    stream.synchronize()
    assert opt.state()["t"] == 1
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        if not after:
            t.add_(1)
        opt.step(grad, lr, t=t)
        if after:
            t.add_(1)
    assert opt.state()["t"] == 1  # captured, not run
    for k in range(3):
        with torch.cuda.stream(stream):
            graph.replay()
            want.step(grad, 0.1)
            torch.randn(1000, device="cuda").sum()
        assert opt.state()["t"] == opt.t == k + 2
    assert float((eager - graphed).abs().max()) <= 2.0 ** -20  # lr is rounded to a float: 3 steps of 0.1 at most, each off by 2^-24 of it, and the factors' last places
    with torch.cuda.stream(stream):
        graphed.copy_(eager)
        state = {k: (v.clone() if isinstance(v, torch.Tensor) else v) for k, v in want.state().items()}
        on = apoe.AdamW(ctx, [again := eager.clone()], bits=bits, seed=5, state=dict(state, t=opt.state()["t"]))
        for k, v in opt.state().items():
            if k != "t":
                v.copy_(want.state()[k])
        for o in (want, opt, on):
            o.step(grad, 0.1)
        assert want.t == opt.t == on.t == 5
    stream.synchronize()
    assert bool((eager == graphed).all()) and bool((eager == again).all())
    del graph
    ctx.close()


def test_a_number_without_gradients(gpu_ctx):
    """A step in which no parameter has a gradient counts, with a tensor as without."""
    import torch
    import apoe
    opt = apoe.AdamW(gpu_ctx, [torch.zeros(8, device="cuda")])
    opt.step([None], 0.1)
    assert opt.state()["t"] == 1
    opt.step([None], 0.1, t=torch.full((1,), 9, dtype=torch.int32, device="cuda"))
    assert opt.state()["t"] == 9
    opt.step([None], 0.1)
    assert opt.state()["t"] == opt.t == 10
    opt.close()


def test_a_capture_without_a_number_after_one_with(gpu_ctx):
    """What the GPU counts cannot be asked during a capture: such a step is refused there, and nothing of it is captured."""
    import torch
    import apoe
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    ctx = apoe.Context(0, stream=stream)
    with torch.cuda.stream(stream):
        p, g = torch.ones(300, device="cuda"), [torch.ones(300, device="cuda")]
        t, total = torch.full((1,), 1, dtype=torch.int32, device="cuda"), torch.zeros(1, device="cuda")
        opt = apoe.AdamW(ctx, [p])
        opt.step(g, 0.1, t=t)
    stream.synchronize()
    kept, graph = p.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        with pytest.raises(apoe.ApoeError, match="capture"):
            opt.step(g, 0.1)
        total.add_(1)
    for k in range(3):
        with torch.cuda.stream(stream):
            graph.replay()
        stream.synchronize()
        assert float(total) == k + 1 and bool((p == kept).all()) and opt.t == 1
    del graph
    ctx.close()
