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
