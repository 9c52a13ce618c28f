"""AdamW over many parameters, moments in 32 bits and in 8, against the formula in 64 bits (needs the GPU).

Tolerances. 32 bits: m' and v' are two fused operations each: 3 2^-24 of their terms (where g and m nearly cancel, that is more than m' has); the step is a
quotient of m' and a root: m' is off by a = 3 2^-24 (|m| + |m'| + |g|), which the quotient passes on as a / ((1 - b1^t) (root + eps)), v' by 3 2^-24 of
itself (its terms are not negative), half of which the root passes on, and the factors, the root and the quotient round six times: 8 2^-24 of the
step in all; p adds two roundings of its own. 8 bits: the code is decided in 64 bits, so it is the reference's unless chance and share agree to 1e-9; p
is stepped from the moments before they are rounded."""
import pytest

from layer_cases import E, TYPES, U, close

pytestmark = pytest.mark.gpu
BETAS, EPS, LR = (0.9, 0.999), 1e-8, 1e-2
SIZES = [1, 255, 256, 257, 1000, 5, 4096, 4097, 12_345, 64]


def mix(h):
    h = ((h ^ (h >> 16)) * 0x85EBCA6B) & 0xFFFFFFFF
    h = ((h ^ (h >> 13)) * 0xC2B2AE35) & 0xFFFFFFFF
    return h ^ (h >> 16)


def chances(seed, step, tensor, n, which):
    """Of each value of a parameter: from its block's number and its place in the block."""
    import torch
    key = mix(mix(mix(torch.tensor(seed)) ^ step) ^ tensor)
    at = torch.arange(n)
    block = mix(mix(key ^ (at // 256)) ^ 0)
    return (mix((block + 2 * (at % 256) + which) & 0xFFFFFFFF).double() + 0.5) / 2 ** 32


def coded(x, list_, chance, keep):
    """(codes, scales, how near each decision was) of x >= 0 by search among all values that a block of its largest can hold."""
    import torch
    n = len(x)
    padded = torch.cat((x, torch.zeros(-n % 256, dtype=x.dtype))).view(-1, 256)
    top = padded.amax(1).float()
    t = top.double().repeat_interleave(256)[:n]
    share = torch.where(t > 0, x / t.clamp(min=1e-300), torch.zeros_like(x)).clamp(max=1.0)
    low = (torch.searchsorted(list_, share, right=True) - 1).clamp(0, len(list_) - 2)
    way = (share - list_[low]) / (list_[low + 1] - list_[low])
    code = low + (chance < way).long()
    return torch.where(x > 0, code.clamp(min=1 if keep else 0), torch.zeros_like(code)), top, (way - chance).abs()


def make(sizes, seed, shift=0, grads=None):
    import torch
    g = torch.Generator().manual_seed(seed)

    def buffers(scale, dtypes):
        out = []
        for n, dt in zip(sizes, dtypes):
            store = torch.full((n + shift + 1,), float("nan"), dtype=getattr(torch, dt), device="cuda")
            store[shift:shift + n] = (scale * torch.randn(n, generator=g) * torch.exp(torch.randn(n, generator=g))).cuda()
            out.append(store[shift:shift + n])
        return out
    types = grads or [TYPES[i % 3] for i in range(len(sizes))]
    return buffers(0.1, ["float32"] * len(sizes)), buffers(0.01, types), g


def step64(p, g, m, v, t, decay, scale):
    g = scale * g
    m, v = m + (1 - BETAS[0]) * (g - m), v + (1 - BETAS[1]) * (g * g - v)  # in this order: a block's largest is rounded to a float, and often lies half way
    step = (m / (1 - BETAS[0] ** t)) / ((v / (1 - BETAS[1] ** t)) ** 0.5 + EPS)
    return p - LR * (decay * p + step), m, v, step


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("shift", [0, 1])
def test_steps(gpu_ctx, bits, shift):
    """Three steps over parameters of many sizes, gradients of each type, copies of each type or none; nothing around a parameter is written."""
    import torch
    import apoe
    params, grads, g = make(SIZES, 1, shift)
    copies = [None if i % 3 == 0 else torch.full((n + 1,), float("nan"), dtype=torch.float16 if i % 3 == 1 else torch.bfloat16, device="cuda")[:n] for i, n in enumerate(SIZES)]
    decay = [0.1 * (i % 2) for i in range(len(SIZES))]
    opt = apoe.AdamW(gpu_ctx, params, copies=copies, bits=bits, betas=BETAS, eps=EPS, weight_decay=decay, seed=77)
    ref = [(p.cpu().double(), torch.zeros(n, dtype=torch.float64), torch.zeros(n, dtype=torch.float64)) for p, n in zip(params, SIZES)]
    lists = ((torch.arange(128).double() / 127) ** 2, (torch.arange(256).double() / 255) ** 4)
    for t in range(1, 4):
        before = [p.cpu().double() for p in params]
        for x in grads:
            x.copy_(x * (torch.randn(x.shape, generator=g).cuda()).to(x.dtype))
        opt.step(grads, LR, grad_scale=0.5)
        assert opt.t == t
        ms, vs = opt.moments()
        for i, n in enumerate(SIZES):
            at = opt.offsets[i]
            _, m0, v0 = ref[i]
            gd = grads[i].cpu().double()
            p, m, v, step = step64(before[i], gd, m0, v0, t, decay[i], 0.5)
            from_m = 3 * E * (m0.abs() + m.abs() + (0.5 * gd).abs()) / ((1 - BETAS[0] ** t) * ((v / (1 - BETAS[1] ** t)) ** 0.5 + EPS))
            got_m, got_v = ms[at:at + n].cpu().double(), vs[at:at + n].cpu().double()
            close(params[i], p, 4 * E * p.abs() + LR * E * (16 * step.abs() + 4 * decay[i] * before[i].abs()) + LR * from_m + 2.0 ** -140, ("p", t, n))
            if bits == 32:
                close(got_m, m, 3 * E * (m0.abs() + m.abs() + (0.5 * gd).abs()) + 2.0 ** -140, ("m", t, n))
                close(got_v, v, 3 * E * (v0 + v + (0.5 * gd) ** 2) + 2.0 ** -140, ("v", t, n))
            else:
                for got, x, list_, which, sign in ((got_m, m, lists[0], 0, m.sign()), (got_v, v, lists[1], 1, 1.0)):
                    code, top, near = coded(x.abs(), list_, chances(77, t, i, n, which), which == 1)
                    want = top.double().repeat_interleave(256)[:n] * list_[code] * sign
                    ok = (got - want).abs() <= 2 * E * want.abs()
                    assert bool((ok | (near < 1e-9)).all()), (which, t, n, int((~ok).sum()))
            if bits == 8:  # the next step goes on from what is stored: codes and scales, whose product has more bits than a float
                st = opt.state()
                blocks = slice(at // 256, at // 256 + -(-n // 256))
                c, r = st["m"][at:at + n].cpu().long(), st["v"][at:at + n].cpu().long()
                tm, tv = (st[k][blocks].cpu().double().repeat_interleave(256)[:n] for k in ("m_scale", "v_scale"))
                got_m, got_v = tm * ((c * c.abs()).double() * (1 / 127 ** 2)), tv * ((r ** 4).double() * (1 / 255 ** 4))
            ref[i] = (None, got_m, got_v)
            if copies[i] is not None:
                assert bool((copies[i] == params[i].to(copies[i].dtype)).all())
    for tensors in (params, grads, copies):
        for x in tensors:
            if x is not None:
                whole = torch.empty(0, dtype=x.dtype, device="cuda").set_(x.untyped_storage())
                assert int(whole.isnan().sum()) == len(whole) - len(x)


def test_more_parameters_than_a_launch_holds(gpu_ctx):
    import torch
    import apoe
    sizes = [3 + (i * 37) % 600 for i in range(150)] + [0, 9]
    for bits in (32, 8):
        params, grads, _ = make(sizes, 2)
        alone = [p.clone() for p in params]
        opt = apoe.AdamW(gpu_ctx, params, bits=bits, weight_decay=0.1)
        opt.step(grads, LR)
        for i, (p, g) in enumerate(zip(alone, grads)):  # a first step does not depend on the codes
            one = apoe.AdamW(gpu_ctx, [p], bits=bits, weight_decay=0.1)
            one.step([g], LR)
            assert bool((p == params[i]).all()), i


def test_a_parameter_without_gradient_stays(gpu_ctx):
    import torch
    import apoe
    for bits in (32, 8):
        params, grads, _ = make([300, 300, 300], 3)
        opt = apoe.AdamW(gpu_ctx, params, bits=bits)
        opt.step(grads, LR)
        before = [p.clone() for p in params], [x.clone() for x in opt.moments()]
        opt.step([grads[0], None, grads[2]], LR)
        assert bool((params[1] == before[0][1]).all()) and not bool((params[0] == before[0][0]).all())
        at = slice(opt.offsets[1], opt.offsets[1] + 300)
        for x, y in zip(opt.moments(), before[1]):
            assert bool((x[at] == y[at]).all())


def test_eight_bits_follow_thirty_two(gpu_ctx):
    """2000 steps with noisy gradients whose sizes differ by 1e4 in a block, some of which stop half way: the moments' means follow (an average that is
    rounded to the nearest code stands still), within the spread of what chance adds. A moment moves by 0.1 (0.001) of its gap to the code
    beside it a step and is then off by up to a gap; its average over the last values has a variance of a gap's square over its decay's
    length: at c codes from zero a gap is 2 / c (4 / c) of the value; v of a block's smallest values is held at code 1 or more."""
    import torch
    import apoe
    gen = torch.Generator().manual_seed(4)
    n = 256 * 40
    size = (10 ** (-4 * torch.rand(n, generator=gen))).cuda()
    off_at_half = torch.arange(n, device="cuda") % 4 == 0
    p = [torch.zeros(n, device="cuda") for _ in range(2)]
    opts = [apoe.AdamW(gpu_ctx, [x], bits=b, weight_decay=0.0, seed=5) for x, b in zip(p, (32, 8))]
    total = [0.0, 0.0]
    for t in range(2000):
        g = size * (1 + 0.5 * torch.randn(n, generator=gen).cuda())
        if t >= 1000:
            g = torch.where(off_at_half, torch.zeros_like(g), g)
        for o in opts:
            o.step([g], 1e-3)
        if t >= 1800:
            for k in (0, 1):
                total[k] = total[k] + opts[k].moments()[1].double() / 200
    large = (size > 0.03) & ~off_at_half   # v a thousandth of the largest and more: code 45 and up, gaps of a tenth
    ratio = total[1][large] / total[0][large]
    assert abs(float(ratio.mean()) - 1) < 0.02, float(ratio.mean())
    gone = (size > 0.03) & off_at_half     # decayed to exp(-0.9) of what they were
    ratio = total[1][gone] / total[0][gone]
    assert abs(float(ratio.mean()) - 1) < 0.05, float(ratio.mean())
    a, b = p[0][large].double(), p[1][large].double()
    assert float((a - b).norm() / a.norm()) < 0.05


def test_state_goes_on(gpu_ctx):
    import torch
    import apoe
    for bits in (32, 8):
        params, grads, _ = make([700, 20, 5000], 5)
        twin = [p.clone() for p in params]
        a, b = apoe.AdamW(gpu_ctx, params, bits=bits, seed=3), apoe.AdamW(gpu_ctx, twin, bits=bits, seed=3)
        for _ in range(2):
            a.step(grads, LR)
            b.step(grads, LR)
        later = apoe.AdamW(gpu_ctx, twin, bits=bits, seed=3, state={k: v.clone() if k != "t" else v for k, v in b.state().items()})
        b.close()
        a.step(grads, LR)
        later.step(grads, LR)
        assert later.t == 3
        for x, y in zip(params, twin):
            assert bool((x == y).all())
        for x, y in zip(a.moments(), later.moments()):
            assert bool((x == y).all())


def test_what_is_not_finite_is_seen(gpu_ctx):
    import torch
    import apoe
    for bits in (32, 8):
        for bad in (float("nan"), float("inf")):
            p, g = torch.zeros(1000, device="cuda"), torch.ones(1000, device="cuda")
            g[300] = bad
            opt = apoe.AdamW(gpu_ctx, [p], bits=bits)
            opt.step([g], LR)
            assert not bool(torch.isfinite(p[300])) or bad == float("inf")
            assert bool(torch.isfinite(p[:256]).all()) and bool(torch.isfinite(p[512:]).all())
            m, v = opt.moments()
            assert not bool(torch.isfinite(m[300])) and not bool(torch.isfinite(v[300])) and bool(torch.isfinite(m[:256]).all()) and bool(torch.isfinite(m[512:]).all())
            opt.step([torch.ones(1000, device="cuda")], LR)
            assert bool(p[300].isnan())


def test_zero_gradients_and_moments(gpu_ctx):
    import torch
    import apoe
    for bits in (32, 8):
        p = torch.ones(600, device="cuda")
        opt = apoe.AdamW(gpu_ctx, [p], bits=bits, weight_decay=0.5)
        opt.step([torch.zeros(600, device="cuda")], 0.1)
        assert bool(((p - 0.95).abs() < 1e-6).all()) and not any(bool(x.any()) for x in opt.moments())


@pytest.mark.parametrize("bits", [32, 8])
def test_without_eps(gpu_ctx, bits):
    """A first step without eps goes by lr against the sign, whatever the gradient's size: v of the smallest, 1e-17, is 1e-37, where floats have all their bits
    (a step: eight roundings)."""
    import torch
    import apoe
    g = torch.tensor([1e-17, -1e-17, 1e-10, 1.0, -1e4], device="cuda")
    p = torch.zeros(5, device="cuda")
    if bits == 8:  # a block each: one that shares a block with far larger ones has a code of one, but the step is taken before that
        g, p = g.repeat_interleave(256), p.repeat_interleave(256)
    opt = apoe.AdamW(gpu_ctx, [p], bits=bits, eps=0.0, weight_decay=0.0)
    opt.step([g], 0.5)
    assert bool(((p + 0.5 * g.sign()).abs() <= 10 * E * 0.5).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_captured(bits):
    """A captured step reads its number and rate when it is replayed."""
    import torch
    import apoe
    params, grads, _ = make([700, 20, 5000], 6)
    twin = [p.clone() for p in params]
    start = [p.clone() for p in params]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    ctx = apoe.Context(0, stream=stream)
    a, b = apoe.AdamW(ctx, params, bits=bits, seed=9), apoe.AdamW(ctx, twin, bits=bits, seed=9)
    t, lr = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(1, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        a.step(grads, lr, t=t)
    assert a.t == 0
    for k in range(1, 5):
        with torch.cuda.stream(stream):
            t.fill_(k)
            lr.fill_(0.01 / k)
            graph.replay()
            b.step(grads, float(torch.tensor(0.01 / k)))
            torch.randn(100, device="cuda").sum()
        stream.synchronize()
        for x, y in zip(params, twin):
            assert bool(((x - y).abs() <= 4 * E * y.abs() + 0.01 * 8 * E).all())
        for x, y in zip(a.moments(), b.moments()):
            assert bool((x == y).all())
    assert not bool((params[0] == start[0]).all())
    del graph
    ctx.close()


def test_closed(gpu_ctx):
    import torch
    import apoe
    p = torch.zeros(10, device="cuda")
    ctx = apoe.Context(0)
    a, b = apoe.AdamW(ctx, [p]), apoe.AdamW(ctx, [p])
    a.close()
    for opt in (a, b):
        if opt is b:
            ctx.close()
        with pytest.raises(apoe.ApoeError, match="closed"):
            opt.step([p], LR)


def test_arrays_that_share_memory_are_refused(gpu_ctx):
    import torch
    import apoe
    store = torch.zeros(2000, device="cuda")
    half = torch.zeros(1000, dtype=torch.float16, device="cuda")
    for params, copies in (([store[:600], store[500:]], None), ([store[:600]] * 2, None), ([store[:1000], store[1000:]], [half, half]), ([store], [store.view(torch.float16)[:2000]])):
        with pytest.raises(apoe.ApoeError, match="share memory"):
            apoe.AdamW(gpu_ctx, params, copies=copies)
    apoe.AdamW(gpu_ctx, [store[:600], store[600:]])


def test_codes_next_to_a_step_of_the_list(gpu_ctx):
    """Chances next to one, for numbers just below a code (or a block's largest, rounded up to a float): they go to the code beneath where the chance is above the
    share, however near both are to one. Of 2^24 values those with such a chance are taken, each with the first or the second moment at a step's end."""
    import torch
    import apoe
    n, seed = 1 << 24, 5
    lists = ((torch.arange(128).double() / 127) ** 2, (torch.arange(256).double() / 255) ** 4)
    g = torch.Generator().manual_seed(3)
    grads = torch.zeros(n)
    blocks = []
    chance = [chances(seed, 1, 0, n, which) for which in (0, 1)]
    for which in (0, 1):
        places = (chance[which] > 1 - 4e-6).nonzero().flatten().tolist()
        assert len(places) > 30
        for at in places:
            block = at // 256
            if block in blocks:
                continue
            blocks.append(block)
            if len(blocks) % 2:  # alone in its block: its largest
                grads[at] = torch.randn(1, generator=g)[0]
                continue
            grads[block * 256 + (at + 1) % 256] = top = float(torch.rand(1, generator=g) + 0.5)
            k = int(torch.randint(20, len(lists[which]) - 1, (1,), generator=g))
            x = top * float(lists[which][k]) ** (1.0 if which == 0 else 0.5)
            grads[at] = torch.nextafter(torch.tensor(x), torch.tensor(0.0))
    at = (torch.tensor(blocks)[:, None] * 256 + torch.arange(256)).flatten()
    x = grads[at].double()
    _, m, v, _ = step64(0.0, x, torch.zeros_like(x), torch.zeros_like(x), 1, 0.0, 1.0)
    opt = apoe.AdamW(gpu_ctx, [torch.zeros(n, device="cuda")], bits=8, betas=BETAS, eps=EPS, seed=seed)
    opt.step([grads.cuda()], LR)
    state = {k: t.cpu() for k, t in opt.state().items() if k != "t"}
    below = 0
    for name, value, list_, which in (("m", m.abs(), lists[0], 0), ("v", v, lists[1], 1)):
        code, top, near = coded(value, list_, chance[which][at], which == 1)
        got = state[name][at].long().abs()
        assert bool((state[name + "_scale"][torch.tensor(blocks)] == top).all())
        bad = (got != code) & (near > 1e-9)
        assert not bool(bad.any()), (name, int(bad.sum()), got[bad].tolist(), code[bad].tolist(), near[bad].tolist())
        t = top.double().repeat_interleave(256)
        below += int(((value > 0) & (chance[which][at] > 1 - 4e-6) & (list_[code] * t < value)).sum())
    assert below > 5  # numbers that stay beneath the next code, against nearly all chances
