"""Layer norm and its gradients against the formula in 64 bits (needs the GPU).

Tolerances. A row's mean is off by at most d0 = 30 2^-24 of the mean magnitude of its values (16 values a thread, a tree over the threads, a factor), so n =
(x - mean) r by d = 2 d0 r and by 30 2^-24 of itself, plus the square of d in r, which the mean's error moves. y: that times |w|, the two operations
with w and b, half a step. grad_x is r times a sum of three terms: each off by 40 2^-24 of its magnitude and by what n is off; grad_w
and grad_b are sums over rows: (rows / workgroups + 80) 2^-24 of the sum of magnitudes, and what n is off."""
import pytest

from layer_cases import E, SMALL, TYPES, U, captured, close, matrix, room

pytestmark = pytest.mark.gpu


def formula(x, w, b, eps, dtype, grad_y=None, grad_skip=None):
    """(values, tolerances)"""
    import torch
    x = x.detach().cpu().double()
    n, d = x.shape
    w = torch.ones(d) if w is None else w.cpu()
    b = torch.zeros(d) if b is None else b.cpu()
    w, b, u, small = w.double(), b.double(), U[dtype], SMALL[dtype]
    c = x - x.mean(1, keepdim=True)
    r = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + eps)
    xn = c * r
    off = 2 * 30 * E * x.abs().mean(1, keepdim=True) * r
    rel = 30 * E + off * off
    n_off = off + rel * xn.abs()
    val, tol = dict(y=xn * w + b), {}
    tol["y"] = u * val["y"].abs() + w.abs() * n_off + 3 * E * (val["y"].abs() + b.abs() + (w * xn).abs()) + small
    if grad_y is not None:
        gy = grad_y.detach().cpu().double()
        g = gy * w
        val["grad_x"] = r * (g - g.mean(1, keepdim=True) - xn * (g * xn).mean(1, keepdim=True))
        size = r * (g.abs() + g.abs().mean(1, keepdim=True) + xn.abs() * (g * xn).abs().mean(1, keepdim=True))
        tol["grad_x"] = (40 * E + rel) * size + r * (n_off * (g * xn).abs().mean(1, keepdim=True) + xn.abs() * (g.abs() * n_off).mean(1, keepdim=True)) + small
        if grad_skip is not None:
            val["grad_x"] = val["grad_x"] + grad_skip.detach().cpu().double()
        tol["grad_x"] += (u + 2 * E) * val["grad_x"].abs()
        val["grad_w"], val["grad_b"] = (gy * xn).sum(0), gy.sum(0)
        sums = (n / 4 + 80) * E
        tol["grad_w"], tol["grad_b"] = sums * (gy * xn).abs().sum(0) + (gy.abs() * n_off).sum(0) + small, sums * gy.abs().sum(0) + small
    return val, tol


def vectors(g, d):
    import torch
    return (1 + 0.3 * torch.randn(d, generator=g)).cuda(), (0.3 * torch.randn(d, generator=g)).cuda()


SIZES = [(1, 1), (1, 1024), (2, 2), (3, 33), (5, 256), (17, 257), (64, 1000), (130, 1024), (9, 1032), (2100, 64), (6, 4096), (5, 4097), (3, 8192), (2, 8191)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d", SIZES)
def test_sizes_and_types(gpu_ctx, n, d, dtype):
    import torch
    import apoe
    g = torch.Generator().manual_seed(n + d)
    for pad, shift, skip in ((0, 0, False), (8, 0, True), (3, 1, True)):
        x, gy = matrix(g, n, d, dtype, 2.0, pad, shift), matrix(g, n, d, dtype, 1.0, pad, shift)
        x += 0.5
        gs = matrix(g, n, d, dtype, 1.0, pad, shift) if skip else None
        w, b = vectors(g, d)
        val, tol = formula(x, w, b, 1e-5, dtype, gy, gs)
        out, untouched = room(n, d, dtype)
        assert apoe.layer_norm(gpu_ctx, x, w, b, out=out) is out
        got = dict(apoe.layer_norm_grad(gpu_ctx, x, w, b, grad_y=gy, grad_skip=gs), y=out)
        assert set(got) == set(val)
        for k in val:
            close(got[k], val[k], tol[k], (k, pad))
        assert untouched()


@pytest.mark.parametrize("dtype", TYPES)
def test_without_vectors_and_parts(gpu_ctx, dtype):
    import torch
    import apoe
    g = torch.Generator().manual_seed(5)
    x, gy = matrix(g, 70, 200, dtype), matrix(g, 70, 200, dtype)
    w, b = vectors(g, 200)
    for ww, bb in ((None, None), (w, None), (None, b)):
        val, tol = formula(x, ww, bb, 1e-3, dtype, gy)
        close(apoe.layer_norm(gpu_ctx, x, ww, bb, eps=1e-3), val["y"], tol["y"])
        got = apoe.layer_norm_grad(gpu_ctx, x, ww, bb, eps=1e-3, grad_y=gy)
        assert set(got) == {"grad_x"} | ({"grad_w"} if ww is not None else set()) | ({"grad_b"} if bb is not None else set())
        for k in got:
            close(got[k], val[k], tol[k], k)


def test_in_place(gpu_ctx):
    import torch
    import apoe
    g = torch.Generator().manual_seed(6)
    x = matrix(g, 5000, 512, "bfloat16", pad=8)
    w, b = vectors(g, 512)
    want = apoe.layer_norm(gpu_ctx, x, w, b)
    apoe.layer_norm(gpu_ctx, x, w, b, out=x)
    assert bool((x == want).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_one_value_and_far_from_zero(gpu_ctx, dtype):
    """A row without any spread gives b; one far from zero with little spread is normed by that spread."""
    import torch
    import apoe
    g = torch.Generator().manual_seed(7)
    x = torch.zeros(6, 300)
    x[1], x[2], x[3] = 5.0, -1000.0, 64.0 + torch.randn(300, generator=g)
    x[4], x[5] = 1e-3 * torch.randn(300, generator=g), 1000.0 * torch.randn(300, generator=g)
    x = x.to(getattr(torch, dtype)).cuda()
    gy = matrix(g, 6, 300, dtype)
    w, b = vectors(g, 300)
    val, tol = formula(x, w, b, 1e-5, dtype, gy)
    close(apoe.layer_norm(gpu_ctx, x, w, b), val["y"], tol["y"], "y")
    got = apoe.layer_norm_grad(gpu_ctx, x, w, b, grad_y=gy)
    for k in got:
        close(got[k], val[k], tol[k], k)


def test_what_is_not_finite_stays_in_its_row(gpu_ctx):
    import torch
    import apoe
    g = torch.Generator().manual_seed(8)
    x = matrix(g, 40, 96, "float32")
    clean = apoe.layer_norm(gpu_ctx, x)
    x[3, 5], x[20, 0] = float("nan"), float("inf")
    y = apoe.layer_norm(gpu_ctx, x)
    rest = [i for i in range(40) if i not in (3, 20)]
    assert bool(y[3].isnan().all()) and bool(y[20].isnan().any()) and bool((y[rest] == clean[rest]).all())


def test_gradient_against_differences(gpu_ctx):
    """The slope of sum(c y) along random directions of x, w and b, from the kernel's own results: y is rounded by 2^-24 of its size, so with steps of 2^-8
    the difference's error is some 2^-15 of the sum of magnitudes, and the third derivative adds 2^-16."""
    import torch
    import apoe
    g = torch.Generator().manual_seed(9)
    n, d, h = 30, 64, 2.0 ** -8
    x, c = matrix(g, n, d, "float32"), matrix(g, n, d, "float32")
    w, b = vectors(g, d)
    grads = apoe.layer_norm_grad(gpu_ctx, x, w, b, grad_y=c)
    for name, t in (("grad_x", x), ("grad_w", w), ("grad_b", b)):
        v = torch.randn(t.shape, generator=g).cuda()
        ends = []
        for s in (h, -h):
            t.add_(v, alpha=s)
            ends.append((apoe.layer_norm(gpu_ctx, x, w, b).double() * c.double()))
            t.add_(v, alpha=-s)
        slope, size = float((ends[0] - ends[1]).sum() / (2 * h)), float(ends[0].abs().sum())
        want = float((grads[name].double() * v.double()).sum())
        assert abs(slope - want) <= 2.0 ** -13 * size, (name, slope, want, size)


def test_no_rows(gpu_ctx):
    import torch
    import apoe
    x = torch.empty(0, 100, device="cuda", dtype=torch.float16)
    w = torch.ones(100, device="cuda")
    assert apoe.layer_norm(gpu_ctx, x, w, w).shape == (0, 100)
    got = apoe.layer_norm_grad(gpu_ctx, x, w, w, grad_y=x)
    assert got["grad_x"].shape == (0, 100) and not bool(got["grad_w"].any()) and not bool(got["grad_b"].any())


def test_the_same_bits_again_and_on_another_stream(gpu_ctx):
    import torch
    import apoe
    g = torch.Generator().manual_seed(10)
    x, gy = matrix(g, 3000, 320, "bfloat16"), matrix(g, 3000, 320, "bfloat16")
    w, b = vectors(g, 320)
    once = apoe.layer_norm_grad(gpu_ctx, x, w, b, grad_y=gy)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = apoe.layer_norm_grad(gpu_ctx, x, w, b, grad_y=gy)
    torch.cuda.current_stream().wait_stream(stream)
    for k in once:
        assert bool((once[k] == again[k]).all()), k


def test_captured():
    import torch
    import apoe
    g = torch.Generator().manual_seed(11)
    x, gy = matrix(g, 700, 320, "float16"), matrix(g, 700, 320, "float16")
    w, b = vectors(g, 320)

    def call(ctx):
        return dict(apoe.layer_norm_grad(ctx, x, w, b, grad_y=gy), y=apoe.layer_norm(ctx, x, w, b))
    ctx = apoe.Context(0, stream=torch.cuda.current_stream())
    want = call(ctx)
    for got in captured(lambda s: apoe.Context(0, stream=s), call):
        for k in want:
            assert bool((got[k] == want[k]).all()), k
    ctx.close()


def test_matrices_past_four_gigabytes(gpu_ctx):
    import torch
    import apoe
    g = torch.Generator().manual_seed(12)
    n, d, gap = 5000, 200, 1 << 19
    x, gy = matrix(g, n, d, "float16"), matrix(g, n, d, "float16")
    w, b = vectors(g, d)
    store = torch.empty((n - 1) * gap + d, dtype=torch.float16, device="cuda")
    far = store.as_strided((n, d), (gap, 1))
    far.copy_(x)
    assert bool((apoe.layer_norm(gpu_ctx, far, w, b) == apoe.layer_norm(gpu_ctx, x, w, b)).all())
    near, away = (apoe.layer_norm_grad(gpu_ctx, t, w, b, grad_y=gy) for t in (x, far))
    for k in near:
        assert bool((near[k] == away[k]).all()), k
