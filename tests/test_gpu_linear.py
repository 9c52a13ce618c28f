"""A linear layer with bias, activation and residual, and its gradients, against 64 bits (needs the GPU).

Tolerances. A sum of K products: 16-bit values multiply exactly, the float32 sum is off by at most (K + 4) 2^-23 of the sum of magnitudes in any order and
with any way of the matrix units to add (each addition off by a whole step at most). float32 matrices go in as three parts of 8 bits, and the products of the
smaller parts that are left out are at most 2^-22 of each product. pre and y are rounded once (half a step); the activation passes on what z is off by times
1.13, its steepest slope, and is off by (8 + z z) 2^-24 of its own terms (the exponent's rounding). gz of 16-bit matrices with an activation is
rounded before it is multiplied: half a step of each of its values (in the sum of magnitudes). The bias' gradient adds up rows in float32."""
import math

import pytest

from layer_cases import E, SMALL, TYPES, U, captured, close, matrix, room

pytestmark = pytest.mark.gpu
ACTS = ["none", "relu", "gelu", "silu"]


def phi(z):
    import torch
    return 0.5 * torch.erfc(-z / math.sqrt(2.0))


def act_of(z, act):
    import torch
    return {"none": lambda: z, "relu": lambda: torch.where(z > 0, z, torch.zeros_like(z)), "gelu": lambda: z * phi(z), "silu": lambda: z * torch.sigmoid(z)}[act]()


def slope_of(z, act):
    import torch
    if act == "gelu":
        return phi(z) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(z)
    return {"none": lambda: torch.ones_like(z), "relu": lambda: (z > 0).double(), "silu": lambda: s * (1 + z * (1 - s))}[act]()


def product(a, b, dtype):
    """a b^T and what the kernel's may be off by, before any rounding of it."""
    import torch
    size = torch.mm(a.abs(), b.abs().t().contiguous())
    return torch.mm(a, b.t().contiguous()), size * ((a.shape[1] + 4) * 2.0 ** -23 + (2.0 ** -22 if dtype == "float32" else 0))


def formula(x, w, bias, act, residual, dtype, grad_y=None, pre=None):
    import torch
    u, small = U[dtype], SMALL[dtype]
    x, w = x.double(), w.double()
    z, off = product(x, w, dtype)
    if bias is not None:
        z = z + bias.double()
    off = off + E * z.abs()
    a = act_of(z, act)
    y = a + (residual.double() if residual is not None else 0)
    val = dict(pre=z, y=y)
    own = 0 if act in ("none", "relu") else (8 + z * z).clamp(max=2.0 ** 20) * E * (a.abs() + (z.abs() * E))
    tol = dict(pre=off + u * z.abs() + small, y=1.13 * off + own + (u + E) * y.abs() + E * a.abs() + small)
    if grad_y is not None:
        gz = grad_y.double()
        loose = torch.zeros_like(gz)
        if act != "none":
            p = pre.double()
            s = slope_of(p, act)
            loose = gz.abs() * (8 + p * p).clamp(max=2.0 ** 20) * E * (s.abs() + (p * torch.exp(-0.5 * p * p)).abs() + 2 * E) if act != "relu" else loose
            gz = gz * s
        rounded = loose + (u * gz.abs() + small if act != "none" and dtype != "float32" else 2 * E * gz.abs())
        for name, a, b, off_a in (("grad_x", gz, w.t().contiguous(), rounded), ("grad_w", gz.t().contiguous(), x.t().contiguous(), rounded.t().contiguous())):
            val[name], off = product(a, b, dtype)
            tol[name] = off * 1.02 + torch.mm(off_a, b.abs().t().contiguous()) + u * val[name].abs() + small
        val["grad_bias"] = gz.sum(0)
        tol["grad_bias"] = (loose + 2 * E * gz.abs()).sum(0) + (gz.shape[0] / 4 + 80) * E * gz.abs().sum(0) + small
    return val, tol


def check(ctx, m, n, k, dtype, act, seed, pad=0, shift=0, bias=True, residual=True, grad=True, out_pad=8):
    import torch
    import apoe
    g = torch.Generator().manual_seed(seed)
    x, w = matrix(g, m, k, dtype, 1.0, pad, shift), matrix(g, n, k, dtype, 1.5 / math.sqrt(k), pad, shift)
    b = torch.randn(n, generator=g).cuda() if bias else None
    r = matrix(g, m, n, dtype, 1.0, pad, shift) if residual else None
    gy = matrix(g, m, n, dtype, 1.0, pad, shift)
    out, outside = room(m, n, dtype, out_pad)
    y, pre = apoe.linear(ctx, x, w, b, act=act, residual=r, want_pre=True, out=out)
    assert y is out
    plain, none = apoe.linear(ctx, x, w, b, act=act, residual=r)
    assert none is None and bool((plain == y).all())
    got = dict(y=y, pre=pre)
    val, tol = formula(x, w, b, act, r, dtype, gy if grad else None, pre)
    if grad:
        gx, outside_x = room(m, k, dtype, out_pad)
        gw, outside_w = room(n, k, dtype, out_pad)
        got.update(apoe.linear_grad(ctx, x, w, gy, act=act, pre=pre if act != "none" else None, grad_x=gx, grad_w=gw))
        assert got["grad_x"] is gx and got["grad_w"] is gw and outside_x() and outside_w()
    assert set(got) == set(val) and outside()
    for name in val:
        close(got[name], val[name], tol[name], (name, m, n, k))


SIZES = [(1, 1, 1), (1, 64, 64), (2, 3, 5), (5, 1000, 8), (16, 64, 128), (17, 40, 1000), (33, 129, 257), (64, 96, 2048), (65, 24, 72), (100, 1, 300), (1, 300, 1), (130, 264, 520), (70, 72, 8200), (300, 130, 64)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_sizes_and_types(gpu_ctx, m, n, k, dtype):
    for i, (pad, shift, out_pad) in enumerate(((0, 0, 8), (8, 0, 3), (5, 3, 1))):
        check(gpu_ctx, m, n, k, dtype, ACTS[(m + i) % 4], m + n + k + i, pad, shift, bias=i != 1, residual=i != 2, out_pad=out_pad)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 17, 4096), (16, 4100, 1032), (4, 33, 264), (16, 64, 4096), (17, 64, 4096), (3, 20, 8192)])
def test_few_rows(gpu_ctx, m, n, k, dtype):
    for act in ("none", "gelu"):
        check(gpu_ctx, m, n, k, dtype, act, m + k, pad=8, grad=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
def test_activations(gpu_ctx, act, dtype):
    check(gpu_ctx, 200, 136, 96, dtype, act, 1)
    check(gpu_ctx, 20, 136, 96, dtype, act, 2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(3700, 3701, 40), (1900, 1912, 72), (4100, 200, 264), (200, 4100, 264), (72, 104, 20_000), (20_000, 40, 72), (640, 5000, 640)])
def test_each_tile_and_cut(gpu_ctx, m, n, k, dtype):
    """Sizes that fill the GPU with the largest tiles, with middle ones, and such that have their inner side cut (one of the three products has it long)."""
    check(gpu_ctx, m, n, k, dtype, "silu", 3)


@pytest.mark.parametrize("dtype", TYPES)
def test_activation_value_by_value(gpu_ctx, dtype):
    """z itself goes through (w is the identity): every activation from far below zero to far above, its tails relative to themselves."""
    import torch
    import apoe
    z = torch.cat((torch.linspace(-14, 14, 4001), torch.tensor([0.0, -0.0, 1e-6, -1e-6, 30.0, -30.0, 100.0, -100.0]))).to(getattr(torch, dtype))
    z = torch.cat((z, torch.zeros(-len(z) % 8, dtype=z.dtype))).view(-1, 8).cuda()
    eye = torch.eye(8, dtype=z.dtype, device="cuda")
    ones = torch.ones_like(z)
    d = z.double()
    for act in ("relu", "gelu", "silu"):
        y, pre = apoe.linear(gpu_ctx, z, eye, act=act, want_pre=True)
        assert bool((pre == z).all())
        want = act_of(d, act)
        close(y, want, U[dtype] * want.abs() + (12 + d * d) * E * want.abs() + SMALL[dtype] + 2.0 ** -126, act)
        gx = apoe.linear_grad(gpu_ctx, z, eye, ones, act=act, pre=pre, grad_w=False, grad_bias=False)["grad_x"]
        want = slope_of(d, act)
        terms = want.abs() + (d * torch.exp(-0.5 * d * d)).abs() + (d * torch.sigmoid(d) * torch.sigmoid(-d)).abs()
        close(gx, want, U[dtype] * want.abs() + (12 + d * d) * E * terms + SMALL[dtype] + 2.0 ** -126, act)


def test_values_of_any_size_in_float32(gpu_ctx):
    """Parts of a float32 value have its exponent: rows and columns from 1e-18 to 1e18 in one matrix, the largest float among them, each result within
    its own terms' rounding."""
    import torch
    import apoe
    g = torch.Generator().manual_seed(4)
    m, n, k = 90, 70, 200
    x = (torch.randn(m, k, generator=g) * 10 ** (36 * torch.rand(m, k, generator=g) - 18)).cuda()
    w = (torch.randn(n, k, generator=g) * 10 ** (36 * torch.rand(n, k, generator=g) - 18)).cuda()
    val, tol = formula(x, w, None, "none", None, "float32")
    close(apoe.linear(gpu_ctx, x, w)[0], val["y"], tol["y"])
    x = torch.zeros(3, 8, device="cuda")
    x[0, 0], x[1, 1], x[2, 2] = torch.finfo(torch.float32).max, -3.4e38, 1e-38
    got = apoe.linear(gpu_ctx, x, torch.eye(8, device="cuda"))[0]
    close(got, x.double(), 2.0 ** -22 * x.double().abs() + 2.0 ** -133)


def test_what_is_not_finite_stays_in_its_row_and_column(gpu_ctx):
    import torch
    import apoe
    for dtype in TYPES:
        g = torch.Generator().manual_seed(5)
        x, w = matrix(g, 100, 64, dtype), matrix(g, 80, 64, dtype)
        clean = apoe.linear(gpu_ctx, x, w)[0]
        x[7, 3], w[11, 60] = float("nan"), float("inf")
        y = apoe.linear(gpu_ctx, x, w)[0]
        rows, cols = [i for i in range(100) if i != 7], [j for j in range(80) if j != 11]
        assert bool(y[7].isnan().all()) and not bool(torch.isfinite(y[:, 11]).any())
        assert bool((y[rows][:, cols] == clean[rows][:, cols]).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_parts_of_the_gradient(gpu_ctx, dtype):
    import torch
    import apoe
    g = torch.Generator().manual_seed(6)
    x, w, gy = matrix(g, 150, 80, dtype), matrix(g, 96, 80, dtype), matrix(g, 150, 96, dtype)
    whole = apoe.linear_grad(gpu_ctx, x, w, gy)
    for name in whole:
        part = apoe.linear_grad(gpu_ctx, x, w, gy, **{k: k == name for k in whole})
        assert set(part) == {name} and bool((part[name] == whole[name]).all())


def test_gradients_against_differences(gpu_ctx):
    """The slope of sum(c y) along random directions, from the kernel's own results in float32: steps of 2^-7, the rounding of y (2^-20 of the sum of
    magnitudes at K = 40) over twice that, and the third derivative's 2^-15."""
    import torch
    import apoe
    g = torch.Generator().manual_seed(7)
    x, w, c = matrix(g, 50, 40, "float32"), matrix(g, 30, 40, "float32", 0.16), matrix(g, 50, 30, "float32")
    b, h = torch.randn(30, generator=g).cuda(), 2.0 ** -7
    for act in ("none", "gelu", "silu"):
        pre = apoe.linear(gpu_ctx, x, w, b, act=act, want_pre=True)[1]
        grads = apoe.linear_grad(gpu_ctx, x, w, c, act=act, pre=pre)
        for name, t in (("grad_x", x), ("grad_w", w), ("grad_bias", b)):
            v = torch.randn(t.shape, generator=g).cuda()
            ends = []
            for s in (h, -h):
                t.add_(v, alpha=s)
                ends.append(apoe.linear(gpu_ctx, x, w, b, act=act)[0].double() * c.double())
                t.add_(v, alpha=-s)
            slope, size = float((ends[0] - ends[1]).sum() / (2 * h)), float(ends[0].abs().sum())
            want = float((grads[name].double() * v.double()).sum())
            reach = float(v.abs().max()) ** 3 * 40 ** 0.5
            assert abs(slope - want) <= (2.0 ** -12 + 2.0 ** -15 * reach) * size, (act, name, slope, want, size)


def test_no_rows(gpu_ctx):
    import torch
    import apoe
    x, w = torch.empty(0, 40, device="cuda", dtype=torch.bfloat16), torch.ones(24, 40, device="cuda", dtype=torch.bfloat16)
    y, pre = apoe.linear(gpu_ctx, x, w, act="gelu", want_pre=True)
    assert y.shape == pre.shape == (0, 24)
    got = apoe.linear_grad(gpu_ctx, x, w, y, act="gelu", pre=pre)
    assert got["grad_x"].shape == (0, 40) and not bool(got["grad_w"].any()) and not bool(got["grad_bias"].any())


def test_no_rows_from_c(gpu_ctx):
    """Through the C-ABI: the weight's and the bias' gradients of no rows are zeros."""
    import ctypes as C
    import torch
    import apoe
    for dtype, code in ((torch.float16, 1), (torch.float32, 0)):
        gw, gb = torch.full((24, 40), 7.0, dtype=dtype, device="cuda"), torch.full((24,), 7.0, device="cuda")
        a = apoe.LinearArgs()
        a.dtype, a.rows, a.cols_in, a.cols_out, a.grad_w, a.grad_bias = code, 0, 40, 24, gw.data_ptr(), gb.data_ptr()
        torch.cuda.synchronize()
        assert apoe.lib().apoe_linear_grad(gpu_ctx.h, C.byref(a)) == 0
        gpu_ctx.synchronize()
        assert not bool(gw.any()) and not bool(gb.any())


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_the_same_bits_again_and_on_another_stream(gpu_ctx, dtype):
    import torch
    import apoe
    g = torch.Generator().manual_seed(8)
    x, w, gy = matrix(g, 1000, 264, dtype), matrix(g, 200, 264, dtype), matrix(g, 1000, 200, dtype)

    def call():
        y, pre = apoe.linear(gpu_ctx, x, w, act="gelu", want_pre=True)
        return dict(apoe.linear_grad(gpu_ctx, x, w, gy, act="gelu", pre=pre), y=y)
    once = call()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = call()
    torch.cuda.current_stream().wait_stream(stream)
    for k in once:
        assert bool((once[k] == again[k]).all()), k


@pytest.mark.parametrize("m", [3, 500])
@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_captured(dtype, m):
    import torch
    import apoe
    g = torch.Generator().manual_seed(9)
    x, w, gy = matrix(g, m, 136, dtype), matrix(g, 72, 136, dtype), matrix(g, m, 72, dtype)

    def call(ctx):
        y, pre = apoe.linear(ctx, x, w, act="silu", want_pre=True)
        return dict(apoe.linear_grad(ctx, x, w, gy, act="silu", pre=pre), y=y)
    ctx = apoe.Context(0, stream=torch.cuda.current_stream())
    want = call(ctx)
    for got in captured(lambda s: apoe.Context(0, stream=s), call):
        for k in want:
            assert bool((got[k] == want[k]).all()), k
    ctx.close()


def test_a_captured_graph_survives_a_workspace_that_grows():
    """The graph's calls keep the workspace that they were captured with; a larger eager call takes another one, and a capture that would have to grow it
    is refused."""
    import torch
    import apoe
    g = torch.Generator().manual_seed(10)
    x, w = matrix(g, 100, 77, "float16"), matrix(g, 40, 77, "float16")
    big = matrix(g, 3000, 1001, "float16")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    ctx = apoe.Context(0, stream=stream)
    with torch.cuda.stream(stream):
        want = apoe.linear(ctx, x, w)[0].clone()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        y = apoe.linear(ctx, x, w)[0]
        with pytest.raises(apoe.ApoeError, match="capture"):
            apoe.linear(ctx, big, big[:500])
    for _ in range(3):
        with torch.cuda.stream(stream):
            y.zero_()
            apoe.linear(ctx, big, big[:500])
            graph.replay()
        stream.synchronize()
        assert bool((y == want).all())
    del graph
    ctx.close()


def test_strides_past_four_gigabytes(gpu_ctx):
    import torch
    import apoe
    g = torch.Generator().manual_seed(11)
    for gap in ((1 << 21), (1 << 26)):  # read where it lies; taken apart first
        store = torch.empty(((40 if gap > 1 << 21 else 1200) - 1) * gap + 64, dtype=torch.float16, device="cuda")
        m = 40 if gap > 1 << 21 else 1200
        x = store.as_strided((m, 64), (gap, 1))
        near = matrix(g, m, 64, "float16")
        x.copy_(near)
        w, gy = matrix(g, 48, 64, "float16"), matrix(g, m, 48, "float16")
        assert bool((apoe.linear(gpu_ctx, x, w)[0] == apoe.linear(gpu_ctx, near, w)[0]).all())
        a, b = (apoe.linear_grad(gpu_ctx, t, w, gy) for t in (x, near))
        for k in a:
            assert bool((a[k] == b[k]).all()), k
        del store, x


@pytest.mark.parametrize("dtype", TYPES)
def test_relu_lets_nothing_back_where_nothing_went_out(gpu_ctx, dtype):
    """An infinity or a NaN in grad_y where pre is zero or below leaves all gradients as a zero there does."""
    import torch
    import apoe
    g = torch.Generator().manual_seed(12)
    x, w, gy = matrix(g, 70, 40, dtype), matrix(g, 24, 40, dtype), matrix(g, 70, 24, dtype)
    pre = apoe.linear(gpu_ctx, x, w, act="relu", want_pre=True)[1]
    pre[3, 5], pre[40, 23], pre[69, 0] = -1.0, 0.0, -0.0
    gy[3, 5] = gy[40, 23] = gy[69, 0] = 0.0
    want = apoe.linear_grad(gpu_ctx, x, w, gy, act="relu", pre=pre)
    gy[3, 5], gy[40, 23], gy[69, 0] = float("inf"), float("nan"), float("-inf")
    got = apoe.linear_grad(gpu_ctx, x, w, gy, act="relu", pre=pre)
    for k in want:
        assert bool(torch.isfinite(want[k]).all()) and bool((got[k] == want[k]).all()), k


def test_small_values_with_large_ones_in_float32(gpu_ctx):
    """Values from 2^-126 to 2^-100 times values around 2^110: the parts of small ones end at 2^-133, which each is off by at most."""
    import torch
    import apoe
    g = torch.Generator().manual_seed(13)
    m, n, k = 90, 70, 200
    x = (torch.randn(m, k, generator=g).sign() * 2 ** (26 * torch.rand(m, k, generator=g, dtype=torch.float64) - 126)).float().cuda()
    w = (torch.randn(n, k, generator=g) * 2.0 ** 110).cuda()
    val, tol = formula(x, w, None, "none", None, "float32")
    close(apoe.linear(gpu_ctx, x, w)[0], val["y"], tol["y"] + 2.0 ** -133 * w.double().abs().sum(1)[None, :])
