"""Newton-Schulz orthogonalisation against the same steps in 64 bits (needs the GPU).

Tolerances, as the 2-norm of the error over that of the result. With products of 22 bits every product is off by about sqrt(side) 2^-24
of its size and the steps raise what is off on the floor of the singular values by the floor's own factor, at most 3.4445^5 = 485: over
these inputs (floors down to 1e-2 of the top) 2e-5 holds. With fp16 products the roundings are of A and of B without its diagonal,
2^-11 each, two a step and not raised with the floor: sqrt(10) 2^-11 = 1.6e-3 where they average (sides over 64; shorter ones are
multiplied like the former), and the output's own rounding, u / sqrt(3), beside it. A result in fp32 of fp16 products is held to the
first of these two."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def reference(x, steps=5, coefs=(3.4445, -4.7750, 2.0315)):
    import torch
    x = x.detach().cpu().double()
    norm = torch.linalg.matrix_norm(x)
    x = x / norm if norm > 0 else x
    turned = x.shape[0] > x.shape[1]
    x = x.T if turned else x
    for _ in range(steps):
        A = x @ x.T
        x = coefs[0] * x + (coefs[1] * A + coefs[2] * A @ A) @ x
    return x.T if turned else x


def matrix(rows, cols, dtype, seed, floor=0.1, batch=None, pad=0):
    import torch
    g = torch.Generator().manual_seed(seed)
    shape = (batch or 1, rows, cols)
    k = min(4, rows, cols)
    x = floor * torch.randn(*shape, generator=g) + (torch.randn(shape[0], rows, k, generator=g) * torch.logspace(0, -1, k)) @ torch.randn(shape[0], k, cols, generator=g)
    x = x.to(getattr(torch, dtype))
    wide = torch.full((*shape[:2], cols + pad), float("nan"), dtype=x.dtype)
    wide[..., :cols] = x
    x = wide.cuda()[..., :cols]
    return x if batch else x[0]


def error(got, want):
    import torch
    got = got.detach().cpu().double()
    return float(torch.linalg.matrix_norm(got - want) / torch.linalg.matrix_norm(want))


def limit(dtype, products):
    return (2e-5 if products == "f32" else 10 ** 0.5 * 2.0 ** -11) + (U[dtype] / 3 ** 0.5 if dtype != "float32" else 0)


SIZES = [(1, 1), (1, 40), (40, 1), (2, 3), (16, 64), (64, 64), (65, 65), (63, 130), (130, 63), (200, 777), (777, 200), (129, 1030), (1024, 300)]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_sizes_and_types(gpu_ctx, rows, cols, dtype):
    import apoe
    for products in ("f16", "f32"):
        x = matrix(rows, cols, dtype, rows * 7 + cols, pad=3)
        got = apoe.orthogonalize(gpu_ctx, x, products=products)
        assert got.shape == x.shape and got.dtype == x.dtype
        assert error(got, reference(x)) < limit(dtype, products), (products, error(got, reference(x)))


@pytest.mark.parametrize("batch,short,long", [(1, 64, 256), (3, 64, 257), (2, 33, 300), (1, 31, 1025), (5, 17, 4095), (1, 64, 4097), (2, 9, 9001), (70, 64, 129), (1, 1, 5000)])
def test_one_short_side(gpu_ctx, batch, short, long):
    """One workgroup a matrix, several, and so many that their sums are joined first; wide and tall, summed into what is there."""
    import torch
    import apoe
    for rows, cols in ((short, long), (long, short)):
        x = matrix(rows, cols, "float32", short + long, batch=batch, pad=3)
        w = torch.randn(batch, rows, cols + 1, device="cuda")[..., :cols]
        want = w.double().cpu()
        got = apoe.orthogonalize(gpu_ctx, x, out=w, alpha=2.0, beta=-1.0)
        for i in {0, batch // 2, batch - 1}:
            r = reference(x[i])
            assert float(torch.linalg.matrix_norm(got[i].double().cpu() - (2 * r - want[i]))) < 2 * 2e-5 * float(torch.linalg.matrix_norm(r)) + 2.0 ** -23 * float(torch.linalg.matrix_norm(want[i]))
        again = apoe.orthogonalize(gpu_ctx, x, alpha=2.0)
        assert bool((again == apoe.orthogonalize(gpu_ctx, x, alpha=2.0)).all())  # sums in a fixed order


@pytest.mark.parametrize("batch,rows,cols", [(1, 100, 4100), (1, 2100, 300), (3, 65, 9000), (1, 129, 3000)])
def test_few_tiles_and_a_long_side(gpu_ctx, batch, rows, cols):
    """Products of few tiles, whose inner side is cut into parts (the last one shorter)."""
    import apoe
    x = matrix(rows, cols, "float32", 8, batch=batch, pad=1)
    for products in ("f16", "f32"):
        got = apoe.orthogonalize(gpu_ctx, x, products=products)
        for i in {0, batch - 1}:
            assert error(got[i], reference(x[i])) < limit("float32", products)


def test_tiles_of_the_large_form(gpu_ctx):
    """Sides at which 128 x 128 tiles are taken (they fill the GPU), beyond whole tiles, wide and tall, one and several."""
    import apoe
    for batch, rows, cols in ((1, 2900, 2900), (8, 1000, 1300), (8, 1290, 901), (300, 100, 90)):
        x = matrix(rows, cols, "bfloat16", 1, batch=batch)
        got = apoe.orthogonalize(gpu_ctx, x)
        for i in {0, batch - 1}:
            assert error(got[i], reference(x[i])) < limit("bfloat16", "f16")


@pytest.mark.parametrize("batch,rows,cols", [(130, 130, 136), (130, 136, 100), (129, 193, 200), (128, 200, 260), (1, 2048, 7000), (14, 300, 4100)])
def test_tiles_by_the_rounds_they_take(gpu_ctx, batch, rows, cols):
    """Batches whose symmetric products take tiles of 192 or of 256, an inner side long enough for 256 in the last product, and long rows
    on tiles of 128."""
    import apoe
    x = matrix(rows, cols, "float32", 4, batch=batch, pad=1)
    got = apoe.orthogonalize(gpu_ctx, x, products="f16")
    for i in {0, batch // 2, batch - 1}:
        assert error(got[i], reference(x[i])) < limit("float32", "f16")


def test_a_low_floor_keeps_its_directions(gpu_ctx):
    """Strong directions 250 times over the floor: an iterate in 16 bits would lose the floor in their rounding (1 % and more)."""
    import apoe
    x = matrix(512, 700, "float32", 5, floor=0.02)
    assert error(apoe.orthogonalize(gpu_ctx, x, products="f16"), reference(x)) < limit("float32", "f16")
    assert error(apoe.orthogonalize(gpu_ctx, x), reference(x)) < 2e-5 * 5  # floor 1 / 250: five times below the others


def test_singular_values_come_near_one(gpu_ctx):
    import torch
    import apoe
    x = matrix(96, 256, "float32", 2)
    s = torch.linalg.svdvals(apoe.orthogonalize(gpu_ctx, x).double().cpu())
    assert 0.6 < float(s.min()) and float(s.max()) < 1.3
    # the cubic step a = 1.5, b = -0.5 converges to the polar factor
    s = torch.linalg.svdvals(apoe.orthogonalize(gpu_ctx, x, steps=40, coefs=(1.5, -0.5, 0.0)).double().cpu())
    assert float((s - 1).abs().max()) < 1e-4


@pytest.mark.parametrize("rows,cols", [(70, 140), (140, 70)])
def test_batches_strides_scale_and_sum(gpu_ctx, rows, cols):
    import torch
    import apoe
    x = matrix(rows, cols, "bfloat16", 3, batch=3, pad=5)
    w = torch.randn(3, rows, cols, device="cuda")
    want = [0.75 * w[i].double().cpu() - 0.02 * reference(x[i]) for i in range(3)]
    out = apoe.orthogonalize(gpu_ctx, x, out=w, alpha=-0.02, beta=0.75)
    assert out is w
    for i in range(3):
        # the matrix's own part is off by limit() of 0.02, the sum by a rounding or two of fp32
        assert float((w[i].double().cpu() - want[i]).abs().max()) < 0.02 * limit("float32", "f16") + 4 * 2.0 ** -24 * 5
    # each one as if alone, in any order of strides between matrices
    alone = [apoe.orthogonalize(gpu_ctx, x[i]) for i in range(3)]
    both = apoe.orthogonalize(gpu_ctx, x[::2])
    for k, i in enumerate((0, 2)):
        assert bool((both[k] == alone[i]).all())
    # in place
    y = x.clone()
    assert bool((apoe.orthogonalize(gpu_ctx, y, out=y)[1] == alone[1]).all())


def test_zero_tiny_huge_and_not_finite(gpu_ctx):
    import torch
    import apoe
    assert not bool(apoe.orthogonalize(gpu_ctx, torch.zeros(50, 70, device="cuda")).any())
    x = matrix(50, 70, "float32", 4)
    want = reference(x)
    for factor in (1e-30, 1e30):  # squares beyond fp32
        assert error(apoe.orthogonalize(gpu_ctx, x * factor), reference(x * factor)) < 2e-5
    assert error(apoe.orthogonalize(gpu_ctx, x * 2.0 ** 20), want) < 2e-5
    x[3, 4] = float("nan")
    assert bool(apoe.orthogonalize(gpu_ctx, x).isnan().all())
    both = torch.stack([x, matrix(50, 70, "float32", 4)])
    assert error(apoe.orthogonalize(gpu_ctx, both)[1], want) < 2e-5  # a neighbour's NaN stays its own


def test_same_bits_every_time_and_symmetric_in_the_side(gpu_ctx):
    import apoe
    x = matrix(300, 500, "bfloat16", 6)
    first = apoe.orthogonalize(gpu_ctx, x)
    for _ in range(3):
        assert bool((apoe.orthogonalize(gpu_ctx, x) == first).all())
    assert bool((apoe.orthogonalize(gpu_ctx, x.T.contiguous()) == first.T).all())


def test_in_a_graph():
    import torch
    import apoe
    stream = torch.cuda.Stream()
    ctx = apoe.Context(0, stream=stream)
    xs = [matrix(100, 230, "bfloat16", s) for s in (1, 2, 3)]
    held, out = xs[0].clone(), torch.empty_like(xs[0])
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        apoe.orthogonalize(ctx, held, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        apoe.orthogonalize(ctx, held, out=out)
    for _ in range(2):
        for x in xs:
            want = apoe.orthogonalize(ctx, x)
            torch.cuda.synchronize()
            held.copy_(x)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert bool((out == want).all())
    ctx.close()


def test_refusals(gpu_ctx):
    import ctypes as C
    import torch
    import apoe
    x = matrix(8, 9, "float32", 1)
    for call, words in ((lambda: apoe.orthogonalize(gpu_ctx, x[0]), "matrix"), (lambda: apoe.orthogonalize(gpu_ctx, x.double()), "float32"),
                        (lambda: apoe.orthogonalize(gpu_ctx, x.cpu()), "on GPU"), (lambda: apoe.orthogonalize(gpu_ctx, x, steps=0), "steps"),
                        (lambda: apoe.orthogonalize(gpu_ctx, x, steps=65), "steps"), (lambda: apoe.orthogonalize(gpu_ctx, x, beta=1.0), "beta without out"),
                        (lambda: apoe.orthogonalize(gpu_ctx, x, out=x.T.contiguous()), "out must be"), (lambda: apoe.orthogonalize(gpu_ctx, x, products="f8"), "products"),
                        (lambda: apoe.orthogonalize(gpu_ctx, x, coefs=(1.0, float("inf"), 0.0)), "finite"), (lambda: apoe.orthogonalize(gpu_ctx, x.T), "contiguous"),
                        (lambda: apoe.orthogonalize(gpu_ctx, x, out=torch.empty(1, 9, device="cuda").expand(8, 9)), "overlap")):
        with pytest.raises(apoe.ApoeError, match=words):
            call()
    assert apoe.orthogonalize(gpu_ctx, x[:0]).shape == (0, 9)
    lib = apoe.lib()
    assert lib.apoe_orthogonalize(gpu_ctx.h, None) == -1
    a = apoe.OrthogonalizeArgs()
    a.batch, a.rows, a.cols, a.steps, a.products = 1, 4, 4, 5, 1
    assert lib.apoe_orthogonalize(gpu_ctx.h, C.byref(a)) == -1 and b"null" in lib.apoe_last_error_string()
    a.in_ = a.out = x.data_ptr()
    for field, value, word in (("in_dtype", 3, b"dtype"), ("products", 2, b"products"), ("rows", 70000, b"side"), ("batch", 70000, b"batch"), ("in_stride", 3, b"overlap")):
        b = apoe.OrthogonalizeArgs.from_buffer_copy(a)
        setattr(b, field, value)
        assert lib.apoe_orthogonalize(gpu_ctx.h, C.byref(b)) == -1 and word in lib.apoe_last_error_string(), field
    host = np.zeros(16, np.float32)
    a.out = host.ctypes.data
    assert lib.apoe_orthogonalize(gpu_ctx.h, C.byref(a)) == -1 and b"device memory" in lib.apoe_last_error_string()
