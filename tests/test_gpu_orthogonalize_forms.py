"""The orthogonalisation with products of 22 bits on its large tiles (needs the GPU), against the same steps in 64 bits on the GPU. Tolerances as
in test_gpu_orthogonalize.py: sqrt(side) 2^-24 a product, fifteen of them: sqrt(15 * 2900) 2^-24 = 1.2e-5, within its 2e-5."""
import pytest

from test_gpu_orthogonalize import limit, matrix

pytestmark = pytest.mark.gpu


def reference(x, steps=5, coefs=(3.4445, -4.7750, 2.0315)):
    import torch
    x = x.detach().double()
    x = x / torch.linalg.matrix_norm(x)
    turned = x.shape[0] > x.shape[1]
    x = x.T.contiguous() if turned else x.contiguous()
    for _ in range(steps):
        gram = torch.mm(x, x.T.contiguous())
        x = coefs[0] * x + torch.mm(coefs[1] * gram + coefs[2] * torch.mm(gram, gram), x)
    return x.T if turned else x


def norm(t):
    import torch
    return float(torch.linalg.matrix_norm(t.double()))


# 128 x 128 tiles for all three products (one matrix, several, tall), for the last product alone, and for X X^T in two groups of waves; a
# pad of 1 takes rows that are no whole vectors
SIZES = [(1, 2900, 2900, 0), (8, 1000, 1304, 0), (8, 1290, 901, 1), (1, 2100, 2105, 3), (1, 2048, 7000, 0), (1, 7001, 2048, 1), (300, 100, 90, 0)]


@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("batch,rows,cols,pad", SIZES)
def test_products_of_22_bits_on_large_tiles(gpu_ctx, batch, rows, cols, pad, dtype):
    import apoe
    x = matrix(rows, cols, dtype, 3, batch=batch, pad=pad)
    got = apoe.orthogonalize(gpu_ctx, x)
    for i in {0, batch // 2, batch - 1}:
        want = reference(x[i])
        assert norm(got[i].double() - want) / norm(want) < limit(dtype, "f32"), i


# symmetric products on 128 x 128 tiles in two groups of waves, both of them or X X^T alone (A A of a shorter side on tiles of 64)
@pytest.mark.parametrize("products", ["f16", "f32"])
@pytest.mark.parametrize("batch,rows,cols,pad", [(14, 513, 600, 0), (5, 900, 1300, 1), (5, 1301, 897, 0), (1, 2500, 2500, 1), (25, 300, 530, 0), (25, 300, 400, 0), (4, 1024, 1024, 0)])
def test_tiles_in_two_groups(gpu_ctx, batch, rows, cols, pad, products):
    import apoe
    x = matrix(rows, cols, "float32", 6, batch=batch, pad=pad)
    got = apoe.orthogonalize(gpu_ctx, x, products=products)
    for i in {0, batch // 2, batch - 1}:
        want = reference(x[i])
        assert norm(got[i].double() - want) / norm(want) < limit("float32", products), i


@pytest.mark.parametrize("products", ["f16", "f32"])
@pytest.mark.parametrize("out", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("batch,rows,cols,pad", [(1, 2100, 2104, 0), (1, 2105, 2100, 1), (1, 900, 903, 1), (1, 300, 4100, 0)])
def test_added_into_what_is_there(gpu_ctx, batch, rows, cols, pad, out, products):
    """float32 in, every type out, both ways out of the last product, wide and tall: out = 0.5 NS(x) - out, off by the half of a result's bound
    and two roundings of what is written."""
    import torch
    import apoe
    x = matrix(rows, cols, "float32", 5, pad=pad)
    w = torch.zeros(rows, cols + pad, dtype=getattr(torch, out), device="cuda")[:, :cols]
    w.copy_(0.1 * torch.randn(rows, cols, device="cuda"))
    old, r = w.double(), reference(x)
    got = apoe.orthogonalize(gpu_ctx, x, out=w, alpha=0.5, beta=-1.0, products=products)
    want = 0.5 * r - old
    u = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8, "float32": 2.0 ** -24}[out]
    assert got is w and norm(w.double() - want) < 0.5 * limit("float32", products) * norm(r) + 2 * u * norm(want)


@pytest.mark.parametrize("products", ["f16", "f32"])
@pytest.mark.parametrize("rows,cols", [(40, 200), (100, 200), (700, 900)])
def test_coefficients_that_pass_the_products_range_give_no_number(gpu_ctx, rows, cols, products):
    """X grows past a norm of 4, or b A passes 15 off its diagonal: nothing finite comes out that could be taken for a result. Within the
    range, large coefficients are as good as others."""
    import torch
    import apoe
    g = torch.Generator().manual_seed(1)
    # one direction, half of whose entries differ in sign: A's entries are 1 / rows, or 1 / 2 between two rows that are all there is
    x = torch.zeros(rows, cols)
    x[3], x[7] = torch.ones(cols), torch.ones(cols)
    x = x.cuda()
    assert not bool(apoe.orthogonalize(gpu_ctx, x, coefs=(8.0, 0.0, 0.0), products=products).isfinite().all())
    assert not bool(apoe.orthogonalize(gpu_ctx, x, steps=1, coefs=(1.0, -40.0, 0.0), products=products).isfinite().all())
    y = (x.cpu() + 0.1 * torch.randn(rows, cols, generator=g)).cuda()
    got = apoe.orthogonalize(gpu_ctx, y, steps=1, coefs=(1.0, -28.0, 27.0), products=products)
    want = reference(y, 1, (1.0, -28.0, 27.0))
    assert norm(got.double() - want) / norm(want) < 28 * limit("float32", products)
