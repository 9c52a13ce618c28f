"""How many bits of gz = grad_y act'(pre) the products of linear's gradient keep for 16-bit matrices (needs the GPU).

Each result is the sum in 32 bits, rounded once: off by half a step of its own size, and by what the sum is off. gz is formed in 32 bits, off by
(12 + p p) 2^-24 of the slope's terms, and goes in as two parts: a rounding of a rounding, u u of its size, where a step of the small numbers is below 2^-34.
A sum of K products is off by at most (2 K + 8) 2^-23 of its terms' magnitudes (both parts of each are added, each addition off by a step at most)."""
import pytest

from layer_cases import E, SMALL, U, matrix
from test_gpu_linear import slope_of

pytestmark = pytest.mark.gpu


def half_step(v, dtype):
    import torch
    exponent = torch.frexp(v.abs())[1] - 1  # of numbers from 1 to 2
    lowest = -14 if dtype == "float16" else -126
    return U[dtype] * torch.ldexp(torch.ones_like(v), exponent.clamp(min=lowest))


def check(ctx, m, n, k, dtype, act, seed=0, size=1.0):
    import torch
    import apoe
    g = torch.Generator().manual_seed(seed)
    x, w, gy, pre = matrix(g, m, k, dtype), matrix(g, n, k, dtype), matrix(g, m, n, dtype, size), matrix(g, m, n, dtype, 2.0)
    got = apoe.linear_grad(ctx, x, w, gy, act=act, pre=pre, grad_bias=False)
    p, gy = pre.double(), gy.double()
    slope = slope_of(p, act)
    gz = gy * slope
    terms = slope.abs() + (p * torch.exp(-0.5 * p * p)).abs() + (p * torch.sigmoid(p) * torch.sigmoid(-p)).abs()
    off = gy.abs() * (12 + p * p) * E * terms + U[dtype] ** 2 * gz.abs() + 2.0 ** -34 * (dtype == "float16") + E * gz.abs()
    if act in ("none", "relu"):
        off = torch.zeros_like(gz)
    for name, a, off_a, b in (("grad_x", gz, off, w.double()), ("grad_w", gz.t().contiguous(), off.t().contiguous(), x.double())):
        want = torch.mm(a, b)
        tol = torch.mm(off_a, b.abs()) + (2 * a.shape[1] + 8) * 2.0 ** -23 * torch.mm(a.abs(), b.abs())
        err = (got[name].double() - want).abs()
        bad = ~(err <= half_step(want.abs() + tol, dtype) + tol + SMALL[dtype] / 2)
        assert not bool(bad.any()), (name, m, n, k, int(bad.sum()), bad.numel())


@pytest.mark.parametrize("act", ["relu", "gelu", "silu"])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("m,n,k", [(1, 1, 300), (65, 1, 40), (1, 65, 72), (130, 70, 264), (500, 333, 129)])
def test_results_are_rounded_once(gpu_ctx, m, n, k, dtype, act):
    check(gpu_ctx, m, n, k, dtype, act, m + n)


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("size", [1e-6, 3e4])
def test_small_and_large_gradients_in_float16(gpu_ctx, size, act):
    """grad_y where float16's own steps are coarse, and up to 65 504, where gz may be above that."""
    check(gpu_ctx, 70, 40, 96, "float16", act, 5, size if size < 1 else 1e3)
    import torch
    import apoe
    gy = torch.full((4, 8), 65504.0 if size > 1 else 2.0 ** -24, dtype=torch.float16, device="cuda")
    pre = torch.full((4, 8), 1.5 if act == "gelu" else 2.5, dtype=torch.float16, device="cuda")  # a slope of 1.12, 1.10
    w, x = 2.0 ** -9 * torch.eye(8, dtype=torch.float16, device="cuda"), torch.ones(4, 8, dtype=torch.float16, device="cuda")
    if size < 1:
        w *= 2.0 ** 20
    got = apoe.linear_grad(gpu_ctx, x, w, gy, act=act, pre=pre, grad_w=False, grad_bias=False)["grad_x"].double()
    want = gy.double() * slope_of(pre.double(), act) * w[0, 0].double()
    assert bool(((got - want).abs() <= half_step(want * 1.001, "float16") * 1.01).all()), (got[0, 0], want[0, 0])


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_infinite_operands_beside_two_parts(gpu_ctx, dtype):
    """An infinity in x, w or grad_y gives what the sum is: an infinity of gz's sign, NaN where it meets a zero or one of the other sign."""
    import torch
    import apoe
    g = torch.Generator().manual_seed(3)
    x, w, gy, pre = matrix(g, 70, 40, dtype), matrix(g, 24, 40, dtype), matrix(g, 70, 24, dtype), matrix(g, 70, 24, dtype)
    gy[1, 3], gy[2, 3], gy[5, 7] = 0.5, 0.0, float("inf")
    pre[1, 3] = pre[2, 3] = pre[5, 7] = 1.0
    w[3, 9] = float("inf")
    x[60, 4] = float("-inf")
    got = apoe.linear_grad(gpu_ctx, x, w, gy, act="gelu", pre=pre)
    gz = gy.double() * slope_of(pre.double(), "gelu")
    for name, a, b in (("grad_x", gz, w.double()), ("grad_w", gz.t().contiguous(), x.double())):
        a, b = a.cpu(), b.cpu()
        want = (a[:, :, None] * b[None]).sum(1)
        have = got[name].cpu().double()
        odd = ~torch.isfinite(want)
        assert int(odd.sum()) > 40 and bool((torch.isfinite(have) == ~odd).all()), name
        assert bool((have.isnan() == want.isnan()).all()) and bool((have[odd & ~want.isnan()] == want[odd & ~want.isnan()]).all()), name


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("m,n,k", [(150, 96, 80), (1489, 1477, 299), (60, 72, 5000)])
def test_parts_of_the_gradient(gpu_ctx, m, n, k, dtype):
    """Each gradient by itself has the bits that it has with the others."""
    import torch
    import apoe
    g = torch.Generator().manual_seed(6)
    x, w, gy, pre = matrix(g, m, k, dtype), matrix(g, n, k, dtype), matrix(g, m, n, dtype), matrix(g, m, n, dtype)
    whole = apoe.linear_grad(gpu_ctx, x, w, gy, act="silu", pre=pre)
    for name in whole:
        part = apoe.linear_grad(gpu_ctx, x, w, gy, act="silu", pre=pre, **{key: key == name for key in whole})
        assert set(part) == {name} and bool((part[name] == whole[name]).all())
