"""What linear and its gradient answer at the edges of their numbers (needs the GPU)."""
import pytest

from layer_cases import TYPES, matrix

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
def test_relu_lets_nothing_back_where_pre_is_nan(gpu_ctx, dtype):
    """A NaN in pre is not above zero: whatever grad_y is there, all gradients are as if it were zero."""
    import torch
    import apoe
    g = torch.Generator().manual_seed(1)
    x, w, gy, pre = matrix(g, 70, 40, dtype), matrix(g, 24, 40, dtype), matrix(g, 70, 24, dtype), matrix(g, 70, 24, dtype)
    pre[3, 5] = pre[40, 23] = pre[69, 0] = float("nan")
    gy[3, 5] = gy[40, 23] = gy[69, 0] = 0.0
    want = apoe.linear_grad(gpu_ctx, x, w, gy, act="relu", pre=pre)
    gy[3, 5], gy[40, 23], gy[69, 0] = 1.0, float("nan"), float("-inf")
    got = apoe.linear_grad(gpu_ctx, x, w, gy, act="relu", pre=pre)
    for k in want:
        assert bool(torch.isfinite(want[k]).all()) and bool((got[k] == want[k]).all()), k


def sums(a, b):
    """a b^T in 64 bits, as 32 bits hold it: an infinity where a sum is beyond them, NaN where infinities meet zeros or each other."""
    import torch
    return torch.stack([(a.double()[i] * b.double()).sum(1) for i in range(a.shape[0])]).float()


def same_kind(got, want):
    import torch
    assert bool((got.isnan() == want.isnan()).all()), (int(got.isnan().sum()), int(want.isnan().sum()))
    odd = torch.isinf(want)
    assert bool((torch.isinf(got) == odd).all()) and bool((got[odd] == want[odd]).all())
    return int(odd.sum()), int(want.isnan().sum())


SHAPES = [(5, 24, 40), (17, 24, 40), (100, 70, 64), (300, 130, 264), (30, 40, 9000), (1500, 900, 72)]  # few rows, small tiles, cuts, larger tiles


@pytest.mark.parametrize("pad,shift", [(0, 0), (3, 1)])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_float_products_beyond_the_largest_number(gpu_ctx, m, n, k, pad, shift):
    """Finite values whose products or sums overflow give infinities, however many rows a call has."""
    import torch
    import apoe
    g = torch.Generator().manual_seed(m)
    x, w, gy = matrix(g, m, k, "float32", 1.0, pad, shift), matrix(g, n, k, "float32", 1.0, pad, shift), matrix(g, m, n, "float32", 1.0, pad, shift)
    for t, rows in ((x, (1, m - 1)), (w, (0, n // 2)), (gy, (2, m // 2))):
        t.abs_().add_(0.5)
        for r in rows:
            t[r] *= 1e30
    y = apoe.linear(gpu_ctx, x, w)[0]
    got = apoe.linear_grad(gpu_ctx, x, w, gy)
    want = sums(x, w)
    assert same_kind(y, want) == (4, 0)
    same_kind(got["grad_x"], sums(gy, w.t().contiguous()))
    same_kind(got["grad_w"], sums(gy.t().contiguous(), x.t().contiguous()))
    clean = torch.isfinite(y)
    assert bool(((y - want)[clean].abs() <= 2.0 ** -20 * want[clean].abs() + (k + 4) * 2.0 ** -23 * want[clean].abs()).all())


@pytest.mark.parametrize("pad,shift", [(0, 0), (3, 1)])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_infinite_floats(gpu_ctx, m, n, k, pad, shift):
    """An infinity times numbers is an infinity, times a zero or beside one of the other sign NaN: the same whatever kernel the sizes choose."""
    import torch
    import apoe
    g = torch.Generator().manual_seed(m + 1)
    x, w, gy = matrix(g, m, k, "float32", 1.0, pad, shift), matrix(g, n, k, "float32", 1.0, pad, shift), matrix(g, m, n, "float32", 1.0, pad, shift)
    inf = float("inf")
    x[1, 3], x[3, 0], x[3, k - 1], w[5, 7], w[6, 3], gy[4, 2], gy[0, n - 1] = inf, inf, -inf, -inf, 0.0, inf, float("nan")
    y = apoe.linear(gpu_ctx, x, w)[0]
    got = apoe.linear_grad(gpu_ctx, x, w, gy)
    infinite, nans = same_kind(y, sums(x, w))
    assert infinite >= m and nans >= 2
    same_kind(got["grad_x"], sums(gy, w.t().contiguous()))
    same_kind(got["grad_w"], sums(gy.t().contiguous(), x.t().contiguous()))
