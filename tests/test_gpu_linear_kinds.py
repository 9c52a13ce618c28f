"""Every kernel that linear's sizes choose (kinds of tiles, whole and with the inner side cut, grad_x and grad_w in one launch and in two, in one and two parts), against 64
bits, with edges that are no multiple of anything (needs the GPU). test_linear_rule.py holds that these sizes reach them. Tolerances: those of test_gpu_linear.py."""
import math

import pytest

from layer_cases import matrix, room
from test_gpu_linear import formula

pytestmark = pytest.mark.gpu

SIZES = {
    16: [(47, 41, 47), (391, 417, 4746), (1289, 1375, 42), (329, 5452, 372), (1541, 337, 1386), (1489, 1477, 2699), (3434, 221, 1811), (255, 1929, 3143), (1040, 1084, 6558),
         (1448, 1473, 5962), (1933, 3154, 339), (6554, 646, 1560), (334, 3790, 2726), (2195, 4819, 997), (4206, 2033, 1078), (2324, 2277, 914), (626, 2305, 3303), (1957, 2642, 1544),
         (4896, 85, 1219), (4781, 4387, 193), (5918, 1810, 1328), (380, 6172, 5753), (3967, 3899, 1088), (6150, 557, 3866), (4266, 1123, 4322), (4482, 1670, 1177), (959, 6261, 1333),
         (6209, 662, 1822), (353, 4126, 3897), (2747, 3595, 1493)],
    32: [(47, 41, 47), (516, 511, 455), (750, 642, 1543), (1603, 1336, 289), (67, 1184, 1695), (385, 78, 4876), (574, 456, 2114), (196, 207, 8309), (1027, 1156, 4222), (5613, 1936, 156),
         (1307, 2713, 709), (41, 8383, 907), (1424, 48, 5540), (146, 1666, 5600), (1277, 195, 8324), (723, 1298, 2706), (4481, 3851, 41), (1855, 8283, 49), (3683, 2200, 489)],
}


def rounded(size):
    """With columns that are read where they lie."""
    m, n, k = size
    return m, -(-n // 8) * 8, -(-k // 8) * 8


def near(got, want, tol, name):
    import torch
    bad = ~((got.double() - want).abs() <= tol)
    assert not bool(bad.any()), (name, int(bad.sum()), [tuple(x.tolist()) for x in bad.nonzero()[:4]])
    assert bool(torch.isfinite(want).all())


def check(ctx, m, n, k, dtype, act, pad, shift):
    import torch
    import apoe
    g = torch.Generator().manual_seed(m + n + k)
    x, w = matrix(g, m, k, dtype, 1.0, pad, shift), matrix(g, n, k, dtype, 1.5 / math.sqrt(k), pad, shift)
    gy, r = matrix(g, m, n, dtype, 1.0, pad, shift), matrix(g, m, n, dtype, 1.0, pad, shift)
    b = torch.randn(n, generator=g).cuda()
    (y, y_rest), (gx, gx_rest), (gw, gw_rest) = room(m, n, dtype), room(m, k, dtype), room(n, k, dtype)
    _, pre = apoe.linear(ctx, x, w, b, act=act, residual=r, want_pre=True, out=y)
    got = apoe.linear_grad(ctx, x, w, gy, act=act, pre=pre if act != "none" else None, grad_x=gx, grad_w=gw)
    val, tol = formula(x, w, b, act, r, dtype, gy, pre)
    for name, t in dict(got, y=y, pre=pre).items():
        near(t, val[name], tol[name], (name, m, n, k, dtype, act))
    assert y_rest() and gx_rest() and gw_rest()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("size", SIZES[16])
def test_sixteen_bits(gpu_ctx, size, dtype):
    check(gpu_ctx, *size, dtype, "gelu", 3, 1)
    check(gpu_ctx, *rounded(size), dtype, "none", 8, 0)
    check(gpu_ctx, *rounded(size), dtype, "silu", 0, 0)


@pytest.mark.parametrize("size", SIZES[32])
def test_floats(gpu_ctx, size):
    check(gpu_ctx, *size, "float32", "silu", 0, 1)  # a float a load, or laid out anew
    check(gpu_ctx, *size, "float32", "none", 3, 1)
    check(gpu_ctx, *rounded(size), "float32", "gelu", 8, 0)
