"""Layer norm of rows that lie far from zero, or whose values are all equal (needs the GPU).

Tolerances. The mean that is taken off first is off by at most d0 = 30 2^-24 of the mean magnitude (16 values a thread, a tree, a factor); what is left of it in the differences is taken
off too, and is then off by 30 2^-24 of their own mean magnitude, each difference rounded twice, by 2^-24 of it and of d0. So n = (x - mean) r is off by
d = (32 d0' + 3 |x - mean|) 2^-24 r with d0' the mean of |x - mean| + d0, and by 40 2^-24 of itself for r, whose terms are squares of those. The gradient: see test_gpu_layer_norm.py."""
import pytest

from layer_cases import E, SMALL, TYPES, U, close, room

pytestmark = pytest.mark.gpu


def formula(x, w, b, eps, dtype, gy):
    import torch
    x, w, b, gy = (t.detach().cpu().double() for t in (x, w, b, gy))
    c = x - x.mean(1, keepdim=True)
    r = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + eps)
    xn = c * r
    d0 = 30 * E * x.abs().mean(1, keepdim=True)
    off = (32 * (c.abs().mean(1, keepdim=True) + d0) + 3 * (c.abs() + d0)) * E * r
    n_off = off + (40 * E + (d0 * r) ** 2 * 2.0 ** -22) * xn.abs()
    y = xn * w + b
    val, tol = dict(y=y), dict(y=U[dtype] * y.abs() + w.abs() * n_off + 3 * E * (y.abs() + b.abs() + (w * xn).abs()) + SMALL[dtype])
    g = gy * w
    mean = lambda t: t.mean(1, keepdim=True)  # noqa: E731
    val["grad_x"] = r * (g - mean(g) - xn * mean(g * xn))
    size = r * (g.abs() + mean(g.abs()) + xn.abs() * mean((g * xn).abs()))
    tol["grad_x"] = (80 * E + (d0 * r) ** 2 * 2.0 ** -22) * size + r * (n_off * mean((g * xn).abs()) + (xn.abs() + n_off) * mean(g.abs() * n_off)) + U[dtype] * val["grad_x"].abs() + SMALL[dtype]
    val["grad_w"] = (gy * xn).sum(0)
    tol["grad_w"] = (x.shape[0] / 4 + 80) * E * (gy * xn).abs().sum(0) + (gy.abs() * n_off).sum(0) + SMALL[dtype]
    return val, tol


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("spread", [0.0, 1.0])
@pytest.mark.parametrize("n,d", [(3, 1), (5, 7), (40, 100), (9, 256), (33, 1000), (20, 1001), (64, 1024), (5, 4099), (3, 8192)])
def test_far_from_zero(gpu_ctx, n, d, spread, dtype):
    """Rows around 0.1 to 10 000 with values a unit apart (as far as their type holds them), and rows of one value, whose norm is zero and b remains."""
    import torch
    import apoe
    g = torch.Generator().manual_seed(n + d)
    where = 10 ** (5 * torch.rand(n, 1, generator=g) - 1) * torch.randn(n, 1, generator=g).sign()
    x = (where + spread * torch.randn(n, d, generator=g)).to(getattr(torch, dtype)).cuda()
    gy = torch.randn(n, d, generator=g).to(x.dtype).cuda()
    w, b = (1 + 0.3 * torch.randn(d, generator=g)).cuda(), (0.3 * torch.randn(d, generator=g)).cuda()
    val, tol = formula(x, w, b, 1e-5, dtype, gy)
    out, untouched = room(n, d, dtype)
    apoe.layer_norm(gpu_ctx, x, w, b, out=out)
    got = dict(apoe.layer_norm_grad(gpu_ctx, x, w, b, grad_y=gy), y=out)
    for k in val:
        close(got[k], val[k], tol[k], k)
    assert untouched()
