"""The operators on matrices that reach past 4 GiB from their first byte (few rows, far apart): bit for bit what the same values close
together give."""
import pytest

pytestmark = pytest.mark.gpu


def far(t, gap):
    """`t` with its rows (or matrices) `gap` elements apart; nothing between them is written."""
    import torch
    shape, step = t.shape, [gap] + list(t.stride())[1:]
    store = torch.empty((shape[0] - 1) * gap + t[0].numel(), dtype=t.dtype, device="cuda")
    v = store.as_strided(shape, step)
    v.copy_(t)
    assert shape[0] * gap * t.element_size() > 1 << 32
    return v


@pytest.mark.parametrize("m", [2, 70, 300])
@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_softmax_loss(gpu_ctx, dtype, m):
    import torch
    import apoe
    g = torch.Generator().manual_seed(m)
    n, d, gap = 17_000, 64, 1 << 18
    gap = gap if dtype == "float16" else gap // 2
    x, q = (torch.randn(k, d, generator=g).to(getattr(torch, dtype)).cuda() for k in (n, m))
    off, idx = torch.arange(m + 1, dtype=torch.int32, device="cuda"), torch.randint(n - 50, n, (m,), generator=g).to(torch.int32).cuda()
    for rows in (False, True):
        gx = far(torch.zeros_like(x), gap) if rows else False
        near = apoe.softmax_loss(gpu_ctx, q, x, off, idx, scale=0.5, grad_queries=True, grad_rows=rows)
        away = apoe.softmax_loss(gpu_ctx, q, far(x, gap), off, idx, scale=0.5, grad_queries=True, grad_rows=gx)
        for k in near:
            assert bool((near[k] == away[k]).all()), k


@pytest.mark.parametrize("short,cols", [(40, 300), (130, 200)])
def test_orthogonalize(gpu_ctx, short, cols):
    import torch
    import apoe
    g = torch.Generator().manual_seed(short)
    x = torch.randn(3, short, cols, generator=g).bfloat16().cuda()
    near = apoe.orthogonalize(gpu_ctx, x)
    out = far(torch.zeros_like(x), (1 << 30) + 64)
    assert bool((apoe.orthogonalize(gpu_ctx, far(x, (1 << 30) + 64), out=out) == near).all())
    rows = far(x[0], (1 << 32) // 2 // (short - 1) // 8 * 8 + 8)
    assert bool((apoe.orthogonalize(gpu_ctx, rows) == apoe.orthogonalize(gpu_ctx, x[0])).all())


def test_gated_residual(gpu_ctx):
    import torch
    import apoe
    g = torch.Generator().manual_seed(1)
    n, d, gap = 5000, 200, 1 << 19
    x, h, gate, gu = (torch.randn(n, d, generator=g).half().cuda() for _ in range(4))
    vec = {k: torch.rand(d, generator=g).cuda() for k in ("scale", "w_post", "w_next")}
    fx, fh = far(x, gap), far(h, gap)
    for a, b in zip(apoe.gated_residual(gpu_ctx, x, h, gate=gate, **vec), apoe.gated_residual(gpu_ctx, fx, fh, gate=gate, **vec)):
        assert bool((a == b).all())
    near, away = (apoe.gated_residual_grad(gpu_ctx, a, b, gate=gate, **vec, grad_u=gu) for a, b in ((x, h), (fx, fh)))
    for k in near:
        assert bool((near[k] == away[k]).all()), k
