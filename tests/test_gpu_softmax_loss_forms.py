"""The softmax loss at sizes that choose each of its forms at the framework's dimension, many stages and several tiles either way (needs the
GPU): the formula in 64 bits, in blocks on the GPU. Tolerances as in test_gpu_softmax_loss.py."""
import pytest

from test_gpu_softmax_loss import U, pack_bits

pytestmark = pytest.mark.gpu


def make(m, n, d, dtype, seed, live):
    """Unit rows, queries that lean to their targets (0 to 3, some of them dead), on the GPU; dead rows hold NaN."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x = rand(n, d)
    x /= x.norm(dim=1, keepdim=True)
    count = torch.arange(m, device="cuda") % 4
    off = torch.zeros(m + 1, dtype=torch.int32, device="cuda")
    off[1:] = torch.cumsum(count, 0)
    idx = torch.randint(0, n, (int(off[-1]),), generator=g, device="cuda", dtype=torch.int32)
    which = torch.repeat_interleave(torch.arange(m, device="cuda"), count)
    q = (2.0 / d ** 0.5 * rand(m, d)).index_add(0, which, x[idx.long()])
    q /= q.norm(dim=1, keepdim=True)
    a = dict(queries=q.to(getattr(torch, dtype)), rows=x.to(getattr(torch, dtype)), t_off=off, t_idx=idx,
             t_val=0.5 + torch.rand(idx.shape[0], generator=g, device="cuda"), scale=16.0, weight=0.5 + torch.rand(m, generator=g, device="cuda"), live=None)
    on = torch.ones(n, dtype=torch.bool, device="cuda")
    if live is not None:
        on = torch.rand(n, generator=g, device="cuda") < live
        a["rows"][~on] = float("nan")
        a["live"] = pack_bits(on.cpu()).cuda()
    return a, on, which


def check(ctx, a, on, which, grad_queries, grad_rows):
    import torch
    import apoe
    got = apoe.softmax_loss(ctx, **a, grad_queries=grad_queries, grad_rows=grad_rows)
    dtype = str(a["queries"].dtype).split(".")[-1]
    u, half = U[dtype], dtype == "float16"
    (m, d), n, scale = a["queries"].shape, a["rows"].shape[0], a["scale"]
    zero = torch.zeros((), dtype=torch.float64, device="cuda")
    X = torch.where(on[:, None], a["rows"].double(), zero)
    XT, XA = X.T.contiguous(), X.abs()
    XAT = XA.T.contiguous()
    gx, tx = torch.zeros_like(X), torch.zeros_like(X)

    def close(name, r, want, tol):
        err = (got[name][r].double() - want).abs()
        assert bool((err <= tol).all()), (name, int((err > tol).sum()), float((err / tol).max()))
    step = max(1, (1 << 24) // n)
    for r0 in range(0, m, step):
        r = slice(r0, min(m, r0 + step))
        Q = a["queries"][r].double()
        z = scale * torch.mm(Q, XT)
        z[:, ~on] = -float("inf")
        e = slice(int(a["t_off"][r0]), int(a["t_off"][r.stop]))
        w = torch.zeros(Q.shape[0], n, dtype=torch.float64, device="cuda").index_put_((which[e] - r0, a["t_idx"][e].long()), a["t_val"][e].double(), accumulate=True)
        w[:, ~on] = 0
        W, lse = w.sum(1), torch.logsumexp(z, 1)
        p = torch.exp(z - lse[:, None])
        at = (w * torch.where(on, z, zero)).sum(1)
        logit = scale * (d + 4) * 2.0 ** -24 * torch.mm(Q.abs(), XAT).amax(1)
        tol_lse = logit + 2.0 ** -20 * (1 + lse.abs())
        close("lse", r, lse, tol_lse)
        close("loss", r, W * lse - at, W * tol_lse + W * logit + 2.0 ** -22 * at.abs())
        c = (scale * a["weight"][r].double() * (W > 0))[:, None]
        G, mass = c * (W[:, None] * p - w), c * (W[:, None] * p + w)
        noise = (2 * u + 2 * logit[:, None] + 2.0 ** -20 + (n + m) * 2.0 ** -24) * mass
        if half:
            noise += 2.0 ** -24 * 4 * c * W[:, None] * p.amax(1, keepdim=True) * on
        if grad_queries:
            want = torch.mm(G, X)
            close("grad_queries", r, want, torch.mm(noise, XA) + u * want.abs() + 2.0 ** -24 * half + 1e-30)
        if grad_rows:
            gx += torch.mm(G.T.contiguous(), Q)
            tx += torch.mm(noise.T.contiguous(), Q.abs())
    if grad_rows:
        close("grad_rows", slice(None), gx, tx + u * gx.abs() + 2.0 ** -24 * half + 1e-30)
        assert not bool(got["grad_rows"][~on].any())


# Tiles of 512 x 32, 256 x 128 (one and several tiles of queries), 256 x 256 with its wide products for both gradients, and 128 x 128 whose rows'
# gradient takes the wide tiles; ragged either way, 1000 columns being no whole number of tiles.
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("m,n,d", [(20, 140_003, 1024), (5, 131_500, 64), (32, 140_100, 1000), (100, 70_003, 1024), (300, 24_003, 1000), (500, 33_003, 1024), (1100, 13_501, 1000), (130, 17_003, 1024)])
def test_forms_of_16_bits(gpu_ctx, m, n, d, dtype):
    for live, grad_queries, grad_rows in ((0.7, True, False), (None, True, True)) if m % 2 == 0 else ((None, True, False), (0.7, True, True)):
        check(gpu_ctx, *make(m, n, d, dtype, m + d, live), grad_queries, grad_rows)
    check(gpu_ctx, *make(m, n, d, dtype, m, 0.9), False, True)
    check(gpu_ctx, *make(m, n, d, dtype, m, 0.3), False, False)


@pytest.mark.parametrize("m,n,d", [(64, 20_003, 1024), (20, 40_003, 1000), (500, 33_003, 1024), (300, 9001, 1000), (2000, 5003, 1024), (70, 3000, 2052)])
def test_forms_of_float(gpu_ctx, m, n, d):
    """Tiles of 128 x 64, 256 x 256 and 128 x 128, the queries' gradient from more than 16 splits and from few, and with the rows' beside it."""
    check(gpu_ctx, *make(m, n, d, "float32", m, 0.7), True, False)
    check(gpu_ctx, *make(m, n, d, "float32", m, None), True, True)
    check(gpu_ctx, *make(m, n, d, "float32", m, None), False, False)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("m", [4, 5, 6, 7, 8, 9])
def test_where_few_queries_end(gpu_ctx, m, dtype):
    """Up to four queries of 16 bits and up to eight of float32 are carried in registers, the last set of them not always full."""
    for n, d, live in ((3, 1024, None), (130, 1032, 0.8), (2500, 1024, 0.3), (20_001, 40, 0.9)):
        a, on, which = make(m, n, d, dtype, m + n, live)
        if bool(on.any()):
            check(gpu_ctx, a, on, which, True, False)
            check(gpu_ctx, a, on, which, False, False)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_pieces_at_many_columns(gpu_ctx, dtype):
    """More exponentials than one piece holds (16 bits: 4096 x 140 003 are 1.07 GiB; float32, whose gradients of the rows have three parts: 4096 x 44 003), with 72 columns."""
    n = 140_003 if dtype == "bfloat16" else 44_003
    check(gpu_ctx, *make(4096, n, 72, dtype, 1, 0.95), True, True)
    check(gpu_ctx, *make(4096, n if dtype == "bfloat16" else 66_003, 72, dtype, 2, None), True, False)
