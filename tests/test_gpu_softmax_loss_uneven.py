"""The softmax loss on inputs of very uneven sizes (needs the GPU): rows of zeros between others, rows far larger than their neighbours,
queries whose weights are far apart. Against the formula in 64 bits; tolerances as in test_gpu_softmax_loss.py, unless a test derives its own."""
import numpy as np
import pytest

from test_gpu_softmax_loss import U, check, make, oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size", [1.0, 1e-3, 1e-5])
@pytest.mark.parametrize("m", [9, 64, 130])
def test_rows_of_zeros_cost_their_neighbours_nothing(gpu_ctx, m, size):
    """32 live rows that are all zero (terms that nobody uses, a tail that is not filled yet) beside rows of any length, float32."""
    a = make(m, 512, 64, "float32", seed=m, scale=8.0 / size)
    a["rows"] *= size
    a["rows"][160:192] = 0
    a["rows"][480:] = 0
    check(gpu_ctx, a, True, False)
    check(gpu_ctx, a, True, True)


def close_by_row(gpu_ctx, a, grad_rows):
    """float32. A logit is off by at most d_ij = scale (dim + 4) 2^-24 sum_k |q_k x_jk|, which is by its own row's size; lse by the mean of
    that, so p_ij is off by a factor of 1 + 2 d_ij + 2 sum_j p_ij d_ij + 2^-20, and the sums by (m + n) 2^-24 of what they add up. What is below
    2^-38 of the largest p |x| of a query is left out, and p |x| of a row has the roundings of two fp16 numbers: 2^-22."""
    import apoe
    got = apoe.softmax_loss(gpu_ctx, **a, grad_queries=True, grad_rows=grad_rows)
    want, _ = oracle(a)
    f64 = lambda t: t.detach().cpu().double().numpy()  # noqa: E731
    q, x, cw = f64(a["queries"]), f64(a["rows"]), f64(a["weight"])
    m, n, d = q.shape[0], x.shape[0], q.shape[1]
    z = a["scale"] * q @ x.T
    p = np.exp(z - want["lse"][:, None])
    w = np.zeros((m, n))
    off, idx = a["t_off"].cpu().numpy(), a["t_idx"].cpu().numpy()
    for i in range(m):
        for e in range(off[i], off[i + 1]):
            w[i, idx[e]] += float(a["t_val"][e])
    logit = a["scale"] * (d + 4) * 2.0 ** -24 * (np.abs(q) @ np.abs(x).T)
    tol_lse = (p * logit).sum(1) + 2.0 ** -20 * (1 + np.abs(want["lse"]))
    c = (cw * a["scale"])[:, None] * (w.sum(1) > 0)[:, None]
    mass = c * (w.sum(1, keepdims=True) * p + w)
    noise = (2 * logit + 2 * tol_lse[:, None] + 2.0 ** -20 + 2.0 ** -22 + (n + m) * 2.0 ** -24) * mass
    lost = n * 2.0 ** -38 * (c * w.sum(1, keepdims=True) * p * np.abs(x).max(1)[None, :]).max(1, keepdims=True)
    tol = dict(lse=tol_lse, loss=w.sum(1) * tol_lse + (w * logit).sum(1) + 2.0 ** -22 * np.abs(w * z).sum(1),
               grad_queries=noise @ np.abs(x) + lost + 2.0 ** -23 * np.abs(want["grad_queries"]),
               grad_rows=noise.T @ np.abs(q) + 2.0 ** -23 * np.abs(want["grad_rows"]) + (n + m) * 2.0 ** -126 * a["scale"])
    for k, t in got.items():
        err = np.abs(f64(t) - want[k])
        bad = ~(err <= tol[k])
        assert not bad.any(), (k, int(bad.sum()), float((err / np.maximum(tol[k], 1e-300)).max()))


@pytest.mark.parametrize("grad_rows", [False, True])
@pytest.mark.parametrize("size", [1e2, 1e4, 1e8])
def test_a_large_row_costs_its_neighbours_nothing(gpu_ctx, size, grad_rows):
    """Rows of length one, and among them some that are far longer and far from every query, float32: what the others' logits and gradients
    are is not worse for it."""
    import torch
    a = make(70, 600, 64, "float32", seed=7, scale=8.0)
    g = torch.Generator().manual_seed(1)
    v = torch.randn(64, generator=g)
    v /= v.norm()
    q = a["queries"].cpu() + v
    x = a["rows"].cpu()
    named = set(a["t_idx"].cpu().tolist())
    for j in (5, 40, 77, 300, 599):
        if j not in named:
            x[j] = -size * v
    a["queries"] = (q / q.norm(dim=1, keepdim=True)).cuda()
    a["rows"] = x.cuda()
    assert float((a["queries"] @ v.cuda()).min()) > 0.2  # every query's logit of those rows is far below the others'
    close_by_row(gpu_ctx, a, grad_rows)


@pytest.mark.parametrize("m", [70, 300])
@pytest.mark.parametrize("apart", [2.0 ** 8, 2.0 ** 22])
@pytest.mark.parametrize("grad_queries", [True, False])
def test_weights_far_apart(gpu_ctx, m, apart, grad_queries):
    """float16, both gradients, one query that weighs 2^22 times what the others do and finds its row, so that it leaves nothing elsewhere. Tolerances:
    a query's weight is taken as 2^11 to 2^12 (with its targets' beside it 2^13), so what is lost among the subnormal numbers, 2^-25 for each row, is
    2^-36 of it; the products take queries times their weights, the largest value as 2^13 to 2^14: 2^-38 of it is lost."""
    import apoe
    import torch
    g = torch.Generator().manual_seed(m)
    n, d, scale = 20_000, 64, 4.0
    v = torch.randn(d, generator=g)
    x = torch.randn(n, d, generator=g) / d ** 0.5 + v / v.norm()  # around one direction, so that the rows' mean is no small part
    x /= x.norm(dim=1, keepdim=True)
    idx = torch.randint(0, n, (m,), generator=g)
    q = torch.randn(m, d, generator=g) / d ** 0.5
    q[0] = 40 * (x[idx[0]] - v / v.norm())
    weight = torch.full((m,), 2.0 ** 14 / apart)
    weight[0] = 2.0 ** 14
    a = dict(queries=q.half().cuda(), rows=x.half().cuda(), t_off=torch.arange(m + 1, dtype=torch.int32).cuda(), t_idx=idx.int().cuda(), t_val=None,
             scale=scale, live=None, weight=weight.cuda())
    got = apoe.softmax_loss(gpu_ctx, **a, grad_queries=grad_queries, grad_rows=True)
    q, x, cw = (a[k].cpu().double().numpy() for k in ("queries", "rows", "weight"))
    z = scale * q @ x.T
    z -= z.max(1, keepdims=True)
    p = np.exp(z) / np.exp(z).sum(1, keepdims=True)
    c = (cw * scale)[:, None]
    w = np.zeros((m, n))
    w[np.arange(m), idx.numpy()] = 1
    G, mass, u = c * (p - w), c * (p + w), U["float16"]
    logit = scale * (d + 4) * 2.0 ** -24 * (np.abs(q) @ np.abs(x).T).max(1, keepdims=True)
    noise = (2 * u + 4 * logit + 2.0 ** -20 + (n + m) * 2.0 ** -24) * mass + 2.0 ** -36 * c
    if grad_queries:
        want = G @ x
        tol = noise @ np.abs(x) + u * np.abs(want) + 2.0 ** -24
        err = np.abs(got["grad_queries"].double().cpu().numpy() - want)
        assert (err <= tol).all(), float((err / tol).max())
    want = G.T @ q
    top = (c * np.abs(q).max(1, keepdims=True)).max()
    tol = noise.T @ np.abs(q) + 2.0 ** -38 * top * (mass / c).sum(0)[:, None] + u * np.abs(want) + 2.0 ** -24
    err = np.abs(got["grad_rows"].double().cpu().numpy() - want)
    assert (err <= tol).all(), float((err / tol).max())


def test_the_queries_gradient_is_as_good_beside_the_rows(gpu_ctx):
    """float16, weights 2^20 apart: grad_queries with grad_rows against grad_queries alone, each against 64 bits, query by query."""
    import apoe
    import torch
    a = make(80, 5000, 64, "float16", seed=3, targets=2, scale=1.0)
    a["weight"] = torch.where(torch.arange(80) % 2 == 0, 2.0 ** 12, 2.0 ** -8).cuda()
    want = oracle(a)[0]["grad_queries"]
    some = np.abs(want).max(1) > 0
    err = {}
    for rows in (False, True):
        got = apoe.softmax_loss(gpu_ctx, **a, grad_queries=True, grad_rows=rows)["grad_queries"].double().cpu().numpy()
        err[rows] = (np.linalg.norm(got - want, axis=1)[some] / np.linalg.norm(want, axis=1)[some])
    # a second rounding of the coefficients, 2^-11 each, beside the result's: sqrt(3 / 2) and what is left to chance
    assert (err[True] <= 1.5 * err[False] + 2.0 ** -11 / 3 ** 0.5).all(), float((err[True] / err[False]).max())


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("m,n,d", [(80, 3000, 64), (300, 5000, 1024), (4000, 500, 1024), (300, 700, 2056)])
def test_the_targets_of_a_query_are_not_rounded_in_its_gradient(gpu_ctx, m, n, d, dtype):
    """With grad_rows too, where the coefficients of both products are in the rows' type: what grad_queries is off by beside its own rounding is by the
    coefficients of the other rows, two roundings of u each, independent: at most four times u sqrt(sum p^2) of a query's weight, and the logits' part."""
    import apoe
    import torch
    a = make(m, n, d, dtype, seed=m, targets=3, scale=10.0)
    a["weight"] = torch.full((m,), 1.0, device="cuda")
    got = apoe.softmax_loss(gpu_ctx, **a, grad_queries=True, grad_rows=True)["grad_queries"].double().cpu().numpy()
    want = oracle(a)[0]["grad_queries"]
    once = torch.from_numpy(want).to(getattr(torch, dtype)).double().numpy()
    q, x = (a[k].cpu().double().numpy() for k in ("queries", "rows"))
    z = a["scale"] * q @ x.T
    p = np.exp(z - z.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    off = a["t_off"].cpu().numpy()
    w, idx = np.zeros((m, n)), a["t_idx"].cpu().numpy()
    for i in range(m):
        for e in range(off[i], off[i + 1]):
            w[i, idx[e]] += float(a["t_val"][e])
    W = w.sum(1)
    logit = a["scale"] * (d + 4) * 2.0 ** -24 * (np.abs(q) @ np.abs(x).T).max(1)
    others = 4 * U[dtype] * np.sqrt((p ** 2).sum(1)) + 4 * logit + 2.0 ** -20
    length = np.linalg.norm(x, axis=1).max()
    some = W > 0
    err, own = np.linalg.norm(got - want, axis=1), np.linalg.norm(once - want, axis=1)
    # own rounding: the value that is rounded is another, so its error is another draw of d values: 1.5 times covers it from 64 columns on
    tol = 1.5 * own + a["scale"] * W * others * length
    assert (err[some] <= tol[some]).all(), float((err[some] / tol[some]).max())
    target = a["scale"] * np.sqrt((w ** 2).sum(1)) * U[dtype] / 12 ** 0.5  # what the targets' rounding alone would come to
    assert float(np.mean(err[some])) < float(np.mean(np.sqrt(own ** 2 + (0.5 * target) ** 2)[some]) + np.mean((a["scale"] * W * (others / 4 + 2 * logit))[some]))


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("odd", [1.0, 0.75, 1.0 + 2.0 ** -9, 1.0 - 2.0 ** -9 / 3, 1.0 + 2.0 ** -12])
def test_equal_weights_do_not_turn_all_targets_the_same_way(gpu_ctx, dtype, odd):
    """Every query weighs the same and names one row; the logits are near zero, so that a row's gradient is its targets' but for 1 / n. The targets' coefficients
    are rounded in the rows' type, all to the same number: along the gradient itself, where the result's roundings average, it has the right length
    whatever the weight's bits are. Off by 2 / n (the probability that rounding takes from one, up to half a unit there) and u / sqrt(values) three times."""
    import apoe
    import torch
    m, n, d = 300, 6000, 256
    a = make(m, n, d, dtype, seed=5, targets=1, scale=0.25)
    a["t_off"] = torch.arange(m + 1, dtype=torch.int32, device="cuda")
    a["t_idx"] = torch.randint(0, n, (m,), generator=torch.Generator().manual_seed(1)).int().cuda()
    a["t_val"] = None
    a["weight"] = torch.full((m,), 64.0 * odd, device="cuda")
    got = apoe.softmax_loss(gpu_ctx, **a, grad_queries=False, grad_rows=True)["grad_rows"].double().cpu().numpy()
    want = oracle(a)[0]["grad_rows"]
    length = float((got * want).sum() / (want * want).sum())
    assert abs(length - 1) < 2 / n + 3 * U[dtype] / (m * d) ** 0.5 + 2.0 ** -20, length - 1
