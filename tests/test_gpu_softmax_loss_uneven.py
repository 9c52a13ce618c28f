"""The softmax loss on inputs of very uneven sizes (needs the GPU): rows of zeros between others, rows far larger than their
neighbours. Against the formula in 64 bits; tolerances as in test_gpu_softmax_loss.py, unless a test derives its own."""
import numpy as np
import pytest

from test_gpu_softmax_loss import check, make, oracle

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
