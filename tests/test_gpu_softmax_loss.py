"""Softmax cross entropy over the rows of a table, and its gradients, against the formula in 64 bits (needs the GPU).

Tolerances. u is half a unit of the type's last place relative to a value: 2^-11 (float16), 2^-8 (bfloat16: 7 bits behind the point), 2^-24 (float32).
 - A logit is a sum of dim products in 32 bits, times the scale: off by at most d = scale (dim + 4) 2^-24 max_j sum_k |q_k x_jk|.
   lse is off by no more than its logits, plus the rounding of exponentials and of their sum: d + 2^-20 (1 + |lse|); a loss by
   |W| times that, plus its targets' logits.
 - A gradient is a sum of coefficients G_ij = c (W p_ij - w_ij) times rows. Coefficients are rounded to the type once or twice, p is
   off by a factor of 1 + 2 d + 2^-20, the sum is in 32 bits, and the result is rounded: the bound below sums these over
   (|W| p_ij + |w_ij|) |x_jk|. float16 coefficients can fall among the subnormal numbers, relative to a group's largest: 2^-24 of the
   largest exponential that shares a row, for every row. What is below the smallest normal float counts as zero: 2^-126 a term.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def make(m, n, d, dtype, seed, targets=2, live=None, graded=True, scale=8.0, pad=0, spread=3.0):
    """Inputs on the GPU; live: share of the rows, or None."""
    import torch
    g = torch.Generator().manual_seed(seed)
    rows = torch.randn(n, d, generator=g)
    rows /= rows.norm(dim=1, keepdim=True)
    count = torch.randint(0, targets + 1, (m,), generator=g)
    off = torch.zeros(m + 1, dtype=torch.int32)
    off[1:] = torch.cumsum(count, 0)
    idx = torch.randint(0, n, (int(off[-1]),), generator=g, dtype=torch.int32)
    q = spread / d ** 0.5 * torch.randn(m, d, generator=g)
    for i in range(m):
        for e in range(int(off[i]), int(off[i + 1])):
            q[i] += rows[int(idx[e])]
    q /= q.norm(dim=1, keepdim=True)
    val = 0.25 + torch.rand(int(off[-1]), generator=g) if graded else None
    words = None
    if live is not None:
        on = torch.rand(n, generator=g) < live
        words = pack_bits(on)
    dt = getattr(torch, dtype)

    def wide(t):
        t = t.to(dt)
        if not pad:
            return t.cuda()
        w = torch.full((t.shape[0], d + pad), float("nan"), dtype=dt)
        w[:, :d] = t
        return w.cuda()[:, :d]
    cuda = lambda t: None if t is None else t.cuda()  # noqa: E731
    return dict(queries=wide(q), rows=wide(rows), t_off=off.cuda(), t_idx=idx.cuda(), t_val=cuda(val), scale=scale, live=cuda(words),
                weight=(torch.rand(m, generator=g) / m).cuda())


def pack_bits(on):
    import torch
    n = on.numel()
    bits = np.zeros((n + 31) // 32 * 32, np.uint8)
    bits[:n] = on.numpy()
    return torch.from_numpy(np.packbits(bits, bitorder="little").view(np.int32).copy())


def oracle(a):
    """The formula in 64 bits on the CPU: (dict of results, dict of tolerances)."""
    f64 = lambda t: t.detach().cpu().double().numpy()  # noqa: E731
    q, x = f64(a["queries"]), f64(a["rows"])
    m, n, d = q.shape[0], x.shape[0], q.shape[1]
    u = U[str(a["queries"].dtype).split(".")[-1]]
    on = np.ones(n, bool)
    if a["live"] is not None:
        on = np.unpackbits(a["live"].cpu().numpy().view(np.uint8), bitorder="little")[:n].astype(bool)
    x = np.where(on[:, None], x, 0.0)
    off, idx = a["t_off"].cpu().numpy(), a["t_idx"].cpu().numpy().astype(np.int64)
    cw = np.ones(m) if a["weight"] is None else f64(a["weight"])
    w = np.zeros((m, n))
    for i in range(m):
        k = off[i + 1] - off[i]
        for e in range(off[i], off[i + 1]):
            if 0 <= idx[e] < n and on[idx[e]]:
                w[i, idx[e]] += 1.0 / k if a["t_val"] is None else float(a["t_val"][e])
    W, named = w.sum(1), np.abs(w).sum(1)
    counts = (named > 0) & (cw != 0)
    q = np.where((named > 0)[:, None] | np.isfinite(q).all(1)[:, None], q, 0.0) if not np.isfinite(q).all() else q
    z = a["scale"] * q @ x.T
    z[:, ~on] = -np.inf
    top = np.where(on.any(), z.max(1), 0.0)
    with np.errstate(divide="ignore"):
        lse = top + np.log(np.exp(z - top[:, None]).sum(1)) if on.any() else np.full(m, -np.inf)
    at = np.where(w != 0, w * np.where(on[None, :], z, 0.0), 0.0).sum(1)
    loss = np.where(named > 0, W * np.where(np.isfinite(lse), lse, 0.0) - at, 0.0)
    p = np.exp(z - np.where(np.isfinite(lse), lse, 0.0)[:, None]) * on[None, :]
    c = np.where(counts, cw * a["scale"], 0.0)
    G = c[:, None] * (W[:, None] * p - w)
    out = dict(loss=loss, lse=lse, grad_queries=G @ x, grad_rows=G.T @ np.where(counts[:, None], q, 0.0))
    logit = a["scale"] * (d + 4) * 2.0 ** -24 * (np.abs(q) @ np.abs(x).T).max(1)
    tol_lse = logit + 2.0 ** -20 * (1 + np.abs(np.where(np.isfinite(lse), lse, 0.0)))
    mass = np.abs(c)[:, None] * (np.abs(W)[:, None] * p + np.abs(w))
    off_p = 2 * u + 2 * logit + 2.0 ** -20 + (n + m) * 2.0 ** -24
    tiny = 2.0 ** -24 * np.abs(c) * (np.abs(W) + named) * p.max(1) * 2 if u == 2.0 ** -11 else np.zeros(m)
    noise = off_p[:, None] * mass + tiny[:, None] * on[None, :]
    tol = dict(loss=np.abs(W) * tol_lse + named * logit + 2.0 ** -22 * np.abs(at), lse=tol_lse,
               grad_queries=noise @ np.abs(x) + u * np.abs(out["grad_queries"]) + 2.0 ** -24 * (u == 2.0 ** -11) + (n + m) * 2.0 ** -126 * a['scale'],
               grad_rows=noise.T @ np.abs(np.where(counts[:, None], q, 0.0)) + u * np.abs(out["grad_rows"]) + 2.0 ** -24 * (u == 2.0 ** -11) + (n + m) * 2.0 ** -126 * a['scale'])
    return out, tol


def check(ctx, a, grad_queries=True, grad_rows=False):
    import apoe
    got = apoe.softmax_loss(ctx, **a, grad_queries=grad_queries, grad_rows=grad_rows)
    want, tol = oracle(a)
    assert set(got) == {"loss", "lse"} | ({"grad_queries"} if grad_queries is not False else set()) | ({"grad_rows"} if grad_rows is not False else set())
    for name, t in got.items():
        v = t.double().cpu().numpy()
        same = (v == want[name]) | (np.abs(v - want[name]) <= tol[name])
        assert same.all(), (name, np.argwhere(~same)[:5], v[~same][:5], want[name][~same][:5], tol[name][~same][:5])
    return got


SIZES = [(1, 1, 8), (1, 4000, 1024), (2, 31, 16), (5, 129, 72), (33, 512, 64), (64, 1000, 136), (65, 513, 1024), (129, 127, 40), (300, 1100, 256)]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("m,n,d", SIZES)
def test_sizes_and_types(gpu_ctx, m, n, d, dtype):
    a = make(m, n, d, dtype, seed=m + n, live=0.6 if n % 2 else None)
    check(gpu_ctx, a, True, False)
    check(gpu_ctx, a, True, True)
    check(gpu_ctx, a, False, True)
    check(gpu_ctx, a, False, False)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("m", [1, 2, 3, 4, 5])
def test_few_queries(gpu_ctx, m, dtype):
    """Queries that are carried in registers (up to four of 16 bits, two of float32, rows of up to 1024 columns), and the sizes around."""
    for n, d, live in ((1, 8, None), (3, 1024, None), (4, 520, None), (5, 1000, 0.5), (33, 16, 0.0), (130, 1032, 0.8), (2500, 1024, 0.3), (70_001, 24, 0.9)):
        a = make(m, n, d, dtype, seed=m + n, live=live, targets=3, scale=12.0, pad=8 if d < 1000 else 0)
        check(gpu_ctx, a, True, False)
        check(gpu_ctx, a, False, False)


def test_few_queries_whose_logits_climb(gpu_ctx):
    """Each row above the last by more than the running exponent bears, in both orders, and below it by hundreds."""
    import torch
    for order in (1, -1):
        a = make(2, 40, 32, "bfloat16", seed=3, scale=100.0)
        x = torch.zeros(40, 32)
        x[:, 0] = torch.arange(40.0) / 8 - 2
        a["rows"] = (x if order == 1 else x.flip(0)).to(torch.bfloat16).contiguous().cuda()
        a["queries"] = torch.eye(2, 32).to(torch.bfloat16).cuda()
        check(gpu_ctx, a, True, False)


@pytest.mark.parametrize("dtype,d", [("float16", 4096), ("bfloat16", 2056), ("float32", 4092), ("float32", 4)])
def test_long_and_short_rows(gpu_ctx, dtype, d):
    check(gpu_ctx, make(70, 300, d, dtype, seed=d), True, True)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
def test_strided_matrices_whose_gaps_hold_nan(gpu_ctx, dtype):
    import torch
    a = make(40, 260, 64, dtype, seed=3, pad=8)
    g = torch.full((40, 80), 7.0, dtype=a["queries"].dtype, device="cuda")
    got = check(gpu_ctx, a, g[:, :64], True)
    assert got["grad_queries"].data_ptr() == g.data_ptr() and bool((g[:, 64:] == 7).all())


@pytest.mark.parametrize("grad_rows", [False, True])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
def test_dead_rows_are_not_looked_at(gpu_ctx, dtype, grad_rows):
    import torch
    for m, n, share in ((3, 700, 0.5), (70, 700, 0.01), (40, 260, 0.0), (130, 1030, 0.0)):
        a = make(m, n, 64, dtype, seed=5, live=share)
        on = np.unpackbits(a["live"].cpu().numpy().view(np.uint8), bitorder="little")[:n].astype(bool)
        bad = torch.from_numpy(~on).cuda()
        a["rows"][bad] = float("nan")
        a["rows"][bad, ::2] = float("inf")
        got = check(gpu_ctx, a, True, grad_rows)
        if share == 0.0:
            assert bool((got["lse"] == float("-inf")).all()) and not bool(got["loss"].any()) and not bool(got["grad_queries"].any())
        if grad_rows:
            assert not bool(got["grad_rows"][bad].any())


def test_live_bits_past_the_last_row_count_nothing(gpu_ctx):
    a = make(20, 45, 32, "float16", seed=1, live=1.1)
    a["live"].fill_(-1)
    check(gpu_ctx, a, True, True)


@pytest.mark.parametrize("grad_rows", [False, True])
def test_targets_of_every_kind(gpu_ctx, grad_rows):
    """No target, one named three times, dead ones, ids past the end, weights that cancel, negative and zero weights, shares."""
    import torch
    a = make(8, 300, 64, "float16", seed=9)
    lists = [[], [7, 7, 7, 8], [5, 299, 300, 2 ** 30], [1, 2], [1, 2], [3, 3], [4, 6], [10]]
    vals = [[], [.1, .2, .3, .4], [1, 1, 1, 1], [.5, -.5], [1, -2], [1, -1], [0, 1], [0]]
    a["t_off"] = torch.tensor(np.cumsum([0] + [len(k) for k in lists]), dtype=torch.int32, device="cuda")
    a["t_idx"] = torch.tensor(sum(lists, []), dtype=torch.int32, device="cuda")
    a["t_val"] = torch.tensor(sum(vals, []), dtype=torch.float32, device="cuda")
    on = torch.ones(300, dtype=torch.bool)
    on[[2, 299]] = False
    a["live"] = pack_bits(on).cuda()
    check(gpu_ctx, a, True, grad_rows)
    check(gpu_ctx, dict(a, t_val=None), True, grad_rows)


@pytest.mark.parametrize("grad_rows", [False, True])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_queries_that_count_nothing_may_hold_anything(gpu_ctx, dtype, grad_rows):
    import apoe
    a = make(50, 400, 64, dtype, seed=2)
    counts = (a["t_off"][1:] - a["t_off"][:-1]).cpu().numpy()
    none = int(np.flatnonzero(counts == 0)[0])
    some = int(np.flatnonzero(counts > 0)[0])
    a["weight"][some] = 0.0
    clean = apoe.softmax_loss(gpu_ctx, **a, grad_queries=True, grad_rows=grad_rows)
    a["queries"][none] = float("nan")
    a["queries"][some] = float("inf")
    got = apoe.softmax_loss(gpu_ctx, **a, grad_queries=True, grad_rows=grad_rows)
    assert float(got["loss"][none]) == 0.0
    for i in (none, some):
        assert not bool(got["grad_queries"][i].any())
    for name in ("grad_rows",) if grad_rows else ():
        assert bool((got[name] == clean[name]).all())


def test_logits_of_any_size(gpu_ctx):
    """Far apart and far from zero: references that differ by hundreds between groups, exponentials that all underflow but one."""
    import torch
    for dtype in ("float16", "bfloat16", "float32"):
        for grad_rows in (False, True):
            a = make(40, 1500, 64, dtype, seed=4, scale=300.0)
            check(gpu_ctx, a, True, grad_rows)
            b = dict(a, rows=a["rows"].clone())
            b["rows"][:700] *= -1.0
            b["rows"][700:] *= 0.0
            check(gpu_ctx, b, True, grad_rows)
            b["rows"] = -torch.ones_like(a["rows"])
            b["queries"] = torch.ones_like(a["queries"])
            check(gpu_ctx, b, True, grad_rows)


def test_a_query_that_is_served_well_keeps_its_small_gradient(gpu_ctx):
    """p_t = 1 - 1e-3 or so: W p_t - w_t is formed in 32 bits. What is left is the other rows' share, to the type's accuracy."""
    import torch
    import apoe
    for dtype in ("bfloat16", "float16"):
        for grad_rows in (False, True):
            a = make(64, 600, 256, dtype, seed=6, targets=1, graded=False, scale=16.0, spread=0.1)
            a["weight"].fill_(1024.0)  # as a loss scale: without it the gradient itself is below float16's normal numbers
            got = apoe.softmax_loss(gpu_ctx, **a, grad_queries=True, grad_rows=grad_rows)
            want, _ = oracle(a)
            u = U[dtype]
            # the loss, about 1.2e-4, is the difference of lse and a target's logit, 23 in base 2, each right to a few roundings of
            # 2^-24 in 32 bits: 4 * 23 * 2^-24 / 1.2e-4 = 4.6 %. p_t rounded to the type would be off by u / 1.2e-4: four times and more
            err = np.linalg.norm(got["grad_queries"].double().cpu().numpy() - want["grad_queries"]) / np.linalg.norm(want["grad_queries"])
            assert err < 2 * u + 4 * 23 * 2.0 ** -24 / 1.2e-4, err


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_a_batch_that_fills_the_gpu_without_splits(gpu_ctx, dtype):
    """4003 queries against 70 rows of 1024 columns, both gradients: the queries' one is written by its product itself."""
    check(gpu_ctx, make(4003, 70, 1024, dtype, seed=5, live=0.8), True, True)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("grad_rows", [False, True])
def test_more_than_one_piece(gpu_ctx, dtype, grad_rows):
    """4096 queries over rows whose exponentials fill more than one piece of 256 MiB, ragged at the end; the formula in blocks on the GPU."""
    import torch
    import apoe
    m, n, d = 4096, 36_011 if dtype == "bfloat16" else 17_003, 16
    g = torch.Generator(device="cuda").manual_seed(1)
    dt = getattr(torch, dtype)
    q = torch.randn(m, d, generator=g, device="cuda").to(dt)
    x = torch.randn(n, d, generator=g, device="cuda").to(dt)
    t_off = torch.arange(m + 1, dtype=torch.int32, device="cuda")
    t_idx = torch.randint(0, n, (m,), generator=g, device="cuda", dtype=torch.int32)
    scale = 0.5
    got = apoe.softmax_loss(gpu_ctx, q, x, t_off, t_idx, scale=scale, grad_queries=True, grad_rows=grad_rows)
    gx = torch.zeros(n, d, dtype=torch.float64, device="cuda")
    X = x.double()
    for r in range(0, m, 512):
        Q = q[r:r + 512].double()
        z = scale * Q @ X.T
        lse = torch.logsumexp(z, 1)
        t = t_idx[r:r + 512].long()
        k = torch.arange(512, device="cuda")
        loss = lse - z[k, t]
        G = torch.exp(z - lse[:, None])
        mass = scale * (G @ X.abs()) + scale * X[t].abs()
        G[k, t] -= 1
        G *= scale
        # |logit| < 50 or so: p is off by 2 d = 2 * 0.5 * 20 * 2^-24 * 50
        off = 2 * U[dtype] + 6e-5 + (n + m) * 2.0 ** -24
        assert bool(((got["loss"][r:r + 512] - loss).abs() <= 6e-5 + 2.0 ** -20 * loss.abs()).all())
        gq = G @ X
        assert bool(((got["grad_queries"][r:r + 512].double() - gq).abs() <= off * mass + U[dtype] * gq.abs()).all())
        gx += G.T.contiguous() @ Q
    if grad_rows:
        err = float((got["grad_rows"].double() - gx).norm() / gx.norm())
        assert err < 2 * U[dtype] + 6e-5, err


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("grad_rows", [False, True])
def test_pieces_of_a_gibibyte(gpu_ctx, dtype, grad_rows):
    """8192 queries over rows whose exponentials pass 1 GiB, ragged, a tenth of them dead and holding NaN; one query in 64 names no row, the others
    up to three, some of them dead. The formula in blocks on the GPU."""
    import torch
    import apoe
    m, n, d = 8192, 35_005 if dtype == "float32" else 70_003, 16
    g = torch.Generator(device="cuda").manual_seed(2)
    dt = getattr(torch, dtype)
    q = torch.randn(m, d, generator=g, device="cuda").to(dt)
    x = torch.randn(n, d, generator=g, device="cuda").to(dt)
    on = torch.rand(n, generator=g, device="cuda") < 0.9
    X = torch.where(on[:, None], x.double(), torch.zeros((), dtype=torch.float64, device="cuda"))
    x[~on] = float("nan")
    count = torch.arange(m, device="cuda") % 4
    t_off = torch.zeros(m + 1, dtype=torch.int32, device="cuda")
    t_off[1:] = torch.cumsum(count, 0)
    t_idx = torch.randint(0, n, (int(t_off[-1]),), generator=g, device="cuda", dtype=torch.int32)
    t_val = torch.rand(t_idx.shape[0], generator=g, device="cuda") + 0.5
    weight = torch.rand(m, generator=g, device="cuda") + 0.5
    scale = 0.5
    got = apoe.softmax_loss(gpu_ctx, q, x, t_off, t_idx, t_val, scale=scale, weight=weight, live=pack_bits(on.cpu()).cuda(), grad_queries=True, grad_rows=grad_rows)
    gx = torch.zeros(n, d, dtype=torch.float64, device="cuda")
    u, tiny = U[dtype], 2.0 ** -24 if dtype == "float16" else 0.0
    for r in range(0, m, 512):
        Q = q[r:r + 512].double()
        z = scale * Q @ X.T
        z[:, ~on] = -float("inf")
        lse = torch.logsumexp(z, 1)
        e0, e1 = int(t_off[r]), int(t_off[r + 512])
        t, k = t_idx[e0:e1].long(), torch.repeat_interleave(torch.arange(512, device="cuda"), count[r:r + 512])
        w = torch.zeros(512, n, dtype=torch.float64, device="cuda").index_put_((k, t), t_val[e0:e1].double(), accumulate=True)
        w[:, ~on] = 0
        W = w.sum(1)
        loss = W * lse - (w * torch.where(on, z, torch.zeros_like(z))).sum(1)
        p = torch.exp(z - lse[:, None])
        c = scale * weight[r:r + 512, None].double()
        mass = c * (W[:, None] * p + w)
        G = c * (W[:, None] * p - w)
        # |logit| < 50 or so: off by 0.5 * 20 * 2^-24 * 50 = 3e-5, p by twice that
        off = 2 * u + 6e-5 + (n + m) * 2.0 ** -24
        assert bool(((got["loss"][r:r + 512] - loss).abs() <= W * (6e-5 + 2.0 ** -20 * lse.abs()) + 6e-5 + 2.0 ** -20 * loss.abs()).all())
        assert bool(((got["lse"][r:r + 512] - lse).abs() <= 3e-5 + 2.0 ** -20 * lse.abs()).all())
        gq = G @ X
        tol = off * (mass @ X.abs()) + u * gq.abs() + 2.0 ** -24 * (dtype == "float16") + tiny * 2 * c * (W[:, None] + 3) * p.max(1, keepdim=True).values * X.abs().sum(0)
        assert bool(((got["grad_queries"][r:r + 512].double() - gq).abs() <= tol).all())
        gx += G.T.contiguous() @ Q
        del z, p, w, mass, G
    if grad_rows:
        assert not bool(got["grad_rows"][~on].any())
        err = float((got["grad_rows"].double() - gx).norm() / gx.norm())
        assert err < 2 * u + 6e-5, err


def test_gradients_against_differences(gpu_ctx):
    """Central differences of the kernel's own loss along random directions, float32. Truncation: the third derivative along a unit
    direction is at most (2 scale)^3 |W| a query; rounding: the losses' own error over the step."""
    import torch
    import apoe
    a = make(24, 300, 64, "float32", seed=12, scale=4.0)
    a["weight"] = None
    got = apoe.softmax_loss(gpu_ctx, **a, grad_queries=True, grad_rows=True)
    g = torch.Generator(device="cuda").manual_seed(3)
    step = 4e-3
    w1 = float(a["t_val"].sum())
    tol = (2 * a["scale"]) ** 3 * step ** 2 / 6 * w1 + 24 * 4 * 70 * 2.0 ** -24 * 3 / step
    for key, grad in (("queries", "grad_queries"), ("rows", "grad_rows")):
        for _ in range(4):
            v = torch.randn(a[key].shape, generator=g, device="cuda")
            v /= v.norm(dim=1, keepdim=True) * (1.0 if key == "queries" else 1.0)
            up = apoe.softmax_loss(gpu_ctx, **dict(a, **{key: a[key] + step * v}))["loss"].double().sum()
            down = apoe.softmax_loss(gpu_ctx, **dict(a, **{key: a[key] - step * v}))["loss"].double().sum()
            have = float((got[grad].double() * v.double()).sum())
            assert abs(float(up - down) / (2 * step) - have) <= tol, (key, float(up - down) / (2 * step), have, tol)


def test_same_bits_every_time(gpu_ctx):
    import apoe
    for grad_rows in (False, True):
        a = make(200, 3000, 128, "float16", seed=8, targets=5)
        first = apoe.softmax_loss(gpu_ctx, **a, grad_queries=True, grad_rows=grad_rows)
        for _ in range(3):
            again = apoe.softmax_loss(gpu_ctx, **a, grad_queries=True, grad_rows=grad_rows)
            for k in first:
                assert bool((first[k] == again[k]).all())


def test_rows_of_a_corpus(gpu_ctx, small_world):
    import torch
    import apoe
    corpus = apoe.Corpus(gpu_ctx, *small_world["corpus"])
    dense = torch.from_numpy(np.asarray(small_world["corpus"][0])).cuda()
    a = make(30, corpus.n, 1024, "float16", seed=2)
    with pytest.raises(apoe.ApoeError, match="half-precision rows"):
        apoe.softmax_loss(gpu_ctx, **dict(a, rows=corpus))
    corpus.make_half_rows()
    via = apoe.softmax_loss(gpu_ctx, **dict(a, rows=corpus), grad_queries=True)
    same = apoe.softmax_loss(gpu_ctx, **dict(a, rows=dense.half()), grad_queries=True)
    for k in same:
        assert bool((via[k] == same[k]).all())
    with pytest.raises(apoe.ApoeError, match="stay as they are"):
        apoe.softmax_loss(gpu_ctx, **dict(a, rows=corpus), grad_rows=True)
    corpus.close()


def test_streams(gpu_ctx):
    """Tensors that another stream is still writing, a context on a caller's stream, and no wait in between."""
    import torch
    import apoe
    a = make(100, 5000, 256, "bfloat16", seed=3)
    want = apoe.softmax_loss(gpu_ctx, **a, grad_queries=True)
    side = torch.cuda.Stream()
    mine = apoe.Context(0, stream=side)
    assert mine.stream == side.cuda_stream
    for ctx in (gpu_ctx, mine):
        for stream in (side, torch.cuda.Stream(), torch.cuda.default_stream()):
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                late = torch.zeros_like(a["queries"])
                for _ in range(20):
                    late += torch.ones_like(late)
                late.copy_(a["queries"])
                got = apoe.softmax_loss(ctx, **dict(a, queries=late), grad_queries=True)
                late.zero_()
                total = got["loss"].sum() + got["grad_queries"].float().sum()
            torch.cuda.synchronize()
            assert bool((got["loss"] == want["loss"]).all()) and bool((got["grad_queries"] == want["grad_queries"]).all())
            assert float(total) == float(want["loss"].sum() + want["grad_queries"].float().sum())
    mine.close()


@pytest.mark.parametrize("grad_rows", [False, True])
def test_in_a_graph(grad_rows):
    """Captured after one call of the same sizes, replayed on new inputs with eager work between."""
    import torch
    import apoe
    stream = torch.cuda.Stream()
    ctx = apoe.Context(0, stream=stream)
    inputs = [make(80, 900, 64, "float16", seed=s) for s in (1, 2, 3)]
    for i in inputs:  # one shape of the lists
        i["t_off"] = torch.arange(81, dtype=torch.int32, device="cuda")
        i["t_idx"] = torch.arange(80, dtype=torch.int32, device="cuda") * 3
        i["t_val"] = None
    held = {k: (v.clone() if torch.is_tensor(v) else v) for k, v in inputs[0].items()}
    with torch.cuda.stream(stream):
        apoe.softmax_loss(ctx, **held, grad_queries=True, grad_rows=grad_rows)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = apoe.softmax_loss(ctx, **held, grad_queries=True, grad_rows=grad_rows)
    for turn in range(2):
        for i in inputs:
            want = apoe.softmax_loss(ctx, **i, grad_queries=True, grad_rows=grad_rows)
            torch.cuda.synchronize()
            for k, v in i.items():
                if torch.is_tensor(v):
                    held[k].copy_(v)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for k in want:
                assert bool((out[k] == want[k]).all()), (turn, k)
    torch.cuda.synchronize()
    ctx.close()


def test_nothing_to_do(gpu_ctx):
    import torch
    import apoe
    a = make(4, 50, 32, "float32", seed=1)
    got = apoe.softmax_loss(gpu_ctx, a["queries"][:0], a["rows"], a["t_off"][:1], a["t_idx"][:0], grad_queries=True, grad_rows=True)
    assert got["loss"].shape == (0,) and got["grad_queries"].shape == (0, 32) and not bool(got["grad_rows"].any())
    got = apoe.softmax_loss(gpu_ctx, a["queries"], a["rows"], torch.zeros(5, dtype=torch.int32, device="cuda"), a["t_idx"][:0], grad_queries=True, grad_rows=True)
    assert not bool(got["loss"].any()) and not bool(got["grad_queries"].any()) and not bool(got["grad_rows"].any()) and bool(torch.isfinite(got["lse"]).all())


def test_refusals(gpu_ctx):
    import ctypes as C
    import torch
    import apoe
    a = make(6, 100, 64, "float16", seed=1)
    bad = [(dict(queries=a["queries"].float()), "float16|float32"), (dict(queries=a["queries"].cpu()), "on GPU"), (dict(queries=a["queries"].double()), "must be"),
           (dict(queries=a["queries"][:, :60]), "shape"), (dict(queries=a["queries"].T.contiguous().T), "contiguous"), (dict(scale=0.0), "scale"),
           (dict(scale=float("nan")), "scale"), (dict(scale=-1.0), "scale"), (dict(t_off=a["t_off"][:-1]), "t_off"), (dict(t_off=a["t_off"].long()), "t_off"),
           (dict(t_val=a["t_val"][:-1]), "t_val"), (dict(live=torch.zeros(3, dtype=torch.int32, device="cuda")), "live"), (dict(weight=a["weight"].double()), "weight"),
           (dict(rows=a["rows"][:0]), "empty"), (dict(queries=a["queries"][:, 1:57], rows=a["rows"][:, 1:57]), "aligned"),
           (dict(queries=a["queries"][:, :20], rows=a["rows"][:, :20]), "multiple"),
           (dict(grad_queries=a["queries"][:5]), "grad_queries"), (dict(grad_rows=a["rows"].float()), "grad_rows")]
    for change, words in bad:
        with pytest.raises(apoe.ApoeError, match=words):
            apoe.softmax_loss(gpu_ctx, **dict(a, **change))
    lib = apoe.lib()
    assert lib.apoe_softmax_loss(gpu_ctx.h, None) == -1
    args = apoe.SoftmaxLossArgs()
    args.dtype, args.n_queries, args.n_rows, args.dim, args.scale = 1, 4, 4, 64, 1.0
    args.q = a["queries"].data_ptr()
    assert lib.apoe_softmax_loss(gpu_ctx.h, C.byref(args)) == -1 and b"corpus" in lib.apoe_last_error_string()
    args.rows = a["rows"].data_ptr()
    assert lib.apoe_softmax_loss(gpu_ctx.h, C.byref(args)) == -1 and b"nothing to compute" in lib.apoe_last_error_string()
    args.loss = a["weight"].data_ptr()
    assert lib.apoe_softmax_loss(gpu_ctx.h, C.byref(args)) == -1 and b"t_off" in lib.apoe_last_error_string()
    for field, value, word in (("dtype", 7, b"dtype"), ("dim", 8192, b"dim"), ("n_rows", 1 << 30, b"row count"), ("q_stride", 32, b"stride"), ("rows_stride", 1 << 20, b"stride")):
        args2 = apoe.SoftmaxLossArgs.from_buffer_copy(args)
        args2.t_off = args2.t_idx = a["t_off"].data_ptr()
        setattr(args2, field, value)
        assert lib.apoe_softmax_loss(gpu_ctx.h, C.byref(args2)) == -1 and word in lib.apoe_last_error_string(), field
    host = np.zeros(4, np.float32)
    args.t_off = args.t_idx = a["t_off"].data_ptr()
    args.loss = host.ctypes.data
    assert lib.apoe_softmax_loss(gpu_ctx.h, C.byref(args)) == -1 and b"device memory" in lib.apoe_last_error_string()
