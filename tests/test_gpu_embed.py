"""Weighted sums of a table's rows, and the gradients of the table and of the weights, against 64 bits (needs the GPU).

Tolerances. A sum of c products in float32, in any order: (c + 3) 2^-24 of the sum of magnitudes (a product is joined to its sum without being rounded;
scale and base are an operation each); a written value half a step more. The table's gradient: the same over a row's entries, one operation more
for every block that a row's entries reach into. A weight's gradient: 16 products a thread, a tree over the threads: 30 2^-24 of the sum of
magnitudes."""
import pytest

from layer_cases import E, SMALL, TYPES, U, captured, close, matrix, room

pytestmark = pytest.mark.gpu


def entries(g, counts, n_table, weights=True, skew=False):
    import torch
    off = torch.zeros(len(counts) + 1, dtype=torch.int32)
    off[1:] = torch.cumsum(torch.tensor(counts), 0)
    total = int(off[-1])
    if skew:
        idx = (n_table ** torch.rand(total, generator=g, dtype=torch.float64)).long().sub(1).clamp(0, n_table - 1)
    else:
        idx = torch.randint(0, n_table, (total,), generator=g)
    val = (torch.rand(total, generator=g) * 2 - 0.5).cuda() if weights else None
    return off.cuda(), idx.to(torch.int32).cuda(), val


def formula(table, idx, off, val, scale, dtype, base=None, grad=None, had=None):
    import torch
    T, idx = table.detach().cpu().double(), idx.cpu().long()
    n = len(idx) if off is None else len(off) - 1
    row = torch.arange(n) if off is None else torch.repeat_interleave(torch.arange(n), (off[1:] - off[:-1]).cpu().long())
    w = torch.ones(len(idx), dtype=torch.float64) if val is None else val.cpu().double()
    on = idx < T.shape[0]
    row_on, idx_on, w_on = row[on], idx[on], w[on]
    d, u, small = T.shape[1], U[dtype], SMALL[dtype]

    def sums(where, k, values):
        return torch.zeros(k, d, dtype=torch.float64).index_add(0, where, values), torch.zeros(k, d, dtype=torch.float64).index_add(0, where, values.abs())
    count = torch.zeros(n, dtype=torch.float64).index_add(0, row, torch.ones(len(row), dtype=torch.float64))[:, None]
    s, size = sums(row_on, n, T[idx_on] * w_on[:, None])
    out = scale * s + (0 if base is None else base.detach().cpu().double())
    val_, tol = dict(out=out), dict(out=u * out.abs() + (count + 3) * E * abs(scale) * size + 2 * E * out.abs() + small)
    if grad is not None:
        G = grad.detach().cpu().double()
        named = torch.zeros(T.shape[0], dtype=torch.float64).index_add(0, idx_on, torch.ones(len(idx_on), dtype=torch.float64))[:, None]
        s, size = sums(idx_on, T.shape[0], G[row_on] * w_on[:, None])
        h = 0 if had is None else had.detach().cpu().double()
        gt = scale * s + h
        val_["grad_table"], tol["grad_table"] = gt, (u + 2 * E) * gt.abs() + (named * 33 / 32 + 6) * E * abs(scale) * size + small
        if had is not None:  # rows that no entry names are not touched
            tol["grad_table"] = torch.where(named > 0, tol["grad_table"], torch.zeros_like(gt))
        gv, size = torch.zeros(len(idx), dtype=torch.float64), torch.zeros(len(idx), dtype=torch.float64)
        gv[on], size[on] = scale * (G[row_on] * T[idx_on]).sum(1), abs(scale) * (G[row_on] * T[idx_on]).abs().sum(1)
        val_["grad_val"], tol["grad_val"] = gv, 30 * E * size + small
    return val_, tol


COUNTS = [[0], [1], [3], [0, 5, 0, 0, 1, 40, 2], [70] * 30, [0] * 50 + [200] + [1] * 50, [1] * 3000, [4] * 1500 + [0] * 100]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: f"{len(c)}x{max(c)}")
@pytest.mark.parametrize("n_table,d,pad", [(1, 8, 0), (300, 33, 3), (50, 1024, 8)])
def test_sizes_and_types(gpu_ctx, counts, n_table, d, pad, dtype):
    import torch
    import apoe
    g = torch.Generator().manual_seed(len(counts) + d)
    n = len(counts)
    off, idx, val = entries(g, counts, n_table)
    table, grad, base = matrix(g, n_table, d, dtype, 1.0, pad), matrix(g, n, d, dtype, 1.0, pad), matrix(g, n, d, dtype, 1.0, pad)
    had, untouched = room(n_table, d, dtype, pad=8)
    had.copy_(matrix(g, n_table, d, dtype))
    want, tol = formula(table, idx, off, val, 0.75, dtype, base, grad, had)
    out, outside = room(n, d, dtype, pad=8)
    apoe.embed(gpu_ctx, table, idx, off, val, 0.75, base, out=out)
    got = apoe.embed_grad(gpu_ctx, table, grad, idx, off, val, 0.75, grad_table=had, grad_val=True, accumulate=True)
    assert got["grad_table"] is had
    for k, t in dict(got, out=out).items():
        close(t, want[k], tol[k], k)
    assert outside() and untouched()
    want, tol = formula(table, idx, off, None, -2.0, dtype, None, grad)
    close(apoe.embed(gpu_ctx, table, idx, off, scale=-2.0), want["out"], tol["out"], "out")
    fresh, untouched = room(n_table, d, dtype)
    close(apoe.embed_grad(gpu_ctx, table, grad, idx, off, scale=-2.0, grad_table=fresh)["grad_table"], want["grad_table"], tol["grad_table"], "grad_table")
    assert untouched()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,n_table,d", [(1, 1, 1), (1, 5, 8192), (33, 7, 4097), (5000, 30_522, 64), (20_000, 70_000, 24), (9000, 300, 256), (4097, 255, 16), (4096, 256, 16), (12_000, 1 << 17, 8)])
def test_one_entry_a_row(gpu_ctx, n, n_table, d, dtype):
    """Tokens: no off, no weights; names as text has them, so that one is a tenth of all."""
    import torch
    import apoe
    g = torch.Generator().manual_seed(n)
    _, idx, _ = entries(g, [1] * n, n_table, False, skew=True)
    table, grad = matrix(g, n_table, d, dtype), matrix(g, n, d, dtype)
    want, tol = formula(table, idx, None, None, 8.0, dtype, None, grad)
    close(apoe.embed(gpu_ctx, table, idx, scale=8.0), want["out"], tol["out"], "out")
    got = apoe.embed_grad(gpu_ctx, table, grad, idx, scale=8.0)
    close(got["grad_table"], want["grad_table"], tol["grad_table"], "grad_table")


@pytest.mark.parametrize("n", [31, 32, 33, 64, 545, 20_000])
def test_every_entry_names_the_same_row(gpu_ctx, n):
    import torch
    import apoe
    g = torch.Generator().manual_seed(n)
    table, grad = matrix(g, 9, 300, "float32"), matrix(g, n, 300, "float32")
    idx = torch.full((n,), 4, dtype=torch.int32, device="cuda")
    want, tol = formula(table, idx, None, None, 1.0, "float32", None, grad)
    got = apoe.embed_grad(gpu_ctx, table, grad, idx)["grad_table"]
    close(got, want["grad_table"], tol["grad_table"])
    assert not bool(got[[0, 1, 2, 3, 5, 6, 7, 8]].any())


def test_names_outside_the_table_count_nothing(gpu_ctx):
    import torch
    import apoe
    g = torch.Generator().manual_seed(3)
    off, idx, val = entries(g, [5] * 100, 40)
    idx[::3] = 40
    idx[1::7] = -1     # as an unsigned number far beyond
    idx[4] = 1 << 30
    table, grad = matrix(g, 40, 72, "bfloat16"), matrix(g, 100, 72, "bfloat16")
    val[idx < 0] = float("nan")  # a weight that is not looked at
    safe = torch.where(idx < 0, torch.full_like(idx, 40), idx)
    clean = torch.where(idx < 0, torch.zeros_like(val), val)
    want, tol = formula(table, safe, off, clean, 1.0, "bfloat16", None, grad)
    close(apoe.embed(gpu_ctx, table, idx, off, val), want["out"], tol["out"], "out")
    got = apoe.embed_grad(gpu_ctx, table, grad, idx, off, val, grad_val=True)
    for k in got:
        close(got[k], want[k], tol[k], k)
    idx.fill_(-1)
    assert not bool(apoe.embed(gpu_ctx, table, idx, off).any())
    assert not bool(apoe.embed_grad(gpu_ctx, table, grad, idx, off)["grad_table"].any())


def test_nothing_there(gpu_ctx):
    import torch
    import apoe
    table, grad = torch.ones(6, 40, device="cuda"), torch.ones(3, 40, device="cuda")
    none, off = torch.empty(0, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    assert not bool(apoe.embed(gpu_ctx, table, none, off).any())
    assert bool((apoe.embed(gpu_ctx, table, none, off, base=grad) == 1).all())
    got = apoe.embed_grad(gpu_ctx, table, grad, none, off, grad_val=True)
    assert not bool(got["grad_table"].any()) and got["grad_val"].shape == (0,)
    had = table.clone()
    apoe.embed_grad(gpu_ctx, table, grad, none, off, grad_table=had, accumulate=True)
    assert bool((had == 1).all())
    assert apoe.embed(gpu_ctx, table, none).shape == (0, 40)
    assert not bool(apoe.embed_grad(gpu_ctx, table, grad[:0], none)["grad_table"].any())
    empty = table[:0]
    some = torch.zeros(3, dtype=torch.int32, device="cuda")
    assert not bool(apoe.embed(gpu_ctx, empty, some).any())
    got = apoe.embed_grad(gpu_ctx, empty, grad, some, grad_val=True)
    assert got["grad_table"].shape == (0, 40) and not bool(got["grad_val"].any())


def test_base_in_place(gpu_ctx):
    import torch
    import apoe
    g = torch.Generator().manual_seed(4)
    off, idx, val = entries(g, [9] * 500, 300)
    table, base = matrix(g, 300, 200, "float16"), matrix(g, 500, 200, "float16")
    want = apoe.embed(gpu_ctx, table, idx, off, val, base=base)
    apoe.embed(gpu_ctx, table, idx, off, val, base=base, out=base)
    assert bool((base == want).all())


def test_gradients_against_differences(gpu_ctx):
    """out is linear in the table and in the weights: the change along a direction is the gradient's product with it, up to rounding (2^-17 of
    the sum of magnitudes at some hundred terms)."""
    import torch
    import apoe
    g = torch.Generator().manual_seed(5)
    off, idx, val = entries(g, [6] * 80, 90)
    table, c = matrix(g, 90, 48, "float32"), matrix(g, 80, 48, "float32")
    grads = apoe.embed_grad(gpu_ctx, table, c, idx, off, val, 0.5, grad_val=True)
    at = apoe.embed(gpu_ctx, table, idx, off, val, 0.5).double()
    for name, t in (("grad_table", table), ("grad_val", val)):
        v = torch.randn(t.shape, generator=g).cuda()
        there = apoe.embed(gpu_ctx, *((t + v, idx, off, val) if name == "grad_table" else (table, idx, off, t + v)), 0.5).double()
        terms = (there - at) * c.double()
        assert abs(float(terms.sum()) - float((grads[name].double() * v.double()).sum())) <= 2.0 ** -17 * float((there.abs() * c.double().abs()).sum()), name


def test_the_same_bits_again_and_on_another_stream(gpu_ctx):
    import torch
    import apoe
    g = torch.Generator().manual_seed(6)
    off, idx, val = entries(g, [40] * 700, 1000, skew=True)
    table, grad = matrix(g, 1000, 264, "float32"), matrix(g, 700, 264, "float32")

    def call():
        return dict(apoe.embed_grad(gpu_ctx, table, grad, idx, off, val, grad_val=True), out=apoe.embed(gpu_ctx, table, idx, off, val))
    once = call()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = call()
    torch.cuda.current_stream().wait_stream(stream)
    for k in once:
        assert bool((once[k] == again[k]).all()), k


def test_captured():
    import torch
    import apoe
    g = torch.Generator().manual_seed(7)
    off, idx, val = entries(g, [20] * 300, 5000, skew=True)
    table, grad = matrix(g, 5000, 136, "bfloat16"), matrix(g, 300, 136, "bfloat16")

    def call(ctx):
        return dict(apoe.embed_grad(ctx, table, grad, idx, off, val, grad_val=True), out=apoe.embed(ctx, table, idx, off, val))
    ctx = apoe.Context(0, stream=torch.cuda.current_stream())
    want = call(ctx)
    for got in captured(lambda s: apoe.Context(0, stream=s), call):
        for k in want:
            assert bool((got[k] == want[k]).all()), k
    ctx.close()


def test_queries_of_the_index_as_they_are_stored(gpu_ctx, small_world):
    """The CSR of learned-sparse queries (the framework's own layout) goes in as it is."""
    import torch
    import apoe
    s_off, s_idx, s_val = (torch.from_numpy(a.astype(t)).cuda() for a, t in zip(small_world["queries"][1:4], ("int32", "int32", "float32")))
    g = torch.Generator().manual_seed(8)
    table = matrix(g, int(s_idx.max()) + 1, 128, "float16")
    want, tol = formula(table, s_idx, s_off, s_val, 0.1, "float16")
    close(apoe.embed(gpu_ctx, table, s_idx, s_off, s_val, 0.1), want["out"], tol["out"])


@pytest.mark.parametrize("n,n_table", [((1 << 20) + 4321, 1000), (70_000, (1 << 25) + 5)])
def test_many_entries_and_many_rows(gpu_ctx, n, n_table):
    """More entries than the sort's workgroups rank at a time, and names of 26 bits (four passes): numbers small enough that every sum is exact."""
    import torch
    import apoe
    g = torch.Generator(device="cuda").manual_seed(9)
    idx = torch.randint(0, n_table, (n,), generator=g, device="cuda")
    idx[: n // 3] %= 40
    grad = torch.randint(-3, 4, (n, 8), generator=g, device="cuda").to(torch.float32)
    table = torch.zeros(n_table, 8, device="cuda")
    want = torch.zeros(n_table, 8, device="cuda").index_add_(0, idx, grad)  # whole numbers below 2^24, in any order
    got = apoe.embed_grad(gpu_ctx, table, grad, idx.to(torch.int32))["grad_table"]
    assert bool((got == want).all())


def test_matrices_past_four_gigabytes(gpu_ctx):
    import torch
    import apoe
    g = torch.Generator().manual_seed(10)
    n, t, d, gap = 300, 40, 136, (1 << 31) // 39 + 5

    def far(m, gap):
        store = torch.empty((m.shape[0] - 1) * gap + m.shape[1], dtype=m.dtype, device="cuda")
        v = store.as_strided(m.shape, (gap, 1))
        v.copy_(m)
        assert m.shape[0] * gap * m.element_size() > 1 << 32
        return v
    table, grad, base = matrix(g, t, d, "float16"), matrix(g, n, d, "float16"), matrix(g, n, d, "float16")
    off, idx, val = entries(g, [4] * n, t)
    wide = far(table, gap)
    near = apoe.embed(gpu_ctx, table, idx, off, val, base=base)
    away = far(torch.zeros_like(base), (1 << 31) // 299 + 3)
    assert bool((apoe.embed(gpu_ctx, wide, idx, off, val, base=far(base, (1 << 31) // 299 + 1), out=away) == near).all())
    near = apoe.embed_grad(gpu_ctx, table, grad, idx, off, val, grad_val=True)
    wide_grad = far(torch.zeros_like(table), gap + 2)
    got = apoe.embed_grad(gpu_ctx, wide, far(grad, (1 << 31) // 299 + 7), idx, off, val, grad_table=wide_grad, grad_val=True)
    for k in near:
        assert bool(((got[k] - near[k]).abs() <= 2.0 ** -10 * near[k].abs() + 2.0 ** -24).all()), k  # rows that begin elsewhere are added up by other threads


@pytest.mark.parametrize("n", [50, 9000])
def test_rows_that_do_not_cover_all_entries(gpu_ctx, n):
    """A part of a batch's rows with all of its entries: those in front of the first row and behind the last one are no row's, and their weights' gradients are
    zeros; the rest is as if the entries had been cut too."""
    import torch
    import apoe
    g = torch.Generator().manual_seed(21)
    off = torch.arange(0, n + 1, 5, dtype=torch.int32).cuda()
    idx, val = torch.randint(0, 300, (n,), generator=g, dtype=torch.int32).cuda(), torch.randn(n, generator=g).cuda()
    table = matrix(g, 300, 40, "float32")
    rows = len(off) - 1
    for first, last in ((2, rows - 3), (0, 4), (rows - 1, rows), (rows, rows), (3, 3)):
        part = off[first:last + 1].contiguous()
        grad = matrix(g, last - first, 40, "float32")
        if first == last:  # entries and no row at all
            for call in (lambda: apoe.embed_grad(gpu_ctx, table, grad, idx, part, val, grad_val=True), lambda: apoe.embed_grad(gpu_ctx, table, grad, idx, part, val)):
                with pytest.raises(apoe.ApoeError, match="without rows"):
                    call()
            continue
        begin, end = int(part[0]), int(part[-1])
        alone = part - begin
        # what the result's memory held before: not zeros
        fill = torch.full((n,), 7.0, device="cuda")
        del fill
        got = apoe.embed_grad(gpu_ctx, table, grad, idx, part, val, grad_val=True)
        want = apoe.embed_grad(gpu_ctx, table, grad, idx[begin:end], alone, val[begin:end], grad_val=True)
        # how many threads share a row hangs on the number of entries: two orders of five additions
        a, b = apoe.embed(gpu_ctx, table, idx, part, val), apoe.embed(gpu_ctx, table, idx[begin:end], alone, val[begin:end])
        terms = apoe.embed(gpu_ctx, table.abs(), idx[begin:end], alone, val[begin:end].abs())
        close(a, b.double(), 2 * (5 + 4) * E * 1.01 * terms.double())
        assert bool((got["grad_val"][begin:end] == want["grad_val"]).all())
        assert not bool(got["grad_val"][:begin].any()) and not bool(got["grad_val"][end:].any())
        # the sums' parts are cut at other places: two orders of at most n additions
        size = torch.zeros(300, 40, device="cuda", dtype=torch.float64)
        row_of = torch.repeat_interleave(torch.arange(last - first, device="cuda"), (alone[1:] - alone[:-1]).long())
        size.index_add_(0, idx[begin:end].long(), (val[begin:end, None] * grad[row_of]).abs().double())
        close(got["grad_table"], want["grad_table"].double(), 2 * (end - begin + 4) * E * size)
