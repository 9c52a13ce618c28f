"""Embed and its gradients at rows wider than a wave holds: groups of 256 and 512 threads, alone and several to a row (needs the GPU). Tolerances: those of
test_gpu_embed.py, whose weights' gradient counts 16 products a thread, six steps of a tree in a wave and up to eight waves."""
import pytest

from layer_cases import TYPES, close, matrix, room
from test_gpu_embed import entries, formula

pytestmark = pytest.mark.gpu

COUNTS = [[70] * 5, [0, 5, 0, 1, 200, 3], [1] * 700, [2] * 40 + [0] + [9] * 30]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: f"{len(c)}x{max(c)}")
@pytest.mark.parametrize("d,pad", [(1025, 0), (2048, 8), (4096, 0), (4097, 3), (8185, 1), (8192, 0)])
def test_csr_rows(gpu_ctx, counts, d, pad, dtype):
    import torch
    import apoe
    n, n_table = len(counts), 60
    g = torch.Generator().manual_seed(n + d)
    off, idx, val = entries(g, counts, n_table, skew=True)
    table, grad, base = matrix(g, n_table, d, dtype, 1.0, pad), matrix(g, n, d, dtype, 1.0, pad), matrix(g, n, d, dtype, 1.0, pad)
    had, untouched = room(n_table, d, dtype, pad=8)
    had.copy_(matrix(g, n_table, d, dtype))
    want, tol = formula(table, idx, off, val, 0.75, dtype, base, grad, had)
    out, outside = room(n, d, dtype, pad=8)
    got = dict(out=apoe.embed(gpu_ctx, table, idx, off, val, 0.75, base, out=out))
    fresh = apoe.embed_grad(gpu_ctx, table, grad, idx, off, val, 0.75, grad_table=False, grad_val=True)["grad_val"]
    got.update(apoe.embed_grad(gpu_ctx, table, grad, idx, off, val, 0.75, grad_table=had, grad_val=True, accumulate=True))
    assert bool((fresh == got["grad_val"]).all())
    for k, t in got.items():
        close(t, want[k], tol[k], k)
    assert outside() and untouched()
    new, untouched = room(n_table, d, dtype)
    want, tol = formula(table, idx, off, val, 0.75, dtype, None, grad)
    close(apoe.embed_grad(gpu_ctx, table, grad, idx, off, val, 0.75, grad_table=new)["grad_table"], want["grad_table"], tol["grad_table"], "grad_table")
    assert untouched()
