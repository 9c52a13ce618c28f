"""Batches for the orthogonalisation that are not matrices one after the other (needs the GPU)."""
import pytest

from test_gpu_orthogonalize import matrix

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,cols", [(5, 40), (70, 90)])
def test_a_repeated_matrix_is_refused(gpu_ctx, rows, cols):
    """A batch that is one matrix repeated (stride 0) does not lie in memory as so many matrices: neither read nor written as if it did."""
    import torch
    import apoe
    x = matrix(rows, cols, "float32", 1)
    both = torch.stack([x, x, x])
    for call in (lambda: apoe.orthogonalize(gpu_ctx, x.expand(3, rows, cols)), lambda: apoe.orthogonalize(gpu_ctx, both, out=torch.empty_like(x).expand(3, rows, cols)),
                 lambda: apoe.orthogonalize(gpu_ctx, both, out=torch.empty(5 * rows, cols, device="cuda").as_strided((3, rows, cols), (rows * cols - 1, cols, 1)))):
        with pytest.raises(apoe.ApoeError, match="overlap"):
            call()
    one = apoe.orthogonalize(gpu_ctx, x)
    for got in (apoe.orthogonalize(gpu_ctx, x.expand(1, rows, cols)), apoe.orthogonalize(gpu_ctx, both)):
        assert all(bool((g == one).all()) for g in got)


@pytest.mark.parametrize("rows,cols", [(5, 40), (70, 90)])
def test_matrices_in_any_distance(gpu_ctx, rows, cols):
    """Every second one of a batch, the last of them at the end of its memory; and one of a batch of none."""
    import torch
    import apoe
    x = matrix(rows, cols, "float32", 2, batch=5)
    want = torch.stack([apoe.orthogonalize(gpu_ctx, x[i]) for i in (0, 2, 4)])
    assert bool((apoe.orthogonalize(gpu_ctx, x[::2]) == want).all())
    assert apoe.orthogonalize(gpu_ctx, x[:0]).shape == (0, rows, cols)
