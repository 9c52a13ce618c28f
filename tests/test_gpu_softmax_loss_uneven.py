"""The softmax loss on inputs of very uneven sizes (needs the GPU): rows of zeros between others. Against the formula in 64 bits;
tolerances as in test_gpu_softmax_loss.py."""
import pytest

from test_gpu_softmax_loss import check, make

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
