"""What linear and its gradient answer at the edges of their numbers (needs the GPU)."""
import pytest

from layer_cases import TYPES, matrix

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
def test_relu_lets_nothing_back_where_pre_is_nan(gpu_ctx, dtype):
    """A NaN in pre is not above zero: whatever grad_y is there, all gradients are as if it were zero."""
    import torch
    import apoe
    g = torch.Generator().manual_seed(1)
    x, w, gy, pre = matrix(g, 70, 40, dtype), matrix(g, 24, 40, dtype), matrix(g, 70, 24, dtype), matrix(g, 70, 24, dtype)
    pre[3, 5] = pre[40, 23] = pre[69, 0] = float("nan")
    gy[3, 5] = gy[40, 23] = gy[69, 0] = 0.0
    want = apoe.linear_grad(gpu_ctx, x, w, gy, act="relu", pre=pre)
    gy[3, 5], gy[40, 23], gy[69, 0] = 1.0, float("nan"), float("-inf")
    got = apoe.linear_grad(gpu_ctx, x, w, gy, act="relu", pre=pre)
    for k in want:
        assert bool(torch.isfinite(want[k]).all()) and bool((got[k] == want[k]).all()), k
