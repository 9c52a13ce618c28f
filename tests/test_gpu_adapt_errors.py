"""What a failed call leaves behind (needs the GPU)."""
import pytest

pytestmark = pytest.mark.gpu


def test_a_call_that_found_no_memory_is_not_reported_by_the_next():
    """8 M rows against a million queries: the groups' sums alone are twice 256 GiB, which the allocation refuses. A smaller call after it works, and
    so does any other operator of the context."""
    import torch
    import apoe
    ctx = apoe.Context(0, stream=torch.cuda.current_stream())
    m, n, d = (1 << 20) - 1, 1 << 23, 8
    q, x = torch.zeros(m, d, dtype=torch.float16, device="cuda"), torch.zeros(n, d, dtype=torch.float16, device="cuda")
    off, idx = torch.zeros(m + 1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    assert 2 * n // 128 * m * 4 > torch.cuda.get_device_properties(0).total_memory
    for _ in range(2):
        with pytest.raises(apoe.ApoeError, match="memory"):
            apoe.softmax_loss(ctx, q, x, off, idx)
        got = apoe.softmax_loss(ctx, q[:70], x[:200], off[:71], idx, grad_queries=True)
        assert float((got["lse"] - torch.log(torch.tensor(200.0, device="cuda"))).abs().max()) < 1e-5
        with pytest.raises(apoe.ApoeError, match="memory"):
            apoe.softmax_loss(ctx, q, x, off, idx)
        assert not bool(apoe.orthogonalize(ctx, torch.zeros(70, 80, device="cuda")).any())
        with pytest.raises(apoe.ApoeError, match="memory"):
            apoe.softmax_loss(ctx, q, x, off, idx)
        y, u = apoe.gated_residual(ctx, torch.ones(3, 16, device="cuda"))
        assert float((u - 1).abs().max()) < 1e-5
    ctx.close()
