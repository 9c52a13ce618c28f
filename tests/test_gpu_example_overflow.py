"""The example's layer leaves a step out whose float16 gradients overflow, and goes on with a smaller loss scale (needs the GPU)."""
import pytest

from test_gpu_layers_together import adapter_of, example, world  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_whose_gradients_overflow(gpu_ctx, example, bits):  # noqa: F811
    import torch
    a = adapter_of(example, gpu_ctx, torch.float16, bits)
    x, terms, rows, t_off, t_idx = world(torch.float16)
    a.step(x, terms, rows, t_off, t_idx, 0.05, 1e-3)
    kept = {k: v.clone() for k, v in {**a.params, **{"copy of " + k: v for k, v in a.copies.items()}, **a.opt.state()}.items() if isinstance(v, torch.Tensor)}
    a.LOSS_SCALE = 2.0 ** 40
    assert not all(bool(torch.isfinite(g).all()) for g in a.gradients(x, terms, rows, t_off, t_idx, 0.05)[1].values())
    loss = a.step(x, terms, rows, t_off, t_idx, 0.05, 1e-3)
    assert bool(torch.isfinite(loss).all()) and a.LOSS_SCALE == 2.0 ** 39 and a.opt.t == 1
    now = {**a.params, **{"copy of " + k: v for k, v in a.copies.items()}, **a.opt.state()}
    for k, v in kept.items():
        assert bool((now[k] == v).all()), k
    for _ in range(40):
        a.step(x, terms, rows, t_off, t_idx, 0.05, 1e-3)
    assert 1.0 <= a.LOSS_SCALE < 2.0 ** 39 and a.opt.t > 1
    assert all(bool(torch.isfinite(p).all()) for p in a.params.values()) and all(bool(torch.isfinite(m).all()) for m in a.opt.moments())
