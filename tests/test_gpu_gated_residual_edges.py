"""The gated residual where its parts are nearly nothing (needs the GPU): gates that are all but open, calls without rows."""
import ctypes as C

import pytest

from test_gpu_gated_residual import close, formula, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["element", "channel"])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("d", [40, 1024])
def test_gates_that_are_all_but_open(gpu_ctx, dtype, kind, d):
    """What is left of a gate at 10 to 14 is 1 - sigmoid = 1e-6 to 5e-5, and its gradient is as right as any other's. The incoming gradients
    are large, so that the gradient of a channel's gate is above one, the size that its tolerance is relative to."""
    import apoe
    a, grads = make(60, d, dtype, d, kind)
    a["gate"] = a["gate"].abs() * 0.5 + 10.0
    for k in grads:
        grads[k] = grads[k] * 2.0 ** 10
    if dtype == "float32":
        for k in grads:
            grads[k] = grads[k] * 2.0 ** 8
    want = formula(a, grads)
    got = apoe.gated_residual_grad(gpu_ctx, **a, **grads)
    for k in got:
        close(got[k], want[k], dtype, 60, k, want["terms"])


@pytest.mark.parametrize("kind", ["none", "channel"])
def test_no_rows_in_a_call_from_c(kind):
    """The vectors' gradients of no rows are zeros, on a context that has no workspace yet too."""
    import apoe
    import torch
    ctx = apoe.Context(0, stream=torch.cuda.current_stream())
    d = 72
    r = apoe.GatedResidualArgs()
    r.dtype, r.rows, r.dim, r.eps = 1, 0, d, 1e-6
    row = torch.ones(1, d, dtype=torch.float16, device="cuda")
    r.x = r.h = r.grad_y = r.grad_u = row.data_ptr()
    out = {k: torch.full((d,), 7.0, device="cuda") for k in ("grad_scale", "grad_w_post", "grad_w_next")}
    for k, t in out.items():
        setattr(r, k, t.data_ptr())
    if kind == "channel":
        gate = torch.ones(d, dtype=torch.float16, device="cuda")
        out["grad_gate"] = torch.full((d,), 7.0, dtype=torch.float16, device="cuda")
        r.gate_kind, r.gate, r.grad_gate = 2, gate.data_ptr(), out["grad_gate"].data_ptr()
    assert apoe.lib().apoe_gated_residual_grad(ctx.h, C.byref(r)) == 0, apoe.lib().apoe_last_error_string()
    ctx.synchronize()
    for k, t in out.items():
        assert not bool(t.any()), k
    ctx.close()
