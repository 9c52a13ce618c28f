"""Outputs that begin where an input does and are written while others still read it: refused before anything runs (needs the GPU, whose memory is looked up)."""
import ctypes as C

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name,kind,fields", [
    ("apoe_embed", "EmbedArgs", dict(out="table")), ("apoe_embed_grad", "EmbedArgs", dict(grad_table="grad")),
    ("apoe_embed_grad", "EmbedArgs", dict(grad_table="table")), ("apoe_embed_grad", "EmbedArgs", dict(grad_val="val")),
    ("apoe_linear", "LinearArgs", dict(y="x")), ("apoe_linear", "LinearArgs", dict(y="w")), ("apoe_linear", "LinearArgs", dict(pre="x")),
    ("apoe_linear", "LinearArgs", dict(pre="y")), ("apoe_linear", "LinearArgs", dict(pre="residual")),
    ("apoe_linear_grad", "LinearArgs", dict(grad_x="grad_y")), ("apoe_linear_grad", "LinearArgs", dict(grad_x="x")), ("apoe_linear_grad", "LinearArgs", dict(grad_x="w")),
    ("apoe_linear_grad", "LinearArgs", dict(grad_w="w")), ("apoe_linear_grad", "LinearArgs", dict(grad_w="grad_y")), ("apoe_linear_grad", "LinearArgs", dict(grad_x="pre")),
    ("apoe_linear_grad", "LinearArgs", dict(grad_w="grad_x"))])
def test_refused(gpu_ctx, name, kind, fields):
    import torch
    import apoe
    a = getattr(apoe, kind)()
    store = torch.full((16, 4096), 7.0, device="cuda")  # a row for each array: 10 x 64 floats at most
    if kind == "EmbedArgs":
        a.dtype, a.n_rows, a.n_table, a.n_entries, a.dim, a.scale = 0, 4, 10, 4, 64, 1.0
        places = ("table", "idx", "val", "out", "grad", "grad_table", "grad_val")
    else:
        a.dtype, a.rows, a.cols_in, a.cols_out, a.act = 0, 4, 64, 64, 2
        places = ("x", "w", "residual", "y", "pre", "grad_y", "grad_x", "grad_w")
    for i, place in enumerate(places):
        setattr(a, place, store[i].data_ptr())
    for to, source in fields.items():
        setattr(a, to, getattr(a, source))
    torch.cuda.synchronize()
    lib = apoe.lib()
    assert getattr(lib, name)(gpu_ctx.h, C.byref(a)) == -1
    assert "the same memory" in lib.apoe_last_error_string().decode()
    gpu_ctx.synchronize()
    assert bool((store == 7).all())


def test_what_may_be_shared(gpu_ctx):
    """embed's out in base, layer_norm's in x, linear's y in its residual, and matrices side by side in one buffer."""
    import torch
    import apoe
    g = torch.Generator().manual_seed(1)
    wide, w = torch.randn(40, 128, generator=g).cuda(), torch.randn(64, 64, generator=g).cuda()
    x, y = wide[:, :64], wide[:, 64:]
    want = apoe.linear(gpu_ctx, x, w, residual=y)[0]
    normed = apoe.layer_norm(gpu_ctx, x)
    assert apoe.linear(gpu_ctx, x, w, residual=y, out=y)[0] is y and bool((y == want).all())
    assert bool((apoe.layer_norm(gpu_ctx, x, out=x) == normed).all())
    idx = torch.arange(40, dtype=torch.int32, device="cuda") % 64
    summed = apoe.embed(gpu_ctx, w, idx, base=y)
    assert bool((apoe.embed(gpu_ctx, w, idx, base=y, out=y) == summed).all())
