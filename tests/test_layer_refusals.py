"""What embed, layer_norm, linear and AdamW refuse before any GPU work: a C program's missing or impossible arguments, and a Python program's tensors
that do not belong to the GPU."""
import ctypes as C
import types

import pytest
import torch

import apoe

CALLS = ("apoe_embed", "apoe_embed_grad", "apoe_layer_norm", "apoe_layer_norm_grad", "apoe_linear", "apoe_linear_grad")


def fake_context():
    """A place for a context whose fields are never looked at: every refusal here comes before that."""
    return C.create_string_buffer(4096)


def refused(name, args, match):
    lib = apoe.lib()
    assert getattr(lib, name)(fake_context(), C.byref(args)) == -1
    assert match in lib.apoe_last_error_string().decode(), lib.apoe_last_error_string()


@pytest.mark.parametrize("name", CALLS)
def test_no_context_and_no_arguments(name):
    lib = apoe.lib()
    assert getattr(lib, name)(None, None) == -1
    assert len(lib.apoe_last_error_string()) > 0


def test_sizes_of_the_argument_structures_match_the_header(tmp_path):
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = ["apoe_embed_args", "apoe_layer_norm_args", "apoe_linear_args", "apoe_adamw_tensor", "apoe_adamw_step_args"]
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "apoe.h"\nint main(void) { printf("' + " ".join(["%zu"] * len(names)) + '\\n", ' + ", ".join(f"sizeof({n})" for n in names) + "); return 0; }\n")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(root, "include"), str(src), "-o", str(tmp_path / "sizes")], check=True)
    out = subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True, text=True).stdout.split()
    assert [int(x) for x in out] == [C.sizeof(s) for s in (apoe.EmbedArgs, apoe.LayerNormArgs, apoe.LinearArgs, apoe.AdamwTensor, apoe.AdamwStepArgs)]


def test_embed():
    def args(**k):
        a = apoe.EmbedArgs()
        a.dtype, a.n_rows, a.n_table, a.n_entries, a.dim, a.scale = 1, 4, 10, 4, 64, 1.0
        for name, v in k.items():
            setattr(a, name, v)
        return a
    for name in ("apoe_embed", "apoe_embed_grad"):
        refused(name, args(dtype=3), "dtype")
        refused(name, args(dim=0), "dim")
        refused(name, args(dim=8193), "dim")
        refused(name, args(n_table=1 << 30), "table")
        refused(name, args(n_entries=1 << 27, off=16), "entries")
        refused(name, args(n_entries=5), "without off")
        refused(name, args(n_rows=0, off=16), "without rows")
        refused(name, args(scale=float("nan")), "scale")
        refused(name, args(table_stride=63), "stride")
    refused("apoe_embed", args(), "out")
    refused("apoe_embed", args(out=16), "table is null")
    refused("apoe_embed", args(out=16, table=16), "idx")
    refused("apoe_embed_grad", args(), "nothing")
    refused("apoe_embed_grad", args(grad_table=16), "grad is null")
    refused("apoe_embed_grad", args(grad_val=16, grad=16), "needs the table")
    refused("apoe_embed_grad", args(grad_val=16, grad=16, table=16, accumulate=1), "accumulate")


def test_layer_norm():
    def args(**k):
        a = apoe.LayerNormArgs()
        a.dtype, a.rows, a.dim, a.eps = 1, 4, 64, 1e-5
        for name, v in k.items():
            setattr(a, name, v)
        return a
    for name in ("apoe_layer_norm", "apoe_layer_norm_grad"):
        refused(name, args(dtype=3), "dtype")
        refused(name, args(dim=0), "dim")
        refused(name, args(dim=8193), "dim")
        refused(name, args(eps=-1.0), "eps")
        refused(name, args(x_stride=1), "stride")
    refused("apoe_layer_norm", args(), "y is null")
    refused("apoe_layer_norm", args(y=16), "x is null")
    refused("apoe_layer_norm_grad", args(), "nothing")
    refused("apoe_layer_norm_grad", args(grad_x=16), "grad_y")


def test_linear():
    def args(**k):
        a = apoe.LinearArgs()
        a.dtype, a.rows, a.cols_in, a.cols_out = 1, 4, 64, 32
        for name, v in k.items():
            setattr(a, name, v)
        return a
    for name in ("apoe_linear", "apoe_linear_grad"):
        refused(name, args(dtype=3), "dtype")
        refused(name, args(act=4), "activation")
        refused(name, args(cols_in=0), "columns")
        refused(name, args(cols_out=65537), "columns")
        refused(name, args(rows=1 << 30), "rows")
        refused(name, args(w_stride=63), "stride")
    refused("apoe_linear", args(x=16, w=16), "null")
    refused("apoe_linear_grad", args(), "nothing")
    refused("apoe_linear_grad", args(grad_x=16), "grad_y")
    refused("apoe_linear_grad", args(grad_x=16, grad_y=16), "w is null")
    refused("apoe_linear_grad", args(grad_bias=16, grad_y=16, act=2), "needs pre")


def test_adamw():
    lib, ctx, out = apoe.lib(), fake_context(), C.c_void_p()

    def create(tensors, bits=32):
        list_ = (apoe.AdamwTensor * len(tensors))(*tensors)
        st = lib.apoe_adamw_create(ctx, len(tensors), list_, bits, 0, C.byref(out))
        return st, lib.apoe_last_error_string().decode()

    def tensor(**k):
        t = apoe.AdamwTensor()
        t.n = 4
        for name, v in k.items():
            setattr(t, name, v)
        return t
    assert lib.apoe_adamw_create(None, 0, None, 32, 0, C.byref(out)) == -1
    assert lib.apoe_adamw_create(ctx, 1, None, 32, 0, C.byref(out)) == -1
    assert create([], 16)[0] == -1 and "bits" in create([], 16)[1]
    for bad, match in ((tensor(), "null"), (tensor(n=1 << 35), "beyond"), (tensor(decay=float("inf")), "decay"), (tensor(p=16, m=16, v=16, copy=16), "copy_dtype")):
        st, message = create([bad])
        assert st == -1 and match in message and not out.value, message
    st, message = create([tensor(p=16, m=16, v=16)], 8)
    assert st == -1 and "m_scale" in message
    assert lib.apoe_adamw_step(None, None) == -1
    assert create([])[0] == 0  # no parameters: nothing to do, and the rules for a step hold
    a = apoe.AdamwStepArgs()
    a.lr, a.beta1, a.beta2, a.eps, a.grad_scale, a.step = 1e-3, 0.9, 0.999, 1e-8, 1.0, 1
    for name, v, match in (("beta1", 1.0, "betas"), ("beta2", -0.1, "betas"), ("eps", -1.0, "eps"), ("lr", float("nan"), "finite"), ("step", 0, "counted")):
        keep = getattr(a, name)
        setattr(a, name, v)
        assert lib.apoe_adamw_step(out, C.byref(a)) == -1 and match in lib.apoe_last_error_string().decode()
        setattr(a, name, keep)
    lib.apoe_adamw_destroy(out)
    lib.apoe_adamw_destroy(None)
    assert lib.apoe_adamw_moments(None, 4, None, None, None, None, None, None) == -1


def test_host_tensors_are_refused_before_any_call():
    ctx = types.SimpleNamespace(device=0, h=None)  # a context's place, without a GPU
    x, w, idx = torch.zeros(4, 64, dtype=torch.float16), torch.zeros(8, 64, dtype=torch.float16), torch.zeros(4, dtype=torch.int32)
    for call in (lambda: apoe.embed(ctx, x, idx), lambda: apoe.embed_grad(ctx, x, x, idx), lambda: apoe.layer_norm(ctx, x), lambda: apoe.layer_norm_grad(ctx, x, grad_y=x),
                 lambda: apoe.linear(ctx, x, w), lambda: apoe.linear_grad(ctx, x, w, x), lambda: apoe.AdamW(ctx, [x.float()])):
        with pytest.raises(apoe.ApoeError):
            call()
