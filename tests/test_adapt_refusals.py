"""What the query adapter's calls refuse before any GPU work: a C program without a context or without arguments, and a Python
program with tensors that do not belong to the GPU (there is no CPU path to fall back to)."""
import types

import pytest
import torch

import apoe

CALLS = ("apoe_softmax_loss", "apoe_orthogonalize", "apoe_gated_residual", "apoe_gated_residual_grad")


@pytest.mark.parametrize("name", CALLS)
def test_no_context_and_no_arguments(name):
    lib = apoe.lib()
    assert getattr(lib, name)(None, None) == -1
    assert len(lib.apoe_last_error_string()) > 0


def test_no_place_for_a_context():
    lib = apoe.lib()
    assert lib.apoe_ctx_create_on_stream(0, None, None) == -1
    assert lib.apoe_ctx_stream(None, None) == -1


def test_sizes_of_the_argument_structures_match_the_header(tmp_path):
    """The binding passes these by address: a field that is missing or of another size would shift all that follow."""
    import ctypes
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "apoe.h"\nint main(void) { printf("%zu %zu %zu\\n", sizeof(apoe_softmax_loss_args),'
                   ' sizeof(apoe_orthogonalize_args), sizeof(apoe_gated_residual_args)); return 0; }\n')
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(root, "include"), str(src), "-o", str(tmp_path / "sizes")], check=True)
    out = subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True, text=True).stdout.split()
    assert [int(x) for x in out] == [ctypes.sizeof(s) for s in (apoe.SoftmaxLossArgs, apoe.OrthogonalizeArgs, apoe.GatedResidualArgs)]


def test_host_tensors_are_refused_before_any_call():
    ctx = types.SimpleNamespace(device=0, handle=None)  # a context's place, without a GPU
    x = torch.zeros(4, 64, dtype=torch.float16)
    for call in (lambda: apoe.gated_residual(ctx, x, x), lambda: apoe.gated_residual_grad(ctx, x, x, grad_u=x),
                 lambda: apoe.orthogonalize(ctx, x), lambda: apoe.softmax_loss(ctx, x, x, None, None)):
        with pytest.raises(apoe.ApoeError):
            call()
