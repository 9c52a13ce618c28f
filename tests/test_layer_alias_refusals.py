"""Outputs that begin where an input does while others still read it, or where another output does: refused by embed, layer_norm, linear and AdamW before any GPU work."""
import ctypes as C

import pytest

import apoe


def status(name, kind, sizes, places, same):
    """The call's status and message with every array at an address of its own, but for `same`: pairs of fields (the first at the second's address) and strides."""
    lib, a = apoe.lib(), getattr(apoe, kind)()
    for k, v in sizes.items():
        setattr(a, k, v)
    for i, place in enumerate(places):
        setattr(a, place, 4096 * (i + 1))
    for k, v in same.items():
        setattr(a, k, getattr(a, v) if isinstance(v, str) else v)
    # a place for a context: device -1 owns no memory, so that a call that is not refused for its aliases is refused for its addresses
    ctx = C.create_string_buffer(b"\xff" * 4096, 4096)
    st = getattr(lib, name)(ctx, C.byref(a))
    return st, lib.apoe_last_error_string().decode()


NORM = ("LayerNormArgs", dict(dtype=1, rows=4, dim=64, eps=1e-5))
EMBED = ("EmbedArgs", dict(dtype=0, n_rows=4, n_table=10, n_entries=4, dim=64, scale=1.0))
LINEAR = ("LinearArgs", dict(dtype=0, rows=4, cols_in=64, cols_out=64, act=2))
FORWARD = dict(apoe_layer_norm=(*NORM, ("x", "w", "b", "y")), apoe_embed=(*EMBED, ("table", "idx", "off", "val", "base", "out")),
               apoe_linear=(*LINEAR, ("x", "w", "bias", "residual", "y", "pre")))
BACK = dict(apoe_layer_norm_grad=(*NORM, ("x", "w", "grad_y", "grad_skip", "grad_x", "grad_w", "grad_b")),
            apoe_embed_grad=(*EMBED, ("table", "idx", "off", "val", "grad", "grad_table", "grad_val")),
            apoe_linear_grad=(*LINEAR, ("x", "w", "pre", "grad_y", "grad_x", "grad_w", "grad_bias")))
CALLS = {**FORWARD, **BACK}


@pytest.mark.parametrize("name,same", [
    ("apoe_layer_norm", dict(y="x", x_stride=128)), ("apoe_layer_norm", dict(y="x", y_stride=65)),
    ("apoe_layer_norm_grad", dict(grad_x="grad_y", grad_y_stride=128)), ("apoe_layer_norm_grad", dict(grad_x="grad_skip", grad_x_stride=72)),
    ("apoe_layer_norm_grad", dict(grad_x="x", x_stride=100)),
    ("apoe_embed", dict(out="base", base_stride=128)), ("apoe_embed", dict(out="base", out_stride=64, base_stride=65)),
    ("apoe_linear", dict(y="residual", residual_stride=128)), ("apoe_linear", dict(y="residual", y_stride=65))])
def test_in_place_with_other_strides(name, same):
    """With one address and two strides a row of the output lies on rows of the input that others still read."""
    st, message = status(name, *CALLS[name], same)
    assert st == -1 and "the same memory" in message, message


@pytest.mark.parametrize("name,same", [
    ("apoe_layer_norm", dict(y="x")), ("apoe_layer_norm", dict(y="x", x_stride=128, y_stride=128)), ("apoe_layer_norm", dict(y="x", x_stride=64)),
    ("apoe_layer_norm", dict(y="x", x_stride=128, rows=1)),
    ("apoe_layer_norm_grad", dict(grad_x="grad_y")), ("apoe_layer_norm_grad", dict(grad_x="grad_skip")), ("apoe_layer_norm_grad", dict(grad_x="x")),
    ("apoe_embed", dict(out="base")), ("apoe_linear", dict(y="residual")), ("apoe_linear", dict(y="residual", y_stride=128, rows=1))])
def test_what_may_be_in_place(name, same):
    """These go on to the check of the addresses."""
    st, message = status(name, *CALLS[name], same)
    assert st == -1 and "device memory" in message, message


@pytest.mark.parametrize("name,same", [
    ("apoe_layer_norm", dict(y="w")), ("apoe_layer_norm", dict(y="b")), ("apoe_layer_norm_grad", dict(grad_x="w")), ("apoe_layer_norm_grad", dict(grad_w="grad_x")),
    ("apoe_layer_norm_grad", dict(grad_b="grad_x")), ("apoe_layer_norm_grad", dict(grad_w="grad_b")),
    ("apoe_embed", dict(out="idx")), ("apoe_embed", dict(out="off")), ("apoe_embed", dict(out="val")),
    ("apoe_embed_grad", dict(grad_val="idx")), ("apoe_embed_grad", dict(grad_val="off")), ("apoe_embed_grad", dict(grad_val="table")),
    ("apoe_embed_grad", dict(grad_val="grad")), ("apoe_embed_grad", dict(grad_val="grad_table")),
    ("apoe_linear", dict(y="bias")), ("apoe_linear", dict(pre="bias")),
    *(("apoe_linear_grad", dict(grad_bias=k)) for k in ("x", "w", "pre", "grad_y", "grad_x", "grad_w"))])
def test_vectors_too(name, same):
    """A vector that others still read, or two outputs at one place."""
    st, message = status(name, *CALLS[name], same)
    assert st == -1 and "the same memory" in message, message


@pytest.mark.parametrize("name,same", [("apoe_layer_norm_grad", dict(grad_w="w", grad_b="x")), ("apoe_linear_grad", dict(grad_bias="pre", act=0))])
def test_what_is_not_read_any_more(name, same):
    """The norm's vectors are added up behind the launch that reads its inputs; without an activation pre is not read."""
    st, message = status(name, *CALLS[name], same)
    assert st == -1 and "device memory" in message, message


@pytest.mark.parametrize("to", [4, 5])
@pytest.mark.parametrize("source", [0, 1, 2, 3, 9])
def test_moments_that_are_read_back(to, source):
    """Of m, m_scale, v, v_scale and both results, each result at another's address (9: at the other result's)."""
    lib, p = apoe.lib(), [4096 * (i + 1) for i in range(6)]
    p[to] = p[9 - to if source == 9 else source]
    assert lib.apoe_adamw_moments(C.create_string_buffer(b"\xff" * 4096, 4096), C.c_uint64(512), *(C.c_void_p(x) for x in p)) == -1
    assert "the same memory" in lib.apoe_last_error_string().decode()
