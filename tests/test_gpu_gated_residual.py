"""A block's norm, gate, residual scale, sum and the norm that follows, and the gradients, against the formula in 64 bits (needs
the GPU; the gradients of the formula by automatic differentiation, and by differences of the kernel's own result).

Tolerances. Everything between a read and a write is 32 bits: about ten operations a value, and sums over a row whose error is at most
dim 2^-24 of the sum of magnitudes but comes as that of a tree (dim / G values, then G threads): 40 2^-24 of the row's scale. Written
values are rounded once: u of the value. Sums over rows: (rows / workgroups + 40) 2^-24 of the sum of magnitudes."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
SMALL = {"float32": 0.0, "float16": 2.0 ** -25, "bfloat16": 0.0}  # half of the smallest number


def make(n, d, dtype, seed, gate="element", vectors=True, pad=0, grad_y=True, grad_u=True):
    import torch
    g = torch.Generator().manual_seed(seed)
    dt = getattr(torch, dtype)

    def mat(scale):
        t = (scale * torch.randn(n, d, generator=g)).to(dt)
        wide = torch.full((n, d + pad), float("nan"), dtype=dt)
        wide[:, :d] = t
        return wide.cuda()[:, :d]
    vec = lambda: (1 + 0.3 * torch.randn(d, generator=g)).cuda() if vectors else None  # noqa: E731
    a = dict(x=mat(1.0), h=mat(3.0), gate=None if gate == "none" else torch.randn(d, generator=g).to(dt).cuda() if gate == "channel" else mat(2.0),
             scale=vec(), w_post=vec(), w_next=vec(), eps=1e-5)
    grads = dict(grad_y=mat(1.0) if grad_y else None, grad_u=mat(1.0) if grad_u else None)
    return a, grads


def formula(a, grads=None):
    import torch
    names = [k for k in ("x", "h", "gate", "scale", "w_post", "w_next") if a[k] is not None]
    v = {k: a[k].detach().cpu().double().requires_grad_() for k in names}
    rms = lambda t: torch.sqrt(t.square().mean(-1, keepdim=True) + a["eps"])  # noqa: E731
    y = v["x"]
    if "h" in v:
        b = v["h"] / rms(v["h"])
        for k in ("scale", "w_post"):
            b = b * v[k] if k in v else b
        y = y + (b * torch.sigmoid(v["gate"]) if "gate" in v else b)
    u = y / rms(y)
    u = u * v["w_next"] if "w_next" in v else u
    out = dict(y=y.detach(), u=u.detach())
    if grads:
        aim = sum((t * grads[k].detach().cpu().double()).sum() for t, k in ((y, "grad_y"), (u, "grad_u")) if grads[k] is not None)
        for k, g in zip(names, torch.autograd.grad(aim, [v[k] for k in names], allow_unused=True)):
            if g is not None:
                out["grad_" + k] = g
        # the terms that the gradients of the norms are differences of (they cancel altogether where dim is 1)
        big = lambda k: v[k].detach().abs().max() if k in v else 1.0  # noqa: E731
        into = sum((g.detach().cpu().double().abs().amax(1, keepdim=True) if g.numel() else torch.zeros(g.shape[0], 1)) * f
                   for g, f in ((grads["grad_y"], 1.0), (grads["grad_u"], big("w_next") / rms(y).detach())) if g is not None)
        out["terms"] = dict(grad_x=into, grad_h=into * big("scale") * big("w_post") / rms(v["h"]).detach() if "h" in v else None)
    return out


def close(got, want, dtype, rows, name, terms=None):
    """Matrices: rounding of the value and of 32-bit work on the row's scale (its largest value, or that of the terms it is a
    difference of); vectors: sums over rows."""
    import torch
    got, want = got.detach().cpu().double(), want
    if want.dim() == 2:
        scale = want.abs().amax(1, keepdim=True) if want.numel() else want.abs()
        if terms and terms.get(name) is not None:
            scale = scale + terms[name]
        tol = U[dtype] * want.abs() + 100 * 2.0 ** -24 * scale + SMALL[dtype]
    else:
        # magnitudes of the terms: the sum's spread over rows is that of terms of size up to the largest total
        tol = (40 + rows / 64) * 2.0 ** -24 * rows ** 0.5 * max(1.0, float(want.abs().max())) + (U[dtype] if got.numel() and name == "grad_gate" else 0) * want.abs() + SMALL[dtype]
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), (name, float(((got - want).abs() / (tol + 1e-300)).max()), int(bad.sum()))


SIZES = [(1, 1), (1, 1024), (3, 33), (5, 256), (17, 257), (64, 1000), (130, 1024), (9, 1032), (700, 64), (6, 4096), (5, 4097), (3, 8192), (2, 8191)]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("n,d", SIZES)
def test_sizes_and_types(gpu_ctx, n, d, dtype):
    import apoe
    for gate, pad in (("element", 0), ("channel", 8), ("none", 3)):
        a, grads = make(n, d, dtype, n + d, gate, pad=pad)
        want = formula(a, grads)
        y, u = apoe.gated_residual(gpu_ctx, **a)
        got = apoe.gated_residual_grad(gpu_ctx, **a, **grads)
        terms = want.pop("terms")
        assert set(got) == {k for k in want if k.startswith("grad_")}
        for name, t in dict(got, y=y, u=u).items():
            close(t, want[name], dtype, n, name, terms)


@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_parts_of_the_operator(gpu_ctx, dtype):
    """Without vectors; one of the incoming gradients alone; no block at all; no norm behind."""
    import apoe
    for grad_y, grad_u in ((True, False), (False, True)):
        a, grads = make(40, 96, dtype, 3, vectors=False, grad_y=grad_y, grad_u=grad_u)
        want, got = formula(a, grads), apoe.gated_residual_grad(gpu_ctx, **a, **grads)
        assert set(got) == {"grad_x", "grad_h", "grad_gate"}
        for k in got:
            close(got[k], want[k], dtype, 40, k)
    a, grads = make(40, 96, dtype, 4, gate="none")
    a.update(h=None, scale=None, w_post=None)
    want = formula(a, grads)
    y, u = apoe.gated_residual(gpu_ctx, **a)
    assert y is a["x"]
    close(u, want["u"], dtype, 40, "u")
    got = apoe.gated_residual_grad(gpu_ctx, **a, **grads)
    assert set(got) == {"grad_x", "grad_w_next"}
    for k in got:
        close(got[k], want[k], dtype, 40, k)
    a, _ = make(40, 96, dtype, 5)
    y, u = apoe.gated_residual(gpu_ctx, **a, want_u=False)
    assert u is None
    close(y, formula(a)["y"], dtype, 40, "y")


def test_many_rows(gpu_ctx):
    """More rows than the gradient has workgroups, several a group; and the same bits every time."""
    import apoe
    a, grads = make(5003, 128, "bfloat16", 1, gate="channel")
    want, first = formula(a, grads), apoe.gated_residual_grad(gpu_ctx, **a, **grads)
    for k in first:
        close(first[k], want[k], "bfloat16", 5003, k)
    for _ in range(3):
        again = apoe.gated_residual_grad(gpu_ctx, **a, **grads)
        assert all(bool((again[k] == first[k]).all()) for k in first)


def test_unit_length(gpu_ctx):
    """eps = 0 and w_next = 1 / sqrt(dim): rows of length one, as the index wants its queries."""
    import torch
    import apoe
    a, _ = make(50, 1024, "float32", 2)
    a["w_next"] = torch.full((1024,), 1 / 32.0, device="cuda")
    _, u = apoe.gated_residual(gpu_ctx, **dict(a, eps=0.0))
    assert float((u.double().norm(dim=1) - 1).abs().max()) < 50 * 2.0 ** -24


def test_rows_of_zeros_and_values_that_are_not_finite_stay_in_their_rows(gpu_ctx):
    import torch
    import apoe
    a, grads = make(20, 64, "float32", 6)
    a["x"][3] = 0
    a["h"][3] = 0
    a["h"][4] = 0
    want = formula(a, grads)
    got = apoe.gated_residual_grad(gpu_ctx, **a, **grads)
    y, u = apoe.gated_residual(gpu_ctx, **a)
    for k, t in dict(got, y=y, u=u).items():
        close(t, want[k], "float32", 20, k)
    assert not bool(u[3].any())
    a["h"][7, 5] = float("nan")
    a["gate"][8] = float("inf")
    a["gate"][9] = -float("inf")
    y2, u2 = apoe.gated_residual(gpu_ctx, **a)
    rest = [i for i in range(20) if i not in (7, 8, 9)]
    assert bool((y2[rest] == y[rest]).all()) and bool((u2[rest] == u[rest]).all()) and bool(u2[7].isnan().any())
    assert bool((y2[9] == a["x"][9]).all())  # a gate that is shut
    assert bool(u2[8].isfinite().all())      # and one that is open
    got2 = apoe.gated_residual_grad(gpu_ctx, **a, **grads)
    assert all(bool((got2[k][rest] == got[k][rest]).all()) for k in ("grad_x", "grad_h", "grad_gate"))
    assert not bool(got2["grad_gate"][9].any()) and not bool(got2["grad_gate"][8].any())


def test_gradients_against_differences(gpu_ctx):
    """Central differences of the kernel's own y and u, float32. The step 2^-6 of inputs of size one leaves a truncation of about
    step^2 / 6 times third derivatives of a few units a value, summed over 30 x 40 terms with random signs, and a rounding of 2^-24 / step."""
    import torch
    import apoe
    a, grads = make(30, 40, "float32", 8, gate="channel")
    got = apoe.gated_residual_grad(gpu_ctx, **a, **grads)

    def aim(b):
        y, u = apoe.gated_residual(gpu_ctx, **b)
        return float((y.double() * grads["grad_y"].double()).sum() + (u.double() * grads["grad_u"].double()).sum())
    g = torch.Generator(device="cuda").manual_seed(1)
    step = 2.0 ** -6
    for key in ("x", "h", "gate", "scale", "w_post", "w_next"):
        v = torch.randn(a[key].shape, generator=g, device="cuda")
        v /= v.norm()  # of length one altogether: the third derivative along it is a few units
        want = (aim(dict(a, **{key: a[key] + step * v})) - aim(dict(a, **{key: a[key] - step * v}))) / (2 * step)
        have = float((got["grad_" + key].double() * v.double()).sum())
        assert abs(want - have) < step ** 2 / 6 * 30 + 1200 ** 0.5 * 8 * 2.0 ** -24 / step, (key, want, have)


def test_no_rows(gpu_ctx):
    import apoe
    a, grads = make(0, 64, "float16", 1, gate="channel")
    y, u = apoe.gated_residual(gpu_ctx, **a)
    assert y.shape == u.shape == (0, 64)
    got = apoe.gated_residual_grad(gpu_ctx, **a, **grads)
    assert not bool(got["grad_scale"].any()) and not bool(got["grad_gate"].any()) and got["grad_x"].shape == (0, 64)


def test_in_a_graph():
    import torch
    import apoe
    stream = torch.cuda.Stream()
    ctx = apoe.Context(0, stream=stream)
    sets = [make(70, 200, "float16", s) for s in (1, 2, 3)]
    held = [{k: (v.clone() if torch.is_tensor(v) else v) for k, v in part.items()} for part in sets[0]]
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        apoe.gated_residual_grad(ctx, **held[0], **held[1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        y, u = apoe.gated_residual(ctx, **held[0])
        out = dict(apoe.gated_residual_grad(ctx, **held[0], **held[1]), y=y, u=u)
    for _ in range(2):
        for a, grads in sets:
            y, u = apoe.gated_residual(ctx, **a)
            want = dict(apoe.gated_residual_grad(ctx, **a, **grads), y=y, u=u)
            torch.cuda.synchronize()
            for have, new in ((held[0], a), (held[1], grads)):
                for k, v in new.items():
                    if torch.is_tensor(v):
                        have[k].copy_(v)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for k in want:
                assert bool((out[k] == want[k]).all()), k
    ctx.close()


def test_refusals(gpu_ctx):
    import ctypes as C
    import torch
    import apoe
    a, grads = make(6, 32, "float16", 1)
    for change, words in ((dict(h=a["h"].float()), "h must be"), (dict(h=a["h"][:5]), "shape"), (dict(gate=a["gate"][:, :31]), "gate"), (dict(gate=a["gate"][0, :31]), "gate"),
                          (dict(scale=a["scale"].half()), "scale"), (dict(w_next=a["w_next"][:-1]), "w_next"), (dict(x=a["x"].cpu()), "on GPU"), (dict(eps=-1.0), "eps"),
                          (dict(eps=float("nan")), "eps"), (dict(h=None), "h is None"), (dict(x=a["x"].T), "contiguous")):
        with pytest.raises(apoe.ApoeError, match=words):
            apoe.gated_residual(gpu_ctx, **dict(a, **change))
        with pytest.raises(apoe.ApoeError, match=words):
            apoe.gated_residual_grad(gpu_ctx, **dict(a, **change), **grads)
    with pytest.raises(apoe.ApoeError, match="neither"):
        apoe.gated_residual_grad(gpu_ctx, **a)
    with pytest.raises(apoe.ApoeError, match="grad_u"):
        apoe.gated_residual_grad(gpu_ctx, **a, grad_u=grads["grad_u"][:5])
    wide = torch.zeros(2, 8200, device="cuda")
    with pytest.raises(apoe.ApoeError, match="dim must be"):
        apoe.gated_residual(gpu_ctx, wide)
    lib = apoe.lib()
    assert lib.apoe_gated_residual(gpu_ctx.h, None) == -1 and lib.apoe_gated_residual_grad(gpu_ctx.h, None) == -1
    r = apoe.GatedResidualArgs()
    r.dtype, r.rows, r.dim, r.eps = 1, 6, 32, 1e-6
    r.x = a["x"].data_ptr()
    assert lib.apoe_gated_residual(gpu_ctx.h, C.byref(r)) == -1 and b"nothing to compute" in lib.apoe_last_error_string()
    r.u = a["h"].data_ptr()
    for field, value, word in (("dtype", 5, b"dtype"), ("gate_kind", 3, b"gate"), ("gate_kind", 1, b"disagree"), ("x_stride", 31, b"overlap"), ("dim", 0, b"dim")):
        b = apoe.GatedResidualArgs.from_buffer_copy(r)
        setattr(b, field, value)
        assert lib.apoe_gated_residual(gpu_ctx.h, C.byref(b)) == -1 and word in lib.apoe_last_error_string(), field
    host = np.zeros(6 * 32, np.float16)
    r.u = host.ctypes.data
    assert lib.apoe_gated_residual(gpu_ctx.h, C.byref(r)) == -1 and b"device memory" in lib.apoe_last_error_string()
