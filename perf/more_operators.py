"""The operators that a query adapter with a layer of its own, or a small encoder in front of an index, is built and trained from, through the
ctypes binding (`apoe.py`); they stand beside the loss, the orthogonalisation and the gated residual of `operators.py`.

  embed   weighted sums of a table's rows (terms of the learned-sparse path, tokens), and the gradients of table and weights
  norm    layer norm of rows, and its gradients
  linear  matrix product with bias, activation and residual, and its gradients
  adamw   one AdamW step over all parameters, moments in 32 bits or in 8

The plain forms are elementary torch operations in 32 bits (rounding the moments to 8 bits: 64), rounded once at the end.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5
BLOCK = 256            # moments in 8 bits: values that share a scale
BETAS, ADAM_EPS, LR = (0.9, 0.999), 1e-8, 1e-3

_ctx = None


# ---- cases ----

def embed_case(name, rows, table, dtype, dim=1024, terms=1, base=False, grad=True, grad_val=False, accumulate=False, pad=0):
    """terms: entries of a row on average (1: exactly one, without weights); pad: elements between the rows of each matrix."""
    c = dict(op="embed", rows=rows, table=table, dtype=dtype, dim=dim, terms=terms, base=base, grad=grad, grad_val=grad_val, accumulate=accumulate, pad=pad)
    return dict(name=name, **c) if name else c


def norm_case(name, rows, dtype, dim=1024, grad=True, skip=False, pad=0):
    c = dict(op="norm", rows=rows, dtype=dtype, dim=dim, grad=grad, skip=skip, pad=pad)
    return dict(name=name, **c) if name else c


def linear_case(name, rows, cols_in, cols_out, dtype, act="none", bias=True, residual=False, grad=True, pad=0):
    c = dict(op="linear", rows=rows, cols_in=cols_in, cols_out=cols_out, dtype=dtype, act=act, bias=bias, residual=residual, grad=grad, pad=pad)
    return dict(name=name, **c) if name else c


def adamw_case(name, layers, width, bits, grad="bf16", copy="bf16", table=0, pad=0):
    """layers: blocks of the parameters that a two-layer MLP with its norm has at this width; table: rows of a table beside them;
    pad: elements by which the parameters begin behind a boundary."""
    c = dict(op="adamw", layers=layers, width=width, bits=bits, grad=grad, copy=copy, table=table, pad=pad)
    return dict(name=name, **c) if name else c


def listed():
    return [
        # the learned-sparse terms of a small serving batch, added to its dense queries on their way to the search
        embed_case("embed_32q_serve", 32, 30_522, "f16", terms=40, base=True, grad=False),
        # training queries as weighted terms in full precision; the term weights learn too, and the table has a gradient from the loss already
        embed_case("embed_777q_f32", 777, 30_522, "f32", terms=40, grad_val=True, accumulate=True, pad=4),
        # the tokens of a batch of passages, forward and back
        embed_case("embed_65k_tokens", 65_536, 30_522, "bf16"),
        # queries of a small serving batch
        norm_case("norm_64_serve", 64, "f16", grad=False),
        # a training step's queries in full precision
        norm_case("norm_10007_f32", 10_007, "f32", pad=4),
        # the tokens of a batch of passages, forward and back, with the gradient that comes past the block
        norm_case("norm_65k", 65_536, "bf16", skip=True),
        # a small serving batch through the first layer of an adapter's block
        linear_case("linear_16_serve", 16, 1024, 4096, "f16", act="gelu", grad=False),
        # odd sizes at full precision, forward and back
        linear_case("linear_777x1001_f32", 777, 1001, 999, "f32", act="silu", residual=True),
        # the two layers of an adapter's block under a large batch
        linear_case("linear_8192_up", 8192, 1024, 4096, "bf16", act="gelu"),
        linear_case("linear_8192_down", 8192, 4096, 1024, "bf16", residual=True, pad=64),
        # the parameters of one adapter's block, masters and moments in full precision
        adamw_case("adamw_block", 1, 1024, 32, grad="f16", copy="f16"),
        # an encoder of twelve layers with its term table, moments in 8 bits
        adamw_case("adamw_encoder_8bit", 12, 1024, 8, table=30_522),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("embed", "norm", "linear", "linear", "adamw"))
    dtype = rng.choice(("f16", "bf16", "f32"))
    pad = rng.choice((0, 0, 8, 64))
    if op == "embed":
        terms = rng.choice((1, 1, 7, 40))
        dim = 1024 if rng.random() < 0.5 else _log_int(rng, 32, 2048)
        return embed_case(None, _log_int(rng, 1, (1 << 25) // (dim * min(terms, 8))), _log_int(rng, 50, 30_522), dtype, dim=dim, terms=terms, base=rng.random() < 0.3,
                          grad=rng.random() < 0.7, grad_val=terms > 1 and rng.random() < 0.5, accumulate=rng.random() < 0.4, pad=pad)
    if op == "norm":
        dim = 1024 if rng.random() < 0.5 else _log_int(rng, 32, 4096)
        return norm_case(None, _log_int(rng, 1, (1 << 26) // dim), dtype, dim=dim, grad=rng.random() < 0.7, skip=rng.random() < 0.5, pad=pad)
    if op == "linear":
        k, n = _log_int(rng, 32, 4096), _log_int(rng, 32, 4096)
        if rng.random() < 0.7:  # most layers have whole sides
            k, n = -(-k // 64) * 64, -(-n // 64) * 64
        most = min(65_536, (1 << 35) // (k * n) // (8 if dtype == "f32" else 1))
        return linear_case(None, _log_int(rng, 1, most), k, n, dtype, act=rng.choice(("none", "relu", "gelu", "silu")), bias=rng.random() < 0.7,
                           residual=rng.random() < 0.4, grad=rng.random() < 0.6, pad=pad)
    return adamw_case(None, rng.randint(1, 8), _log_int(rng, 32, 1024), rng.choice((8, 32)), grad=dtype, copy=rng.choice(("none", "f16", "bf16")),
                      table=rng.choice((0, _log_int(rng, 50, 30_522))), pad=rng.choice((0, 0, 1)))


# ---- what a program has in hand ----

def _context():
    global _ctx
    if _ctx is None:
        sys.path.insert(1, os.path.join(os.getcwd(), "allan-poe_amd"))
        import apoe
        _ctx = apoe.Context(0, stream=torch.cuda.current_stream())
    return _ctx


def _strided(t, pad):
    """`t` with `pad` elements between its rows."""
    if not pad:
        return t.contiguous()
    wide = torch.empty(*t.shape[:-1], t.shape[-1] + pad, dtype=t.dtype, device=t.device)
    wide[..., t.shape[-1]:] = 1.0
    view = wide[..., :t.shape[-1]]
    view.copy_(t)
    return view


def adamw_sizes(case):
    """(number of values, weight decay) of each parameter: an MLP's matrices decay, vectors do not."""
    w = case["width"]
    layer = [(4 * w * w, 0.1), (4 * w, 0.0), (4 * w * w, 0.1), (w, 0.0), (w, 0.0), (w, 0.0)]
    return ([(case["table"] * w, 0.01)] if case["table"] else []) + layer * case["layers"]


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, generator=g, device=DEV)  # noqa: E731
    state = dict(case=case)
    if own:
        state["ctx"] = _context()
    if case["op"] == "adamw":
        _prepare_adamw(state, g, rand)
        return state
    dt, pad = TYPES[case["dtype"]], case["pad"]
    put = lambda t: _strided(t.to(dt), pad)  # noqa: E731
    n = case["rows"]
    if case["op"] == "embed":
        t, d = case["table"], case["dim"]
        if case["terms"] == 1:
            off, total, val = None, n, None
        else:
            total = n * case["terms"]
            off = torch.full((n + 1,), total, dtype=torch.int32, device=DEV)
            off[0] = 0
            off[1:n] = torch.randint(0, total + 1, (n - 1,), generator=g, device=DEV).sort().values.to(torch.int32)  # some queries are empty, some long
            val = torch.rand(total, generator=g, device=DEV) * 2.0
        # terms as text has them: the r-th most frequent about 1 / r as often
        idx = torch.exp(torch.rand(total, generator=g, device=DEV, dtype=torch.float64) * math.log(t)).long().sub_(1).clamp_(0, t - 1)
        state.update(table=put(rand(t, d) / math.sqrt(d)), idx=idx.to(torch.int32), off=off, val=val, base=put(rand(n, d) / math.sqrt(d)) if case["base"] else None,
                     scale=0.125 if case["terms"] > 1 else math.sqrt(d))
        if case["grad"]:
            state.update(grad=put(1e-2 * rand(n, d)), had=put(1e-2 * rand(t, d)) if case["accumulate"] else None)
    elif case["op"] == "norm":
        d = case["dim"]
        x = rand(n, d) * (0.5 + torch.rand(n, 1, generator=g, device=DEV)) + 0.3 * rand(n, 1)
        state.update(x=put(x), w=1.0 + 0.1 * rand(d), b=0.1 * rand(d))
        if case["grad"]:
            state.update(grad=put(1e-2 * rand(n, d)), skip=put(1e-2 * rand(n, d)) if case["skip"] else None)
    else:
        k, c = case["cols_in"], case["cols_out"]
        state.update(x=put(rand(n, k)), w=put(rand(c, k) / math.sqrt(k)), bias=0.1 * rand(c) if case["bias"] else None, residual=put(rand(n, c)) if case["residual"] else None)
        if case["grad"]:
            state.update(grad=put(1e-2 * rand(n, c)))
            if case["act"] != "none":  # kept by the forward call of the same step: as it was rounded there
                z = state["x"].float() @ state["w"].float().T
                state.update(pre=put(z if state["bias"] is None else z + state["bias"]))
    return state


def _prepare_adamw(state, g, rand):
    """Parameters, gradients and moments each in one buffer, every parameter at a block's beginning; what lies between them stays as it is."""
    case = state["case"]
    sizes = adamw_sizes(case)
    blocks = [-(-n // BLOCK) for n, _ in sizes]
    first = [sum(blocks[:i]) for i in range(len(sizes))]
    total, pad = sum(blocks) * BLOCK, case["pad"]
    count = torch.tensor(blocks, device=DEV)
    tensor = torch.repeat_interleave(torch.arange(len(sizes), device=DEV), count)                      # of each block
    inside = torch.arange(len(tensor), device=DEV) - torch.tensor(first, device=DEV)[tensor]           # its number in there
    used = (inside[:, None] * BLOCK + torch.arange(BLOCK, device=DEV)) < torch.tensor([n for n, _ in sizes], device=DEV)[tensor][:, None]
    flat = lambda t: torch.cat((torch.zeros(pad, dtype=t.dtype, device=DEV), t))[pad:]                 # noqa: E731
    spread = torch.exp(1.5 * rand(total))                                                              # gradients differ in size by orders of magnitude
    grads = flat((1e-3 * rand(total) * spread).to(TYPES[case["grad"]]))
    m, v = 3e-4 * rand(total) * spread * used.reshape(-1), 1e-6 * spread * spread * (0.5 + torch.rand(total, generator=g, device=DEV)) * used.reshape(-1)
    params = flat(0.03 * rand(total))
    copy = None if case["copy"] == "none" else flat(torch.zeros(total, dtype=TYPES[case["copy"]], device=DEV))
    if case["bits"] == 8:
        mb, vb = m.view(-1, BLOCK), v.view(-1, BLOCK)
        ms, vs = mb.abs().amax(1), vb.amax(1)
        codes = (torch.sign(mb) * torch.round(127 * (mb.abs() / ms[:, None]).sqrt())).to(torch.int8).reshape(-1)
        roots = torch.round(255 * (vb / vs[:, None]).sqrt().sqrt()).clamp_(min=1).mul_(used).to(torch.uint8).reshape(-1)
        moments = dict(m=codes, v=roots, m_scale=ms, v_scale=vs)
    else:
        moments = dict(m=m, v=v)
    state.update(params=params, grads=grads, copy=copy, moments=moments, t=100, seed=1234, tensor=tensor, inside=inside, used=used,
                 decay=torch.tensor([d for _, d in sizes], device=DEV)[tensor][:, None])
    if own:
        import apoe
        at = [f * BLOCK for f in first]
        view = lambda t: [t[a:a + n] for a, (n, _) in zip(at, sizes)]  # noqa: E731
        state["views"] = view(grads)
        state["opt"] = apoe.AdamW(state["ctx"], view(params), copies=None if copy is None else view(copy), bits=case["bits"], betas=BETAS, eps=ADAM_EPS,
                                  weight_decay=[d for _, d in sizes], seed=state["seed"], state=dict(moments, t=state["t"]))


# ---- one pass ----

def run(state):
    op = state["case"]["op"]
    if own:
        return {"embed": _own_embed, "norm": _own_norm, "linear": _own_linear, "adamw": _own_adamw}[op](state)
    return {"embed": _plain_embed, "norm": _plain_norm, "linear": _plain_linear, "adamw": _plain_adamw}[op](state)


def _own_embed(s):
    import apoe
    c = s["case"]
    out = dict(out=apoe.embed(s["ctx"], s["table"], s["idx"], off=s["off"], val=s["val"], scale=s["scale"], base=s["base"]))
    if c["grad"]:
        out.update(apoe.embed_grad(s["ctx"], s["table"], s["grad"], s["idx"], off=s["off"], val=s["val"], scale=s["scale"], grad_val=c["grad_val"],
                                   grad_table=s["had"] if c["accumulate"] else True, accumulate=c["accumulate"]))
    return out


def _own_norm(s):
    import apoe
    out = dict(y=apoe.layer_norm(s["ctx"], s["x"], s["w"], s["b"], eps=EPS))
    if s["case"]["grad"]:
        out.update(apoe.layer_norm_grad(s["ctx"], s["x"], s["w"], s["b"], eps=EPS, grad_y=s["grad"], grad_skip=s["skip"]))
    return out


def _own_linear(s):
    import apoe
    c = s["case"]
    y, pre = apoe.linear(s["ctx"], s["x"], s["w"], s["bias"], act=c["act"], residual=s["residual"], want_pre=c["grad"] and c["act"] != "none")
    out = dict(y=y)
    if c["grad"]:
        out.update(apoe.linear_grad(s["ctx"], s["x"], s["w"], s["grad"], act=c["act"], pre=s.get("pre"), grad_bias=c["bias"]))
        if pre is not None:
            out["pre"] = pre
    return out


def _own_adamw(s):
    s["opt"].step(s["views"], LR, grad_scale=0.5)
    m, v = s["opt"].moments()
    return dict(params=s["params"], copy=s["copy"], m=m, v=v) if s["copy"] is not None else dict(params=s["params"], m=m, v=v)


def _plain_embed(s):
    c, n, d = s["case"], s["case"]["rows"], s["case"]["dim"]
    dt, t = s["table"].dtype, s["idx"].long()
    which = torch.arange(n, device=DEV) if s["off"] is None else \
        torch.repeat_interleave(torch.arange(n, device=DEV), (s["off"][1:] - s["off"][:-1]).long(), output_size=t.numel())
    rows = s["table"][t].float()
    weighted = rows if s["val"] is None else rows * s["val"][:, None]
    y = torch.zeros(n, d, device=DEV).index_add_(0, which, weighted) * s["scale"]
    if s["base"] is not None:
        y = y + s["base"].float()
    out = dict(out=y.to(dt))
    if c["grad"]:
        g = s["grad"].float()[which]
        if c["grad_val"]:
            out["grad_val"] = (rows * g).sum(1) * s["scale"]
        if s["val"] is not None:
            g = g * s["val"][:, None]
        gt = torch.zeros(c["table"], d, device=DEV).index_add_(0, t, g) * s["scale"]
        out["grad_table"] = s["had"].copy_(gt + s["had"].float()) if c["accumulate"] else gt.to(dt)
    return out


def _plain_norm(s):
    x, dt = s["x"].float(), s["x"].dtype
    x = x - x.mean(1, keepdim=True)
    r = torch.rsqrt((x * x).mean(1, keepdim=True) + EPS)
    xn = x * r
    out = dict(y=(xn * s["w"] + s["b"]).to(dt))
    if s["case"]["grad"]:
        g = s["grad"].float()
        out["grad_w"], out["grad_b"] = (g * xn).sum(0), g.sum(0)
        g = g * s["w"]
        gx = r * (g - g.mean(1, keepdim=True) - xn * (g * xn).mean(1, keepdim=True))
        out["grad_x"] = (gx if s["skip"] is None else gx + s["skip"].float()).to(dt)
    return out


def _act(z, act):
    if act == "relu":
        return z.clamp_min(0.0)
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z * torch.sigmoid(z) if act == "silu" else z


def _slope(z, act):
    if act == "relu":
        return (z > 0).float()
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    o = torch.sigmoid(z)
    return o * (1.0 + z * (1.0 - o))


def _plain_linear(s):
    c, dt = s["case"], s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.T
    if s["bias"] is not None:
        z = z + s["bias"]
    y = _act(z, c["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = dict(y=y.to(dt))
    if c["grad"]:
        gz = s["grad"].float()
        if c["act"] != "none":
            out["pre"] = z.to(dt)
            gz = gz * _slope(s["pre"].float(), c["act"])
        out["grad_x"], out["grad_w"] = (gz @ w).to(dt), (gz.T @ x).to(dt)
        if c["bias"]:
            out["grad_bias"] = gz.sum(0)
    return out


WORD = 0xFFFFFFFF


def _mix(h):
    """A 32-bit number's bits mixed (in 64-bit integers): shifts and odd multipliers."""
    h = ((h ^ (h >> 16)) * 0x85EBCA6B) & WORD
    h = ((h ^ (h >> 13)) * 0xC2B2AE35) & WORD
    return h ^ (h >> 16)


def _chances(s, which):
    """A number between 0 and 1 for every value of every block, for the first (0) or the second (1) moment."""
    key = _mix(_mix(_mix(torch.tensor(s["seed"], device=DEV)) ^ s["t"]) ^ s["tensor"])
    block = _mix(_mix(key ^ (s["inside"] & WORD)) ^ (s["inside"] >> 32))
    at = torch.arange(BLOCK, device=DEV)
    return (_mix((block[:, None] + 2 * at + which) & WORD).double() + 0.5) / 2 ** 32


def _rounded(x, top, power, steps, chance):
    """Codes of x >= 0: x = top (code / steps)^power, up or down by chance so that x is the mean."""
    w = (x / top[:, None].double() * float(steps ** power)).nan_to_num(0.0).clamp_(max=float(steps ** power))
    low = torch.floor(w.pow(1.0 / power))
    low -= (low ** power > w).double()
    low += ((low + 1) ** power <= w).double()
    up = chance < (w - low ** power) / ((low + 1) ** power - low ** power)
    return (low + up.double()).clamp_(max=steps)


def _plain_adamw(s):
    c = s["case"]
    s["t"] += 1
    used, t, wide = s["used"], s["t"], c["bits"] == 8
    p, g = s["params"].view(-1, BLOCK), s["grads"].view(-1, BLOCK).float() * 0.5
    mom = s["moments"]
    if wide:
        cm, cv = mom["m"].view(-1, BLOCK).double(), mom["v"].view(-1, BLOCK).double()
        m, v = mom["m_scale"][:, None].double() * (cm * cm.abs() / 127.0 ** 2), mom["v_scale"][:, None].double() * (cv ** 4 / 255.0 ** 4)
        g = g.double()
    else:
        m, v = mom["m"].view(-1, BLOCK), mom["v"].view(-1, BLOCK)
    m = (m + (1 - BETAS[0]) * (g - m)) * used
    v = (v + (1 - BETAS[1]) * (g * g - v)) * used
    step = (m / (1 - BETAS[0] ** t) / (torch.sqrt(v / (1 - BETAS[1] ** t)) + ADAM_EPS)).float()
    p.copy_(torch.where(used, p - LR * (s["decay"] * p + step), p))
    if s["copy"] is not None:
        s["copy"].view(-1, BLOCK).copy_(torch.where(used, p.to(s["copy"].dtype), s["copy"].view(-1, BLOCK)))
    if wide:
        ms, vs = m.abs().amax(1).float(), v.amax(1).float()
        cm = _rounded(m.abs(), ms, 2, 127, _chances(s, 0)) * torch.sign(m)
        cv = torch.maximum(_rounded(v, vs, 4, 255, _chances(s, 1)), (v > 0).double())
        mom["m"].view(-1, BLOCK).copy_(cm)
        mom["v"].view(-1, BLOCK).copy_(cv)
        mom["m_scale"].copy_(ms)
        mom["v_scale"].copy_(vs)
        out = dict(m=(ms[:, None].double() * (cm * cm.abs() / 127.0 ** 2)).float().view(-1), v=(vs[:, None].double() * (cv ** 4 / 255.0 ** 4)).float().view(-1))
    else:
        mom["m"].copy_(m.view(-1))
        mom["v"].copy_(v.view(-1))
        out = dict(m=mom["m"], v=mom["v"])
    out["params"] = s["params"]
    if s["copy"] is not None:
        out["copy"] = s["copy"]
    return out


# ---- what a pass cannot do without ----

def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2, "none": 0}
    if case["op"] == "adamw":
        n = sum(c for c, _ in adamw_sizes(case))
        moments = 16 if case["bits"] == 32 else 4 + 16 / BLOCK + 8  # with the values that the codes stand for, written once
        return {"bytes": n * (8 + moments + size[case["grad"]] + size[case["copy"]]), "flops": 15.0 * n}
    e, n = size[case["dtype"]], case["rows"]
    if case["op"] == "embed":
        t, d, entries = case["table"], case["dim"], n * case["terms"]
        named = sum(1.0 - math.exp(-entries * math.log((r + 1) / r) / math.log(t)) for r in range(1, t))  # rows that are named at least once
        move = e * d * (named + n * (1 + case["base"])) + entries * (4 + 4 * (case["terms"] > 1))
        flops = 2.0 * entries * d
        if case["grad"]:
            move += e * d * (n + t * (1 + case["accumulate"])) + 4 * entries * case["grad_val"]
            flops *= 2 + case["grad_val"]
        return {"bytes": move, "flops": flops}
    if case["op"] == "norm":
        d = case["dim"]
        move, flops = 2 * n * d * e + 8 * d, 8.0 * n * d
        if case["grad"]:
            move += (2 + case["skip"]) * n * d * e + 8 * d
            flops += 16.0 * n * d
        return {"bytes": move, "flops": flops}
    k, c = case["cols_in"], case["cols_out"]
    move, flops = e * (n * k + c * k + n * c * (1 + case["residual"])) + 4 * c * case["bias"], 2.0 * n * k * c
    if case["grad"]:
        move += e * (n * c * (1 + (case["act"] != "none")) + n * k + c * k) + 4 * c * case["bias"]
        flops *= 3
    return {"bytes": move, "flops": flops}


# ---- the same in 64 bits, from the definitions ----

def exact(case, seed):
    s = prepare(case, seed)
    return {"embed": _exact_embed, "norm": _exact_norm, "linear": _exact_linear, "adamw": _exact_adamw}[case["op"]](case, s)


def _exact_embed(case, s):
    """The matrix of weights that entries make, times the table; its gradients by the two transposed products, a slice of columns at a time."""
    n, t, d = case["rows"], case["table"], case["dim"]
    off = torch.arange(n + 1, device=DEV) if s["off"] is None else s["off"].long()
    entries = torch.arange(s["idx"].numel(), device=DEV)
    row = torch.searchsorted(off, entries, right=True) - 1
    col = s["idx"].long()
    val = torch.ones(col.numel(), dtype=torch.float64, device=DEV) if s["val"] is None else s["val"].double()
    out, grad_table, grad_val = torch.empty(n, d, dtype=torch.float64, device=DEV), None, None
    if case["grad"]:
        grad_table = torch.empty(t, d, dtype=torch.float64, device=DEV)
        grad_val = torch.zeros(col.numel(), dtype=torch.float64, device=DEV) if case["grad_val"] else None
    for a in range(0, d, 64):
        z = min(d, a + 64)
        table = s["table"][:, a:z].double()
        part = torch.zeros(n, z - a, dtype=torch.float64, device=DEV).index_add_(0, row, table[col] * val[:, None])
        out[:, a:z] = s["scale"] * part + (s["base"][:, a:z].double() if case["base"] else 0)
        if case["grad"]:
            up = s["scale"] * s["grad"][:, a:z].double()[row]
            grad_table[:, a:z] = (s["had"][:, a:z].double() if case["accumulate"] else 0) + torch.zeros(t, z - a, dtype=torch.float64, device=DEV).index_add_(0, col, up * val[:, None])
            if grad_val is not None:
                grad_val += (up * table[col]).sum(1)
    found = dict(out=out)
    if case["grad"]:
        found["grad_table"] = grad_table
        if grad_val is not None:
            found["grad_val"] = grad_val
    return found


def _exact_norm(case, s):
    """The forward pass in 64 bits; its gradients by automatic differentiation of that."""
    x, w, b = (s[k].double().requires_grad_(case["grad"]) for k in ("x", "w", "b"))
    var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
    y = (x - mean) / torch.sqrt(var + EPS) * w + b
    out = dict(y=y.detach())
    if case["grad"]:
        gx, out["grad_w"], out["grad_b"] = torch.autograd.grad((y * s["grad"].double()).sum(), (x, w, b))
        out["grad_x"] = gx if s["skip"] is None else gx + s["skip"].double()
    return out


def _exact_linear(case, s):
    x, w = s["x"].double(), s["w"].double()
    z = torch.mm(x, w.t().contiguous())
    if s["bias"] is not None:
        z += s["bias"].double()
    act = case["act"]
    zz = z.detach().requires_grad_(True)
    a = zz * 0.5 * torch.erfc(-zz / math.sqrt(2.0)) if act == "gelu" else zz / (1 + torch.exp(-zz)) if act == "silu" else torch.where(zz > 0, zz, torch.zeros_like(zz)) if act == "relu" else zz
    out = dict(y=a.detach() + (s["residual"].double() if case["residual"] else 0))
    if case["grad"]:
        if act != "none":
            out["pre"] = z
            kept = s["pre"].double().requires_grad_(True)
            a = kept * 0.5 * torch.erfc(-kept / math.sqrt(2.0)) if act == "gelu" else kept / (1 + torch.exp(-kept)) if act == "silu" else torch.where(kept > 0, kept, torch.zeros_like(kept))
            gz, = torch.autograd.grad((a * s["grad"].double()).sum(), kept)
        else:
            gz = s["grad"].double()
        out["grad_x"], out["grad_w"] = torch.mm(gz, w), torch.mm(gz.t().contiguous(), x)
        if case["bias"]:
            out["grad_bias"] = gz.sum(0)
    return out


def _exact_adamw(case, s):
    """Value by value on the parameters' own range; codes by search in the list of all values that a block can hold."""
    t, used = s["t"] + 1, s["used"].reshape(-1)
    s["t"] = t
    b1, b2 = (torch.tensor(b, dtype=torch.float64, device=DEV) for b in BETAS)
    block = torch.arange(used.numel(), device=DEV) // BLOCK
    at, block = torch.nonzero(used).reshape(-1), block[used]
    mom = s["moments"]
    squares, fourth = (torch.arange(128, device=DEV).double() / 127) ** 2, (torch.arange(256, device=DEV).double() / 255) ** 4
    if case["bits"] == 8:
        c = mom["m"][at].long()
        m, v = mom["m_scale"][block].double() * squares[c.abs()] * c.sign(), mom["v_scale"][block].double() * fourth[mom["v"][at].long()]
    else:
        m, v = mom["m"][at].double(), mom["v"][at].double()
    g = s["grads"][at].double() / 2
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g ** 2
    p = s["params"][at].double()
    p = p * (1 - LR * s["decay"].reshape(-1)[block].double()) - LR * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)) ** 0.5 + ADAM_EPS)
    out = dict(params=s["params"].double().index_copy_(0, at, p))
    if s["copy"] is not None:
        out["copy"] = s["copy"].double().index_copy_(0, at, p)
    for name, x, list_, which in (("m", m, squares, 0), ("v", v, fourth, 1)):
        if case["bits"] == 8:
            top = torch.zeros(s["tensor"].numel(), dtype=torch.float64, device=DEV).index_reduce_(0, block, x.abs(), "amax").float().double()[block]
            share = (x.abs() / top).clamp(max=1.0)
            low = (torch.searchsorted(list_, share, right=True) - 1).clamp(0, len(list_) - 2)
            up = _chances(s, which).reshape(-1)[at] < (share - list_[low]) / (list_[low + 1] - list_[low])
            code = low + up
            if which:
                code = torch.where(x > 0, code.clamp(min=1), code)
            x = top * list_[code] * x.sign()
        out[name] = torch.zeros(used.numel(), dtype=torch.float64, device=DEV).index_copy_(0, at, x)
    return out
