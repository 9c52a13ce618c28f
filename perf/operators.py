"""The operators that fit a query adapter to a stored index, through the ctypes binding (`apoe.py`): a few learned rows
and matrices move the queries, the documents and their graph stay as they are.

  loss      softmax cross entropy of queries over the rows of a corpus (or of any table: passages of a batch, terms of a
            vocabulary), without keeping the logits, with its gradients
  ortho     a matrix gradient made (nearly) orthogonal by Newton-Schulz products
  residual  norm of a block's output, its gate and residual scale, the sum, and the norm that follows, with gradients

The plain forms are elementary torch operations in 32 bits, rounded once at the end.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
COEFS = (3.4445, -4.7750, 2.0315)   # of the quintic, over all steps
STEPS = 5
EPS = 1e-6

_ctx = None


# ---- cases ----

def loss_case(name, queries, rows, dtype, dim=1024, grad_queries=True, grad_rows=False, live=1.0, targets=1, pad=0, scale=30.0):
    """live: share of the rows that a mask leaves (1: no mask); targets: the largest number of relevant rows a query has;
    pad: elements between the rows of each matrix."""
    c = dict(op="loss", queries=queries, rows=rows, dtype=dtype, dim=dim, grad_queries=grad_queries, grad_rows=grad_rows, live=live,
             targets=targets, pad=pad, scale=scale)
    return dict(name=name, **c) if name else c


def ortho_case(name, batch, rows, cols, dtype, pad=0):
    c = dict(op="ortho", batch=batch, rows=rows, cols=cols, dtype=dtype, pad=pad)
    return dict(name=name, **c) if name else c


def residual_case(name, rows, dtype, dim=1024, gate="element", grad=True, grad_y=False, pad=0):
    c = dict(op="residual", rows=rows, dtype=dtype, dim=dim, gate=gate, grad=grad, grad_y=grad_y, pad=pad)
    return dict(name=name, **c) if name else c


def listed():
    return [
        # one click of one user against a small index, learned from at once: the time to the query's gradient
        loss_case("loss_1q_4k", 1, 4000, "f16", scale=20.0),
        # relevance of a validation set on part of an index (the rest is deleted), no gradient, at the rows' full precision
        loss_case("loss_777q_100k_live", 777, 99_991, "f32", grad_queries=False, live=0.7, targets=3),
        # queries and passages of one batch, every other passage a negative; both encoders learn
        loss_case("loss_batch_4096", 4096, 4096, "bf16", grad_rows=True, scale=20.0),
        # the term table of the learned-sparse path under a batch of token vectors, both learn
        loss_case("loss_vocab_2048", 2048, 30_522, "bf16", grad_rows=True, pad=64),
        # an adapter's step against a whole index of a million documents, which stays
        loss_case("loss_1024q_1m", 1024, 1_000_000, "f16", targets=3),
        # the gradient of the adapter's matrix
        ortho_case("ortho_1024", 1, 1024, 1024, "bf16"),
        # an odd matrix at full precision
        ortho_case("ortho_777x1001_f32", 1, 777, 1001, "f32"),
        # wide layers of an encoder that is trained with the index, four at a time
        ortho_case("ortho_4x1024x4096", 4, 1024, 4096, "bf16"),
        ortho_case("ortho_4096", 1, 4096, 4096, "bf16", pad=64),
        # queries of a small serving batch on their way to the search
        residual_case("residual_64_serve", 64, "f16", grad=False),
        # a training step's queries in full precision, one gate value for each channel
        residual_case("residual_10007_f32", 10_007, "f32", gate="channel", pad=4),
        # rows of a corpus that is encoded again, forward and back
        residual_case("residual_65k", 65_536, "bf16", grad_y=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("loss", "loss", "ortho", "residual"))
    if op == "loss":
        dtype = rng.choice(("f16", "bf16", "f32"))
        queries = _log_int(rng, 1, 4096)
        rows = _log_int(rng, 50, min(1_000_000, 1_000_000 * 1024 // queries // (8 if dtype == "f32" else 1)))
        grad_rows = rows * queries < 1 << 28 and rng.random() < 0.4
        return loss_case(None, queries, rows, dtype, dim=1024 if rng.random() < 0.6 else 8 * _log_int(rng, 4, 128), grad_queries=rng.random() < 0.8,
                         grad_rows=grad_rows, live=rng.choice((1.0, 1.0, 0.9, 0.3)), targets=rng.randint(1, 5), pad=rng.choice((0, 0, 8, 64)),
                         scale=round(rng.uniform(1.5, 2.5) * math.log(rows), 1))
    if op == "ortho":
        dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
        rows, cols = _log_int(rng, 16, 1200 if dtype == "f32" else 4096), _log_int(rng, 16, 1200 if dtype == "f32" else 4096)
        batch = min(rng.choice((1, 1, 2, 5)), max(1, (1 << 24) // (rows * cols)))
        return ortho_case(None, batch, rows, cols, dtype, pad=rng.choice((0, 0, 3, 64)))
    dtype = rng.choice(("f16", "bf16", "f32"))
    dim = 1024 if rng.random() < 0.6 else _log_int(rng, 32, 4096)
    return residual_case(None, _log_int(rng, 1, (1 << 26) // dim), dtype, dim=dim, gate=rng.choice(("none", "element", "channel")),
                         grad=rng.random() < 0.7, grad_y=rng.random() < 0.5, pad=rng.choice((0, 0, 8, 64)))


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


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, generator=g, device=DEV)  # noqa: E731
    dt = TYPES[case["dtype"]]
    state = dict(case=case)
    if own:
        state["ctx"] = _context()
    if case["op"] == "loss":
        n, m, d = case["rows"], case["queries"], case["dim"]
        rows = rand(n, d)
        rows /= rows.norm(dim=1, keepdim=True)
        rows = rows.to(dt)
        # up to `targets` relevant rows a query, now and then none; graded
        count = torch.randint(1, case["targets"] + 1, (m,), generator=g, device=DEV)
        if m > 8:
            count[torch.randint(0, m, (m // 50 + 1,), generator=g, device=DEV)] = 0
        t_off = torch.zeros(m + 1, dtype=torch.int32, device=DEV)
        t_off[1:] = torch.cumsum(count, 0)
        total = int(t_off[-1])
        t_idx = torch.randint(0, n, (total,), generator=g, device=DEV, dtype=torch.int32)
        t_val = torch.randint(1, 4, (total,), generator=g, device=DEV).float()
        which = torch.repeat_interleave(torch.arange(m, device=DEV), count)
        t_val = t_val / torch.zeros(m, device=DEV).index_add(0, which, t_val)[which]
        # a query leans to its relevant rows, among the many rows that it does not lie far from: what there is to learn
        near = torch.zeros(m, d, device=DEV).index_add(0, which, rows[t_idx.long()].float())
        queries = near + 3.0 / math.sqrt(d) * rand(m, d)
        queries /= queries.norm(dim=1, keepdim=True)
        live = None
        if case["live"] < 1.0:
            bits = torch.zeros(-(-n // 32) * 32, dtype=torch.long, device=DEV)
            bits[:n] = (torch.rand(n, generator=g, device=DEV) < case["live"]).long()
            live = (bits.view(-1, 32) << torch.arange(32, device=DEV)).sum(1)
            live = torch.where(live >= 1 << 31, live - (1 << 32), live).to(torch.int32)
        weight = torch.full((m,), 1.0 / m, device=DEV)
        state.update(queries=_strided(queries.to(dt), case["pad"]), rows=_strided(rows, case["pad"]), t_off=t_off, t_idx=t_idx, t_val=t_val,
                     live=live, weight=weight)
    elif case["op"] == "ortho":
        b, r, c = case["batch"], case["rows"], case["cols"]
        # a few strong directions over a floor, as gradients have them
        k = min(16, r, c)
        left = rand(b, r, k) * torch.logspace(0, -2, k, device=DEV)
        right = rand(b, k, c)
        x = 0.1 * rand(b, r, c)
        for i in range(b):
            x[i] += left[i] @ right[i]
        state.update(x=_strided((1e-3 * x).to(dt), case["pad"]))
    else:
        n, d = case["rows"], case["dim"]
        x = rand(n, d)
        x /= x.norm(dim=1, keepdim=True)
        state.update(x=_strided(x.to(dt), case["pad"]), h=_strided((0.3 * rand(n, d)).to(dt), case["pad"]),
                     gate=None if case["gate"] == "none" else rand(d).to(dt) if case["gate"] == "channel" else _strided(rand(n, d).to(dt), case["pad"]),
                     scale=0.05 + 0.01 * rand(d), w_post=1.0 + 0.1 * rand(d), w_next=(1.0 + 0.05 * rand(d)) / math.sqrt(d))
        if case["grad"]:
            state.update(grad_u=_strided((1e-2 * rand(n, d)).to(dt), case["pad"]), grad_y=_strided((1e-2 * rand(n, d)).to(dt), case["pad"]) if case["grad_y"] else None)
    return state


# ---- one pass ----

def run(state):
    op = state["case"]["op"]
    if own:
        return {"loss": _own_loss, "ortho": _own_ortho, "residual": _own_residual}[op](state)
    return {"loss": _plain_loss, "ortho": _plain_ortho, "residual": _plain_residual}[op](state)


def _own_loss(s):
    import apoe
    c = s["case"]
    return apoe.softmax_loss(s["ctx"], s["queries"], s["rows"], s["t_off"], s["t_idx"], s["t_val"], scale=c["scale"], weight=s["weight"], live=s["live"],
                             grad_queries=c["grad_queries"], grad_rows=c["grad_rows"])


def _own_ortho(s):
    import apoe
    return dict(out=apoe.orthogonalize(s["ctx"], s["x"], steps=STEPS, coefs=COEFS))


def _own_residual(s):
    import apoe
    y, u = apoe.gated_residual(s["ctx"], s["x"], s["h"], gate=s["gate"], scale=s["scale"], w_post=s["w_post"], w_next=s["w_next"], eps=EPS)
    if not s["case"]["grad"]:
        return dict(y=y, u=u)
    grads = apoe.gated_residual_grad(s["ctx"], s["x"], s["h"], gate=s["gate"], scale=s["scale"], w_post=s["w_post"], w_next=s["w_next"], eps=EPS,
                                     grad_y=s["grad_y"], grad_u=s["grad_u"])
    return dict(grads, y=y, u=u)


def _plain_loss(s):
    c = s["case"]
    q, x, dt = s["queries"].float(), s["rows"].float(), s["queries"].dtype
    m, n = q.shape[0], x.shape[0]
    logits = (q @ x.T) * c["scale"]
    w, t = s["t_val"], s["t_idx"].long()
    which = torch.repeat_interleave(torch.arange(m, device=DEV), (s["t_off"][1:] - s["t_off"][:-1]).long(), output_size=t.numel())
    if s["live"] is not None:
        alive = ((s["live"][:, None] >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1).bool().reshape(-1)[:n]
        logits.masked_fill_(~alive, float("-inf"))
        w = w * alive[t]
    top = logits.amax(1)
    top = torch.where(top > float("-inf"), top, torch.zeros_like(top))
    lse = top + torch.log(torch.exp(logits - top[:, None]).sum(1))
    total = torch.zeros(m, device=DEV).index_add(0, which, w)
    at = torch.zeros(m, device=DEV).index_add(0, which, torch.where(w != 0, w * logits[which, t], torch.zeros_like(w)))
    out = dict(loss=torch.where(total != 0, total * lse, torch.zeros_like(lse)) - at, lse=lse)
    if c["grad_queries"] or c["grad_rows"]:
        p = logits.sub_(lse[:, None]).exp_().mul_(total[:, None])
        p.index_put_((which, t), -w, accumulate=True)
        p *= (s["weight"] * c["scale"])[:, None]
        if c["grad_queries"]:
            out["grad_queries"] = (p @ x).to(dt)
        if c["grad_rows"]:
            out["grad_rows"] = (p.T @ q).to(dt)
    return out


def _plain_ortho(s):
    x = s["x"].float()
    x = x / torch.sqrt((x * x).sum((1, 2), keepdim=True))
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.transpose(1, 2).contiguous()
    a, b, c = COEFS
    for _ in range(STEPS):
        gram = x @ x.transpose(1, 2).contiguous()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    if tall:
        x = x.transpose(1, 2).contiguous()
    return dict(out=x.to(s["x"].dtype))


def _plain_residual(s):
    dt = s["x"].dtype
    x, h = s["x"].float(), s["h"].float()
    scale, w_post, w_next = s["scale"], s["w_post"], s["w_next"]
    rh = torch.rsqrt((h * h).mean(1, keepdim=True) + EPS)
    hn = h * rh
    gate = None if s["gate"] is None else torch.sigmoid(s["gate"].float())
    open_ = 1.0 if gate is None else gate
    y = x + scale * open_ * hn * w_post
    ry = torch.rsqrt((y * y).mean(1, keepdim=True) + EPS)
    yn = y * ry
    out = dict(y=y.to(dt), u=(yn * w_next).to(dt))
    if not s["case"]["grad"]:
        return out
    gu = s["grad_u"].float()
    out["grad_w_next"] = (gu * yn).sum(0)
    gyn = gu * w_next
    gy = ry * (gyn - yn * (gyn * yn).mean(1, keepdim=True))
    if s["grad_y"] is not None:
        gy = gy + s["grad_y"].float()
    out["grad_x"] = gy.to(dt)
    out["grad_scale"] = (gy * open_ * hn * w_post).sum(0)
    if gate is not None:
        gg = gy * scale * hn * w_post * gate * (1.0 - gate)
        out["grad_gate"] = (gg.sum(0) if gate.dim() == 1 else gg).to(dt)
    gn = gy * scale * open_
    out["grad_w_post"] = (gn * hn).sum(0)
    gh = gn * w_post
    out["grad_h"] = (rh * (gh - hn * (gh * hn).mean(1, keepdim=True))).to(dt)
    return out


# ---- what a pass cannot do without ----

def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}[case["dtype"]]
    if case["op"] == "loss":
        n, m, d = case["rows"], case["queries"], case["dim"]
        products = 1 + case["grad_queries"] + case["grad_rows"]
        move = size * d * ((m + n) + m * case["grad_queries"] + n * case["grad_rows"]) + m * 4 * (2 + 2 * case["targets"] + 3)
        return {"bytes": move + (n / 8 if case["live"] < 1 else 0), "flops": 2.0 * m * n * d * products}
    if case["op"] == "ortho":
        lo, hi = sorted((case["rows"], case["cols"]))
        # two products that are symmetric and one that is not, a step
        return {"bytes": 2.0 * size * case["batch"] * lo * hi, "flops": case["batch"] * STEPS * (lo * lo * hi + lo ** 3 + 2.0 * lo * lo * hi)}
    n, d = case["rows"], case["dim"]
    gate = n if case["gate"] == "element" else 1 if case["gate"] == "channel" else 0
    move, flops = (4 * n + gate) * d * size + 12 * d, 14.0 * n * d
    if case["grad"]:
        move += (n * (3 + case["grad_y"]) + gate) * d * size + 12 * d
        flops += 30.0 * n * d
    return {"bytes": move, "flops": flops}


# ---- the same in 64 bits, from the definitions ----

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "loss":
        return _exact_loss(case, s)
    if case["op"] == "ortho":
        outs = []
        for x in s["x"].double():
            x = x / torch.linalg.matrix_norm(x)
            wide = x if x.shape[0] <= x.shape[1] else x.T.contiguous()
            eye = torch.eye(wide.shape[0], dtype=torch.float64, device=DEV)
            for _ in range(STEPS):
                gram = torch.mm(wide, wide.T.contiguous())
                wide = torch.mm(COEFS[0] * eye + COEFS[1] * gram + COEFS[2] * torch.mm(gram, gram), wide)
            outs.append(wide if x.shape[0] <= x.shape[1] else wide.T)
        return dict(out=torch.stack(outs))
    return _exact_residual(case, s)


def _exact_loss(case, s):
    """Row blocks of the softmax matrix: loss_i = sum_t w_it (lse_i - s_it), its gradient by s is (sum_t w_it) p_ij - w_ij."""
    q, x = s["queries"].double(), s["rows"].double()
    n = x.shape[0]
    share = torch.zeros(n, dtype=torch.bool, device=DEV)
    if s["live"] is None:
        share[:] = True
    else:
        ids = torch.arange(n, device=DEV)
        share = (s["live"][ids // 32].long() >> (ids % 32)) & 1 == 1
    off = s["t_off"].tolist()
    loss, lse, gq, gx = [], [], [], torch.zeros_like(x) if case["grad_rows"] else None
    for r0 in range(0, q.shape[0], 512):
        r1 = min(q.shape[0], r0 + 512)
        z = case["scale"] * torch.mm(q[r0:r1], x.T)
        z[:, ~share] = -float("inf")
        want = torch.zeros_like(z)
        e0, e1 = off[r0], off[r1]
        if e1 > e0:
            lens = torch.tensor([off[i + 1] - off[i] for i in range(r0, r1)], device=DEV)
            at = torch.repeat_interleave(torch.arange(r1 - r0, device=DEV), lens)
            want.index_put_((at, s["t_idx"][e0:e1].long()), s["t_val"][e0:e1].double(), accumulate=True)
        want[:, ~share] = 0
        l = torch.logsumexp(z, 1)
        total = want.sum(1)
        loss.append(torch.where(total == 0, torch.zeros_like(l), (want * torch.where(want == 0, torch.zeros_like(z), l[:, None] - z)).sum(1)))
        lse.append(l)
        if case["grad_queries"] or case["grad_rows"]:
            gz = torch.softmax(z, 1) * total[:, None] - want
            gz *= case["scale"] * s["weight"][r0:r1, None].double()
            if case["grad_queries"]:
                gq.append(torch.mm(gz, x))
            if case["grad_rows"]:
                gx += torch.mm(gz.T.contiguous(), q[r0:r1])
    out = dict(loss=torch.cat(loss), lse=torch.cat(lse))
    if case["grad_queries"]:
        out["grad_queries"] = torch.cat(gq)
    if case["grad_rows"]:
        out["grad_rows"] = gx
    return out


def _exact_residual(case, s):
    """The forward pass in 64 bits; its gradients by automatic differentiation of that."""
    names = [k for k in ("x", "h", "gate", "scale", "w_post", "w_next") if s[k] is not None]
    v = {k: s[k].double().requires_grad_(case["grad"]) for k in names}
    norm = lambda t: t / torch.sqrt(t.square().mean(-1, keepdim=True) + EPS)  # noqa: E731
    block = norm(v["h"]) * v["w_post"] * v["scale"]
    y = v["x"] + (block if s["gate"] is None else block / (1 + torch.exp(-v["gate"])))
    u = norm(y) * v["w_next"]
    out = dict(y=y.detach(), u=u.detach())
    if case["grad"]:
        aim = (u * s["grad_u"].double()).sum()
        if s["grad_y"] is not None:
            aim = aim + (y * s["grad_y"].double()).sum()
        for k, g in zip(names, torch.autograd.grad(aim, [v[k] for k in names])):
            out["grad_" + k] = g
    return out
