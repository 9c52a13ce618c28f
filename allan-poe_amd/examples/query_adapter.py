"""Fits a query adapter to a stored index: the encoder of the queries has changed, the documents and their graph stay.

    python allan-poe_amd/examples/query_adapter.py [--docs 20000] [--train 32768] [--steps 300] [--batch 512] [--block mlp]

The corpus is the synthetic one whose dense rows have neighbours. The "new encoder" gives vectors that lean away from the
documents' space (a fixed rotation mixed in), so a search with them misses most of what is relevant. What is known is a set of
judgements, rows that are relevant to each training query. The adapter is one residual block on the query,

    n = norm(x) w_pre,  h = W n,  y = x + scale sigmoid(gate) w_post norm(h),  q = y / |y|

and it learns from the softmax cross entropy of q over every document: `apoe.gated_residual` (and its gradient) is the frame,
`apoe.softmax_loss` the loss over the corpus' half-precision rows, and the matrix W takes steps that `apoe.orthogonalize` makes
from its momentum. Nothing of the index is built again; the same graph is searched before and after. Prints one line of JSON.

With --block mlp the adapter is a layer of the kind that encoders have, and reads the query's learned-sparse terms too:

    e = x + s sum_t val_t E[t],  n = layer_norm(e),  y = e + W2 gelu(W1 n + b1) + b2,  q = y / |y|

through `apoe.embed`, `apoe.layer_norm` and `apoe.linear` and their gradients; all of it, the table of the terms among it, takes its steps from
`apoe.AdamW` (--bits 8: with moments in 8 bits), which writes the half-precision copies that the next step multiplies with.
"""
import argparse
import json
import os
import sys
import time

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import apoe  # noqa: E402
import apoe_synth as S  # noqa: E402

DIM = 1024


class QueryAdapter:
    """The adapter's parameters (float32 masters), one training step, and the map itself."""

    LOSS_SCALE = 1024.0  # gradients travel as float16

    def __init__(self, ctx, dim=DIM, seed=0):
        g = torch.Generator().manual_seed(seed)
        dev = f"cuda:{ctx.device}"
        self.ctx, self.dim = ctx, dim
        self.W = (torch.randn(dim, dim, generator=g) / dim ** 0.5).to(dev)
        self.gate = torch.zeros(dim, device=dev)
        self.scale = torch.full((dim,), 0.5 / dim ** 0.5, device=dev)  # beside a query of length one the block starts at a quarter
        self.w_pre, self.w_post = torch.ones(dim, device=dev), torch.ones(dim, device=dev)
        self.unit = torch.full((dim,), 1 / dim ** 0.5, device=dev)     # the last norm gives length one
        self.vectors = dict(gate=self.gate, scale=self.scale, w_pre=self.w_pre, w_post=self.w_post)
        self.momentum = {k: torch.zeros_like(v) for k, v in dict(self.vectors, W=self.W).items()}

    def _block(self, x):
        n = apoe.gated_residual(self.ctx, x, w_next=self.w_pre)[1]
        return n, n @ self.W.half().T, dict(gate=self.gate.half(), scale=self.scale, w_post=self.w_post, w_next=self.unit, eps=1e-12)

    def __call__(self, x):
        """Adapted queries of unit length, float16 [m, dim]."""
        n, h, parts = self._block(x)
        return apoe.gated_residual(self.ctx, x, h, **parts)[1]

    def step(self, x, corpus, t_off, t_idx, temperature, lr, beta=0.95):
        """One step on queries x and the rows that are relevant to each; returns the losses [m] (on the GPU)."""
        n, h, parts = self._block(x)
        y, q = apoe.gated_residual(self.ctx, x, h, **parts)
        weight = torch.full((x.shape[0],), self.LOSS_SCALE / x.shape[0], device=x.device)
        out = apoe.softmax_loss(self.ctx, q, corpus, t_off, t_idx, scale=1 / temperature, weight=weight, grad_queries=True)
        g = apoe.gated_residual_grad(self.ctx, x, h, **parts, grad_u=out["grad_queries"])
        gn = g["grad_h"] @ self.W.half()
        pre = apoe.gated_residual_grad(self.ctx, x, w_next=self.w_pre, grad_u=gn)
        grads = dict(gate=g["grad_gate"].float(), scale=g["grad_scale"], w_post=g["grad_w_post"], w_pre=pre["grad_w_next"],
                     W=(g["grad_h"].T @ n).float())
        for k, grad in grads.items():
            self.momentum[k].mul_(beta).add_(grad, alpha=1 / self.LOSS_SCALE)
        # the matrix: a step of the same size along every direction that its momentum names
        apoe.orthogonalize(self.ctx, self.momentum["W"], out=self.W, alpha=-lr, beta=1.0, products="f16")
        for k, v in self.vectors.items():  # the vectors: the momentum's direction, at a size of their own
            m = self.momentum[k]
            v.sub_(m * (lr * 0.1 * v.norm().clamp_min(1.0 / self.dim ** 0.5) / m.norm().clamp_min(1e-30)))
        return out["loss"]


class MlpAdapter:
    """The layer's parameters (float32 masters and copies in `dtype` that the products take), its map and one training step. `terms` is the CSR
    of the queries' learned-sparse terms: offsets, term ids, weights."""

    LOSS_SCALE = 1024.0  # gradients travel as float16; halved when they overflow
    SCALE = 0.1          # of the terms' sum

    def __init__(self, ctx, dim=DIM, hidden=2 * DIM, vocab=S.VOCAB, dtype=torch.float16, bits=32, seed=0):
        g = torch.Generator().manual_seed(seed)
        dev = f"cuda:{ctx.device}"
        self.ctx, self.dtype = ctx, dtype
        rand = lambda *shape: torch.randn(*shape, generator=g).to(dev)  # noqa: E731
        self.params = dict(E=torch.zeros(vocab, dim, device=dev), w=torch.ones(dim, device=dev), b=torch.zeros(dim, device=dev), W1=rand(hidden, dim) / dim ** 0.5,
                           b1=torch.zeros(hidden, device=dev), W2=0.02 * rand(dim, hidden) / hidden ** 0.5, b2=torch.zeros(dim, device=dev))
        matrices = ("E", "W1", "W2")
        self.copies = {k: self.params[k].to(dtype) for k in matrices}
        self.unit = torch.full((dim,), 1 / dim ** 0.5, device=dev)
        in_type = {k: v for k, v in self.copies.items() if dtype != torch.float32}  # float32: the products take the masters themselves
        self.opt = apoe.AdamW(ctx, list(self.params.values()), copies=[in_type.get(k) for k in self.params], bits=bits,
                              weight_decay=[0.01 if k in matrices else 0.0 for k in self.params], seed=seed)

    def _matrix(self, name):
        return self.params[name] if self.dtype == torch.float32 else self.copies[name]

    def _layer(self, x, terms):
        off, idx, val = terms
        e = apoe.embed(self.ctx, self._matrix("E"), idx, off, val, scale=self.SCALE, base=x)
        n = apoe.layer_norm(self.ctx, e, self.params["w"], self.params["b"])
        h, pre = apoe.linear(self.ctx, n, self._matrix("W1"), self.params["b1"], act="gelu", want_pre=True)
        y, _ = apoe.linear(self.ctx, h, self._matrix("W2"), self.params["b2"], residual=e)
        return e, n, h, pre, y

    def __call__(self, x, terms):
        """Adapted queries of unit length [m, dim]."""
        return apoe.gated_residual(self.ctx, self._layer(x, terms)[-1], w_next=self.unit, eps=1e-12)[1]

    def gradients(self, x, terms, rows, t_off, t_idx, temperature):
        """(losses [m], gradients of LOSS_SCALE times their mean by every parameter)."""
        e, n, h, pre, y = self._layer(x, terms)
        off, idx, val = terms
        q = apoe.gated_residual(self.ctx, y, w_next=self.unit, eps=1e-12)[1]
        weight = torch.full((x.shape[0],), self.LOSS_SCALE / x.shape[0], device=x.device)
        out = apoe.softmax_loss(self.ctx, q, rows, t_off, t_idx, scale=1 / temperature, weight=weight, grad_queries=True)
        gy = apoe.gated_residual_grad(self.ctx, y, w_next=self.unit, eps=1e-12, grad_u=out["grad_queries"])["grad_x"]
        two = apoe.linear_grad(self.ctx, h, self._matrix("W2"), gy)
        one = apoe.linear_grad(self.ctx, n, self._matrix("W1"), two["grad_x"], act="gelu", pre=pre)
        norm = apoe.layer_norm_grad(self.ctx, e, self.params["w"], self.params["b"], grad_y=one["grad_x"], grad_skip=gy)  # y = e + ..: past the layer
        table = apoe.embed_grad(self.ctx, self._matrix("E"), norm["grad_x"], idx, off, val, scale=self.SCALE)["grad_table"]
        return out["loss"], dict(E=table, w=norm["grad_w"], b=norm["grad_b"], W1=one["grad_w"], b1=one["grad_bias"], W2=two["grad_w"], b2=two["grad_bias"])

    def step(self, x, terms, rows, t_off, t_idx, temperature, lr):
        loss, grads = self.gradients(x, terms, rows, t_off, t_idx, temperature)
        if torch.stack([torch.isfinite(g).all() for g in grads.values()]).all():
            self.opt.step([grads[k] for k in self.params], lr, grad_scale=1 / self.LOSS_SCALE)
        else:  # a moment that is not finite never is again, in 8 bits its whole block
            self.LOSS_SCALE /= 2
        return loss


def rows_of(csr, at):
    """The CSR of the rows `at`."""
    off, idx, val = csr
    off = off.long()
    count = off[at + 1] - off[at]
    new = torch.zeros(len(at) + 1, dtype=torch.long, device=idx.device)
    new[1:] = count.cumsum(0)
    entries = torch.arange(int(new[-1]), device=idx.device) + torch.repeat_interleave(off[at] - new[:-1], count)
    return new.to(torch.int32), idx[entries], val[entries]


def judgements(queries, dense, k):
    """CSR of the k rows closest to each query (what people or logs would say)."""
    idx = (queries @ dense.T).topk(k, dim=1).indices.to(torch.int32)
    off = torch.arange(0, idx.numel() + 1, k, dtype=torch.int32, device=idx.device)
    return off, idx.reshape(-1)


def recall(ctx, corpus, graph, dense, sparse, wanted, cands, k=10):
    """Share of the wanted rows among the first k that a dense search of the stored graph returns."""
    queries = apoe.Queries(ctx, dense.float(), *sparse)
    ids, _, _ = apoe.search(ctx, corpus, queries, graph, (1.0, 0.0, 0.0), cands)
    queries.close()
    found = torch.from_numpy(ids[:, :k].astype("int64")).to(wanted.device)
    return float((found[:, :, None] == wanted[:, None, :].long()).any(1).float().mean())


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--docs", type=int, default=20_000)
    p.add_argument("--train", type=int, default=32768)
    p.add_argument("--held-out", type=int, default=512)
    p.add_argument("--steps", type=int, default=300)
    p.add_argument("--batch", type=int, default=512)
    p.add_argument("--block", choices=("gated", "mlp"), default="gated")
    p.add_argument("--bits", type=int, choices=(8, 32), default=32, help="of the moments of --block mlp")
    p.add_argument("--lr", type=float, default=None, help="0.05, with --block mlp 0.001")
    p.add_argument("--temperature", type=float, default=0.05)
    p.add_argument("--cands", type=int, default=128)
    args = p.parse_args(argv)
    mlp = args.block == "mlp"
    if args.lr is None:
        args.lr = 0.001 if mlp else 0.05
    dev = "cuda:0"
    ctx = apoe.Context(0, stream=torch.cuda.current_stream())
    rows = S.latent_corpus(args.docs, device=dev)
    corpus = apoe.Corpus(ctx, *rows)
    corpus.make_half_rows()
    graph, build_ms = apoe.build_graph(ctx, corpus, K=64, iters=10, degree=32, join=1)

    said = S.latent_queries(args.train + args.held_out, device=dev)
    old, csr = said[0], (said[1].to(torch.int32), said[2].to(torch.int32), said[3])  # what the old encoder said, and the queries' terms
    g = torch.Generator().manual_seed(1)
    turn = torch.linalg.qr(torch.randn(DIM, DIM, generator=g)).Q.to(dev)
    new = old + 1.5 * old @ turn                                        # what the new one says
    new = (new / new.norm(dim=1, keepdim=True)).half()
    t_off, t_idx = judgements(old[:args.train], rows[0], 3)
    held, sparse = new[args.train:], S.latent_queries(args.held_out, seed=7, device=dev)[1:]
    wanted = judgements(old[args.train:], rows[0], 10)[1].view(-1, 10)

    before = recall(ctx, corpus, graph, held, sparse, wanted, args.cands)
    adapter = MlpAdapter(ctx, bits=args.bits) if mlp else QueryAdapter(ctx)
    losses = []
    torch.cuda.synchronize()
    start = time.perf_counter()
    for step in range(args.steps):
        at = torch.randint(0, args.train, (args.batch,), generator=g).to(dev)
        idx = t_idx.view(-1, 3)[at].reshape(-1)
        off = torch.arange(0, 3 * args.batch + 1, 3, dtype=torch.int32, device=dev)
        warm = min(1.0, 4.0 * (args.steps - step) / args.steps)         # the last quarter's steps shrink
        if mlp:
            losses.append(adapter.step(new[at], rows_of(csr, at), corpus, off, idx, args.temperature, args.lr * warm).mean())
        else:
            losses.append(adapter.step(new[at], corpus, off, idx, args.temperature, args.lr * warm).mean())
    torch.cuda.synchronize()
    took = time.perf_counter() - start
    mapped = adapter(held, rows_of(csr, torch.arange(args.train, args.train + args.held_out, device=dev))) if mlp else adapter(held)
    after = recall(ctx, corpus, graph, mapped, sparse, wanted, args.cands)
    limit = recall(ctx, corpus, graph, old[args.train:], sparse, wanted, args.cands)
    for part in (graph, corpus, ctx):
        part.close()
    return dict(block=args.block, docs=args.docs, build_ms=round(build_ms, 1), steps=args.steps, batch=args.batch, ms_per_step=round(1e3 * took / args.steps, 3),
                loss_first=round(float(losses[0]), 3), loss_last=round(float(torch.stack(losses[-10:]).mean()), 3),
                recall_at_10_before=round(before, 4), recall_at_10_after=round(after, 4), recall_at_10_old_encoder=round(limit, 4))


if __name__ == "__main__":
    print(json.dumps(main()))
