"""Trains a small language model on packed documents of tokens from a teacher's top logits: the tokens'
embedding, scaled, a block of causal attention with a norm of each query and key head before the
turn, a gated two-layer part, and logits from the same table.  Padding is a token of -1, and a row of
the teacher without an entry.

Every product, norm, gradient and the loss is a call of katsu_amd.ops on float32 device tensors; the
update is torch's.   python examples/lm_distill.py [steps]
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from katsu_amd import ops  # noqa: E402

LENS = [37, 150, 1, 64]  # the documents of a batch, the last tokens of each padding
PAD = 5
VOCAB, WIDTH, HEADS, KV_HEADS, DIM, HIDDEN, TOP = 211, 96, 6, 2, 24, 160, 7
SCALE, TAU, ALPHA = WIDTH ** 0.5, 2.0, 0.5


def parameters(gen, dev):
    """Weights by name; the last dimension is a product's output, but the table's."""
    def normal(rows, cols, size):
        return torch.randn(rows, cols, generator=gen) * size
    p = {"table": normal(VOCAB, WIDTH, 1 / WIDTH), "wq": normal(WIDTH, HEADS * DIM, WIDTH ** -0.5),
         "wk": normal(WIDTH, KV_HEADS * DIM, WIDTH ** -0.5),
         "wv": normal(WIDTH, KV_HEADS * DIM, WIDTH ** -0.5),
         "wo": normal(HEADS * DIM, WIDTH, (HEADS * DIM) ** -0.5),
         "w1": normal(WIDTH, HIDDEN, WIDTH ** -0.5), "w2": normal(WIDTH, HIDDEN, WIDTH ** -0.5),
         "w3": normal(HIDDEN, WIDTH, HIDDEN ** -0.5)}
    for n in ("pre1", "pre2", "pre3"):
        p[n] = torch.ones(WIDTH)
    for n in ("nq", "nk"):
        p[n] = torch.ones(DIM)
    return {k: v.to(dev) for k, v in p.items()}


def step(p, tokens, ids, teacher, cu, table, positions):
    """(each row's loss, gradients of their mean by name) of one batch: int32 tokens [T], the teacher's
    top logits and their columns [T, TOP]."""
    t = tokens.shape[0]
    seqs = dict(cu_q=cu, cu_k=cu)
    x = ops.embedding(tokens, p["table"], scale=SCALE)
    # The norm before the first part: nothing is added to x.
    _, h1, s1 = ops.block_norm(x, x, w_pre=p["pre1"], alpha=0.0)
    q0, k0, v = (ops.matmul(h1, p[w]).view(t, -1, DIM) for w in ("wq", "wk", "wv"))
    how = dict(table=table, positions=positions, w_q=p["nq"], w_k=p["nk"])
    q, k = ops.qk_norm_rotary(q0, k0, **how)
    a, lse = ops.attention(q, k, v, **seqs)
    a = a.view(t, -1)
    o1 = ops.matmul(a, p["wo"])
    y1, h2, s2 = ops.block_norm(x, o1, w_pre=p["pre2"], alpha=ALPHA)
    u, w = ops.matmul(h2, p["w1"]), ops.matmul(h2, p["w2"])
    m = ops.mul(u, w)
    o2 = ops.matmul(m, p["w3"])
    y2, h3, s3 = ops.block_norm(y1, o2, w_pre=p["pre3"], alpha=ALPHA)
    logits = ops.gemm(h3, p["table"], t, VOCAB, WIDTH, trans_b=True)
    mean = torch.full((1,), 1.0 / t, device=x.device).expand(t)
    loss, dlogits = ops.distillation_step(logits, ids, teacher, mean, TAU, out=logits)

    g = {"table": ops.gemm(dlogits, h3, VOCAB, WIDTH, t, trans_a=True)}

    def product(x, name, gy):  # the gradients of x @ p[name]
        gx, g[name] = torch.zeros_like(x), torch.zeros_like(p[name])
        ops.matmul_vjp(x, p[name], gy, gx, g[name])
        return gx
    zero = torch.zeros_like(x)
    dh3 = ops.gemm(dlogits, p["table"], t, WIDTH, VOCAB)
    dy1, do2, _, _, g["pre3"] = ops.block_norm_backward(zero, dh3, y2, o2, s3, w_pre=p["pre3"],
                                                        alpha=ALPHA)
    dm = product(m, "w3", do2)
    dh2 = product(h2, "w1", ops.mul(dm, w))
    ops.accumulate(product(h2, "w2", ops.mul(dm, u)), dh2)
    dx, do1, _, _, g["pre2"] = ops.block_norm_backward(dy1, dh2, y1, o1, s2, w_pre=p["pre2"],
                                                       alpha=ALPHA)
    da = product(a, "wo", do1).view(t, HEADS, DIM)
    dq, dk, dv = ops.attention_backward(da, q, k, v, a.view(t, HEADS, DIM), lse, **seqs)
    dq, dk, g["nq"], g["nk"] = ops.qk_norm_rotary_backward(dq, dk, q0, k0, out_q=dq, out_k=dk,
                                                           **how)
    dh1 = product(h1, "wq", dq.view(t, -1))
    for name, d in (("wk", dk), ("wv", dv)):
        ops.accumulate(product(h1, name, d.view(t, -1)), dh1)
    dx, *_, g["pre1"] = ops.block_norm_backward(dx, dh1, x, x, s1, w_pre=p["pre1"], alpha=0.0)
    # The table's other gradient is there already.
    ops.embedding_backward(dx, tokens, VOCAB, scale=SCALE, out=g["table"], beta=1.0)
    return loss, g


def batch(gen, dev):
    """Tokens, the teacher's top logits and their columns, the documents' starts, the table of angles,
    each token's position."""
    t = sum(LENS)
    tokens = torch.randint(0, VOCAB, (t,), generator=gen)
    top = (torch.randn(t, VOCAB, generator=gen) * 2).topk(TOP, dim=1)
    ids, at = top.indices, 0
    for n in LENS:
        at += n
        pad = slice(at - min(PAD, n - 1), at)
        tokens[pad], ids[pad] = -1, -1
    cu = torch.tensor([0] + LENS, dtype=torch.int32).cumsum(0, dtype=torch.int32).to(dev)
    positions = torch.cat([torch.arange(n, dtype=torch.int32) for n in LENS]).to(dev)
    return (tokens.int().to(dev), ids.int().to(dev), top.values.to(dev), cu,
            ops.rotary_table(max(LENS), DIM, device=dev), positions)


def train(steps, rate=0.1, max_norm=1.0, seed=0):
    """The mean losses of `steps` steps on one batch."""
    gen, dev = torch.Generator().manual_seed(seed), torch.device("cuda:0")
    p, data = parameters(gen, dev), batch(gen, dev)
    losses = []
    for _ in range(steps):
        loss, g = step(p, *data)
        ops.clip_grad_norm([g[k] for k in p], max_norm)
        for k in p:
            p[k].sub_(g[k], alpha=rate)
        losses.append(ops.sum(loss))
    return [v.item() / sum(LENS) for v in losses]


if __name__ == "__main__":
    for i, v in enumerate(train(int(sys.argv[1]) if len(sys.argv) > 1 else 20)):
        print(f"step {i}: loss {v:.4f}")
