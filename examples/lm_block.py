"""Trains one block of a language model on packed documents with the library's operators: norms,
gates and residuals between the parts, rotary positions, causal attention within each document, a
gated two-layer part, a squared-error loss, and gradients clipped by their global norm.

Every product, norm and gradient is a call of katsu_amd.ops on float32 device tensors; the update is
torch's.   python examples/lm_block.py [steps]
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from katsu_amd import ops  # noqa: E402

LENS = [37, 150, 1, 64]  # the documents of a batch
WIDTH, HEADS, KV_HEADS, DIM, HIDDEN, OUT = 96, 6, 2, 24, 160, 32
ALPHA = 0.5              # of what a part adds to the residual


def parameters(gen, dev):
    """Weights by name; the last dimension is a product's output."""
    def normal(rows, cols):
        return torch.randn(rows, cols, generator=gen) * rows ** -0.5
    p = {"wq": normal(WIDTH, HEADS * DIM), "wk": normal(WIDTH, KV_HEADS * DIM),
         "wv": normal(WIDTH, KV_HEADS * DIM), "wo": normal(HEADS * DIM, WIDTH),
         "w1": normal(WIDTH, HIDDEN), "w2": normal(WIDTH, HIDDEN), "w3": normal(HIDDEN, WIDTH),
         "out": normal(WIDTH, OUT)}
    for n in ("pre1", "post1", "pre2", "post2", "pre3", "gate1", "gate2"):
        p[n] = torch.ones(WIDTH)
    return {k: v.to(dev) for k, v in p.items()}


def step(p, x, target, cu, table, positions):
    """(loss, gradients by name) of one batch: x [tokens, WIDTH], target [tokens, OUT]."""
    t = x.shape[0]
    seqs = dict(cu_q=cu, cu_k=cu)
    # The norm before the first part: nothing is added to x.
    _, h1, s1 = ops.block_norm(x, x, w_pre=p["pre1"], alpha=0.0)
    q0, k0, v = (ops.matmul(h1, p[w]).view(t, -1, DIM) for w in ("wq", "wk", "wv"))
    q, k = ops.rotary(q0, k0, table, positions)
    a, lse = ops.attention(q, k, v, **seqs)
    a = a.view(t, -1)
    o1 = ops.matmul(a, p["wo"])
    y1, h2, s2 = ops.block_norm(x, o1, p["gate1"], p["post1"], p["pre2"], ALPHA)
    u, w = ops.matmul(h2, p["w1"]), ops.matmul(h2, p["w2"])
    m = ops.mul(u, w)
    o2 = ops.matmul(m, p["w3"])
    y2, h3, s3 = ops.block_norm(y1, o2, p["gate2"], p["post2"], p["pre3"], ALPHA)
    diff = ops.add(ops.matmul(h3, p["out"]), -target)
    loss = ops.sum(ops.mul(diff, diff))

    g = {}

    def product(x, name, gy):  # the gradients of x @ p[name]
        gx, g[name] = torch.zeros_like(x), torch.zeros_like(p[name])
        ops.matmul_vjp(x, p[name], gy, gx, g[name])
        return gx
    zero = torch.zeros_like(x)
    dh3 = product(h3, "out", ops.add(diff, diff))
    dy1, do2, g["gate2"], g["post2"], g["pre3"] = ops.block_norm_backward(
        zero, dh3, y2, o2, s3, p["gate2"], p["post2"], p["pre3"], ALPHA)
    dm = product(m, "w3", do2)
    dh2 = product(h2, "w1", ops.mul(dm, w))
    ops.accumulate(product(h2, "w2", ops.mul(dm, u)), dh2)
    _, do1, g["gate1"], g["post1"], g["pre2"] = ops.block_norm_backward(
        dy1, dh2, y1, o1, s2, p["gate1"], p["post1"], p["pre2"], ALPHA)
    da = product(a, "wo", do1).view(t, HEADS, DIM)
    dq, dk, dv = ops.attention_backward(da, q, k, v, a.view(t, HEADS, DIM), lse, **seqs)
    dq, dk = ops.rotary(dq, dk, table, positions, inverse=True, out_q=dq, out_k=dk)
    dh1 = product(h1, "wq", dq.view(t, -1))
    for name, d in (("wk", dk), ("wv", dv)):
        ops.accumulate(product(h1, name, d.view(t, -1)), dh1)
    *_, g["pre1"] = ops.block_norm_backward(zero, dh1, x, x, s1, w_pre=p["pre1"], alpha=0.0)
    return loss, g


def batch(gen, dev):
    """x, target, the documents' starts, the table of angles, each token's position."""
    t = sum(LENS)
    x, target = (torch.randn(t, n, generator=gen).to(dev) for n in (WIDTH, OUT))
    cu = torch.tensor([0] + LENS, dtype=torch.int32).cumsum(0, dtype=torch.int32).to(dev)
    positions = torch.cat([torch.arange(n, dtype=torch.int32) for n in LENS]).to(dev)
    return x, target, cu, ops.rotary_table(max(LENS), DIM, device=dev), positions


def train(steps, rate=0.02, max_norm=1.0, seed=0):
    """The losses of `steps` steps on one batch."""
    gen, dev = torch.Generator().manual_seed(seed), torch.device("cuda:0")
    p, data = parameters(gen, dev), batch(gen, dev)
    losses = []
    for _ in range(steps):
        loss, g = step(p, *data)
        ops.clip_grad_norm([g[k] for k in p], max_norm)
        for k in p:
            p[k].sub_(g[k], alpha=rate)
        losses.append(loss)
    return [v.item() for v in losses]


if __name__ == "__main__":
    for i, v in enumerate(train(int(sys.argv[1]) if len(sys.argv) > 1 else 20)):
        print(f"step {i}: loss {v:.3f}")
