"""The language-model operators together, as examples/lm_block.py runs them: its loss and all its
gradients against torch's automatic differentiation of the same block in float64, and a loss that
falls."""
import math

import pytest
import torch

from examples import lm_block as E

pytestmark = pytest.mark.gpu


def _norm(t):
    return t * (t.square().mean(1, keepdim=True) + 1e-6).rsqrt()


def _plain(p, x, target, cu, table, positions):
    """The block from its formulas, documents one by one."""
    c, s = table[positions.long()].split(E.DIM // 2, 1)
    c, s = c[:, None], s[:, None]

    def turn(t):
        a, b = t.split(E.DIM // 2, 2)
        return torch.cat([a * c - b * s, a * s + b * c], 2)
    h = _norm(x) * p["pre1"]
    q, k, v = ((h @ p[w]).view(len(x), -1, E.DIM) for w in ("wq", "wk", "wv"))
    q, k = turn(q), turn(k)
    a = []
    for i, j in zip(cu[:-1].tolist(), cu[1:].tolist()):
        for head in range(E.HEADS):
            kv = head // (E.HEADS // E.KV_HEADS)
            z = q[i:j, head] @ k[i:j, kv].T / math.sqrt(E.DIM)
            z = z + torch.full_like(z, -math.inf).triu(1)
            a.append(z.softmax(1) @ v[i:j, kv])
    a = torch.cat([torch.cat(a[n:n + E.HEADS], 1) for n in range(0, len(a), E.HEADS)])
    y = x + E.ALPHA * p["gate1"] * _norm(a @ p["wo"]) * p["post1"]
    h = _norm(y) * p["pre2"]
    o = ((h @ p["w1"]) * (h @ p["w2"])) @ p["w3"]
    y = y + E.ALPHA * p["gate2"] * _norm(o) * p["post2"]
    return ((_norm(y) * p["pre3"] @ p["out"] - target) ** 2).sum()


def test_gradients(dev):
    """Relative to each gradient's norm within 1e-4: a dozen float32 stages of sums of at most some
    hundred terms, gamma(300) = 1.8e-5 each at the worst, of either sign."""
    gen = torch.Generator().manual_seed(1)
    p, data = E.parameters(gen, dev), E.batch(gen, dev)
    for k in p:  # weights of norms and gates away from one
        if p[k].dim() == 1:
            p[k] = (1 + 0.3 * torch.randn(E.WIDTH, generator=gen)).to(dev)
    loss, g = E.step(p, *data)
    wide = {k: v.double().cpu().requires_grad_() for k, v in p.items()}
    x, target, cu, table, positions = (t.cpu() for t in data)
    want = _plain(wide, x.double(), target.double(), cu, table.double(), positions)
    want.backward()
    assert abs(loss.item() - want.item()) <= 1e-5 * want.item()
    assert set(g) == set(p)
    for k in p:
        d = (g[k].double().cpu() - wide[k].grad).norm() / wide[k].grad.norm()
        assert d <= 1e-4, (k, d.item())


def test_loss_falls(dev):
    losses = E.train(12)
    assert all(math.isfinite(v) for v in losses) and losses[-1] < losses[0]
