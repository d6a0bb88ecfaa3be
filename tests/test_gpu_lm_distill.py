"""Embedding, head norms with the turn and distillation together with the other operators, as
examples/lm_distill.py runs them: its losses and all its gradients against torch's automatic
differentiation of the same model in float64, and that it trains."""
import math

import pytest
import torch

from examples import lm_distill as E

pytestmark = pytest.mark.gpu


def _norm(t):
    return t * (t.square().mean(-1, keepdim=True) + 1e-6).rsqrt()


def _plain(p, tokens, ids, teacher, cu, table, positions):
    """The losses from the formulas, documents one by one."""
    c, s = table[positions.long()].split(E.DIM // 2, 1)
    c, s = c[:, None], s[:, None]

    def turn(t):
        a, b = t.split(E.DIM // 2, 2)
        return torch.cat([a * c - b * s, a * s + b * c], 2)
    real = (tokens >= 0)[:, None]
    x = torch.where(real, p["table"][tokens.long().clamp(min=0)] * E.SCALE, 0.0)
    h = _norm(x) * p["pre1"]
    q, k, v = ((h @ p[w]).view(len(x), -1, E.DIM) for w in ("wq", "wk", "wv"))
    q, k = turn(_norm(q) * p["nq"]), turn(_norm(k) * p["nk"])
    a = []
    for i, j in zip(cu[:-1].tolist(), cu[1:].tolist()):
        for head in range(E.HEADS):
            kv = head // (E.HEADS // E.KV_HEADS)
            z = q[i:j, head] @ k[i:j, kv].T / math.sqrt(E.DIM)
            z = z + torch.full_like(z, -math.inf).triu(1)
            a.append(z.softmax(1) @ v[i:j, kv])
    a = torch.cat([torch.cat(a[n:n + E.HEADS], 1) for n in range(0, len(a), E.HEADS)])
    y = x + E.ALPHA * (a @ p["wo"])
    h = _norm(y) * p["pre2"]
    y = y + E.ALPHA * (((h @ p["w1"]) * (h @ p["w2"])) @ p["w3"])
    logits = _norm(y) * p["pre3"] @ p["table"].T
    log_p = (teacher / E.TAU).log_softmax(1)
    log_s = (logits / E.TAU).log_softmax(1).gather(1, ids.long().clamp(min=0))
    loss = E.TAU ** 2 * (log_p.exp() * (log_p - log_s)).sum(1)
    return torch.where(ids[:, 0] >= 0, loss, 0.0)


def test_gradients(dev):
    """Relative to each gradient's norm within 1e-4: some twenty float32 stages of sums of at most some
    hundred terms, gamma(300) = 1.8e-5 each at the worst, of either sign."""
    gen = torch.Generator().manual_seed(1)
    p, data = E.parameters(gen, dev), E.batch(gen, dev)
    for k in p:  # weights of norms away from one
        if p[k].dim() == 1:
            p[k] = (1 + 0.3 * torch.randn(len(p[k]), generator=gen)).to(dev)
    loss, g = E.step(p, *data)
    wide = {k: v.double().cpu().requires_grad_() for k, v in p.items()}
    tokens, ids, teacher, cu, table, positions = (t.cpu() for t in data)
    want = _plain(wide, tokens, ids, teacher.double(), cu, table.double(), positions)
    want.mean().backward()
    assert (ids[:, 0] < 0).sum() == (tokens < 0).sum() == 15
    assert ((loss.double().cpu() - want.detach()).abs() <= 1e-4 * want.detach().mean()).all()
    assert set(g) == set(p)
    for k in p:
        d = (g[k].double().cpu() - wide[k].grad).norm() / wide[k].grad.norm()
        assert d <= 1e-4, (k, d.item())


def test_trains(dev):
    losses = E.train(12)
    assert len(losses) == 12 and all(math.isfinite(v) and v > 0 for v in losses)
