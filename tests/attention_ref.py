"""Attention over packed sequences in float64, from its definition, and error bounds of a
float32 or bfloat16 evaluation of it.

Bounds.  u = 2^-24, gamma(n) = n u / (1 - n u) as for any float32 sum.  A score's error is at most
ds = gamma(D + 4) scale sum|q||k| + 4 u |s|: its products, scaling, and the rounding of the
exponential's argument.  A probability is a quotient of exponentials: relative error at most
e = 2 ds + gamma(Lk) + 2^-20 (the hardware exponential and quotient).  Where the probabilities are
operands in bfloat16, 2^-8 more.  A sum of n products of such factors adds gamma(n), and an output
in bfloat16 2^-8 of itself.  In the backward pass the probabilities come from the forward pass's
lse, whose error is e as well: 2 e in all; delta = do.o takes the error of the out it is given.
"""
import math

import torch

U = 2.0 ** -24


def gamma(n):
    return n * U / (1 - n * U)


def starts(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def visible(lq, lk, causal):
    i = torch.arange(lq)[:, None]
    j = torch.arange(lk)[None, :]
    return (j <= i + lk - lq) if causal else torch.ones(lq, lk, dtype=torch.bool)


def forward(q, k, v, q_lens, k_lens, causal, scale, slots=None):
    """(out, lse, bound of out, bound of lse) in float64; q, k, v any type, on the CPU.
    slots: tokens kept for each sequence's keys (its length if None)."""
    half = q.dtype is torch.bfloat16
    q, k, v = q.double(), k.double(), v.double()
    tq, heads, d = q.shape
    group = heads // k.shape[1]
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full((heads, tq), -math.inf, dtype=torch.float64)
    ltol = torch.zeros((heads, tq), dtype=torch.float64)
    qa, ka = 0, 0
    for n, (lq, lk) in enumerate(zip(q_lens, k_lens)):
        see = visible(lq, lk, causal)
        for h in range(heads):
            if lq == 0 or lk == 0:
                continue
            Q, K, V = q[qa:qa + lq, h], k[ka:ka + lk, h // group], v[ka:ka + lk, h // group]
            s = (Q @ K.T) * scale
            ds = gamma(d + 4) * scale * (Q.abs() @ K.abs().T) + 4 * U * s.abs()
            s = s.masked_fill(~see, -math.inf)
            some = see.any(1)
            m = torch.where(some, s.max(1).values, 0.0)
            p = (s - m[:, None]).exp()
            tot = p.sum(1)
            p = p / torch.where(some, tot, 1.0)[:, None]
            e = 2 * ds.masked_fill(~see, 0).max(1).values + gamma(lk) + 2.0 ** -20
            e = e + (2.0 ** -8 if half else 0)
            o = p @ V
            out[qa:qa + lq, h] = o
            tol[qa:qa + lq, h] = (e + gamma(lk))[:, None] * (p @ V.abs()) + (
                2.0 ** -8 if half else U) * o.abs()
            lse[h, qa:qa + lq] = torch.where(some, m + tot.log(), -math.inf)
            ltol[h, qa:qa + lq] = torch.where(some, e + 4 * U * (m.abs() + tot.log().abs()), 0.0)
        qa += lq
        ka += lk if slots is None else slots[n]
    return out, lse, tol, ltol


def backward(do, q, k, v, q_lens, k_lens, causal, scale):
    """((dq, dk, dv), their bounds) in float64."""
    half = q.dtype is torch.bfloat16
    w = 2.0 ** -8 if half else 0.0
    out, _, otol, ltol = forward(q, k, v, q_lens, k_lens, causal, scale)
    do, q, k, v = do.double(), q.double(), k.double(), v.double()
    heads, d = q.shape[1:]
    group = heads // k.shape[1]
    grads = [torch.zeros_like(t) for t in (q, k, v)]
    tols = [torch.zeros_like(t) for t in (q, k, v)]
    qa, ka = 0, 0
    for lq, lk in zip(q_lens, k_lens):
        see = visible(lq, lk, causal)
        for h in range(heads):
            if lq == 0 or lk == 0:
                continue
            at, kt = (slice(qa, qa + lq), h), (slice(ka, ka + lk), h // group)
            Q, K, V, G = q[at], k[kt], v[kt], do[at]
            s = ((Q @ K.T) * scale).masked_fill(~see, -math.inf)
            p = torch.where(see.any(1)[:, None], s.softmax(1), 0.0)
            e = 2 * (ltol[h, qa:qa + lq] - (0 if not half else 2.0 ** -8)).clamp(min=0)[:, None]
            dp = G @ V.T
            delta = (G * out[at]).sum(1, keepdim=True)
            ds = p * (dp - delta)
            edp = gamma(d + 4) * (G.abs() @ V.abs().T)
            ede = (G.abs() * (otol[at] + gamma(d + 4) * out[at].abs())).sum(1, keepdim=True)
            eds = (e + 8 * U + w) * ds.abs() + p * (edp + ede)
            grads[0][at] += scale * ds @ K
            tols[0][at] += scale * (eds + gamma(lk) * ds.abs()) @ K.abs()
            grads[1][kt] += scale * ds.T @ Q
            tols[1][kt] += scale * (eds + gamma(group * lq) * ds.abs()).T @ Q.abs()
            grads[2][kt] += p.T @ G
            tols[2][kt] += ((e + w + gamma(group * lq)) * p).T @ G.abs()
        qa, ka = qa + lq, ka + lk
    for g, t in zip(grads, tols):
        t += max(w, 4 * U) * g.abs()
    return grads, tols


def assert_close(got, ref, tol, what):
    got = got.double().cpu()
    bad = ~((got - ref).abs() <= tol)
    bad &= ~(got.isinf() & (got == ref))
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} beyond the bound, worst "
                           f"{((got - ref).abs() / tol)[bad].max().item():.2f} times it")
