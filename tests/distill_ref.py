"""Distillation's loss and gradient in float64, with bounds on what float32 arithmetic may be off."""
import math

import torch

U = 2.0 ** -24


def gamma(n):
    return n * U / (1 - n * U)


def _softmax(x, mask):
    """(probabilities, distances below the largest, log of the total, mean distance) over the mask's
    places; zeros where it has none."""
    some = mask.any(1, keepdim=True)
    x = x.masked_fill(~mask, -math.inf)
    top = torch.where(some, x.amax(1, keepdim=True), 0.0)
    d = (top - x).masked_fill(~mask, math.inf)
    total = (-d).exp().sum(1, keepdim=True)
    p = torch.where(some, (-d).exp() / torch.where(some, total, 1.0), 0.0)
    d = torch.where(mask, d, 0.0)
    return p, d, torch.where(some, total.log(), 0.0), (p * d).sum(1, keepdim=True)


def reference(z, ids, t, tau, dloss):
    """(loss, gradient, their bounds); finite logits but for -inf.

    A difference of logits over tau has an error of 4 u of itself, its exponential that and 2^-22 more,
    so that a total's terms are off by 4 u times their mean distance, weighted as in the total: far
    ones add nothing.  A total adds gamma of its longest chain, a thread's share of the row and 16
    joins, and 2^-22 for each time that its reference moves: once for four values of a thread at most,
    and in the joins.  Logarithms and short sums round once each.  What is below 2^-126 may be none."""
    rows, v = z.shape
    real = (ids >= 0) & (ids < v)
    td = t.double().masked_fill(~real, -math.inf)
    some = (real & (td > -math.inf)).any(1)
    mask = real & some[:, None] & (td > -math.inf)
    p, dt, lt, mean_t = _softmax(td / tau, mask)
    all_p, dz, lz, mean_z = _softmax(z.double() / tau, z.double() > -math.inf)
    at = ids.long().clamp(0, max(v - 1, 0))
    zk = torch.where(mask, dz.gather(1, at), 0.0)
    gone = mask & (z.double().gather(1, at) == -math.inf) & (p > 0)
    terms = torch.where(p > 0, (zk - dt) - lt + lz, 0.0)
    loss = torch.where(gone.any(1), math.inf, (p * terms).sum(1) * tau ** 2)

    share = -(-v // (128 if v <= 16384 else 256))
    rel_l = gamma(share + 16) + 4 * U * mean_z + (-(-share // 4) + 26) * 2.0 ** -22
    rel_t = gamma(ids.shape[1]) + 2.0 ** -21 + 4 * U * mean_t
    rel_p = rel_t + 4 * U * dt + 2.0 ** -21 + gamma(ids.shape[1])
    each = 6 * U * (dt + zk + lt.abs() + lz.abs()) + rel_l + rel_t
    ltol = (p * (each + rel_p * terms.abs()) + 2.0 ** -126 * terms.abs()).sum(1) * tau ** 2
    ltol = ltol + 6 * U * loss.abs().nan_to_num(posinf=0.0) + 2.0 ** -147

    want = torch.zeros_like(dz).scatter_add_(1, at, p)
    wtol = torch.zeros_like(dz).scatter_add_(1, at, p * rel_p)
    g = (tau * dloss.double())[:, None]
    grad = torch.where(some[:, None], (all_p - want) * g, 0.0)
    gtol = (all_p * (4 * U * dz + 2.0 ** -21 + rel_l) + wtol + 2.0 ** -120) * g.abs()
    gtol = gtol + (torch.finfo(z.dtype).eps / 2 + 2 * U) * (grad.abs() + gtol) + 2.0 ** -126
    return (torch.where(some, loss, 0.0), grad, torch.where(some, ltol, 0.0),
            torch.where(some[:, None], gtol, 0.0))


def close(got, want, tol):
    got = got.double().cpu()
    err = (got - want).abs()
    bad = ~((got == want) | (err <= tol))
    assert not bad.any(), (err - tol)[bad].max()
