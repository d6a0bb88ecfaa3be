"""Attention and its gradient on operands that share memory between tokens or heads (broadcast ones
and overlapping windows), whose rows past a sequence's end are no zeros in a tile, and on keys that
every query sees with probability zero."""
import math

import pytest
import torch

from katsu_amd import ops
from tests.attention_ref import assert_close, backward, forward, starts

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16]
LENS = [45, 100, 1, 70]  # none a multiple of a tile's rows


def _cu(lens, dev):
    return torch.tensor(starts(lens), dtype=torch.int32, device=dev)


def _shared(shape, how, g, dt):
    """A [tokens, heads, channels] tensor whose tokens are one row, whose heads are one, or
    whose tokens are windows that begin 8 values after each other."""
    t, h, d = shape
    if how == "tokens":
        return torch.randn(1, h, d, generator=g).to(dt), lambda x: x.expand(t, h, d)
    if how == "heads":
        return torch.randn(t, 1, d, generator=g).to(dt), lambda x: x.expand(t, h, d)
    return (torch.randn(h, t * 8 + d, generator=g).to(dt),
            lambda x: x.as_strided((t, h, d), (8, t * 8 + d, 1)))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("d", [64, 128, 40, 16])
@pytest.mark.parametrize("which", ["q", "k", "v", "dout"])
@pytest.mark.parametrize("how", ["tokens", "heads", "windows"])
@pytest.mark.parametrize("causal", [True, False])
def test_shared_memory(dev, dt, d, which, how, causal):
    heads, kv, t = 4, 2, sum(LENS)
    g = torch.Generator().manual_seed(4)
    host, card = {}, {}
    for name in ("q", "k", "v", "dout"):
        shape = (t, kv if name in ("k", "v") else heads, d)
        if name == which:
            base, view = _shared(shape, how, g, dt)
            host[name], card[name] = view(base), view(base.to(dev))
        else:
            host[name] = torch.randn(*shape, generator=g).to(dt)
            card[name] = host[name].to(dev)
    assert card[which].stride() == host[which].stride()
    print(dt, d, which, how, causal, flush=True)
    seqs = dict(cu_q=_cu(LENS, dev), cu_k=_cu(LENS, dev), causal=causal)
    q, k, v = card["q"], card["k"], card["v"]
    out, lse = ops.attention(q, k, v, **seqs)
    got = ops.attention_backward(card["dout"], q, k, v, out, lse, **seqs)
    ops3 = [host[n] for n in ("q", "k", "v")]
    ro, rl, to, tl = forward(*ops3, LENS, LENS, causal, d ** -0.5)
    assert_close(out, ro, to, "out")
    assert_close(lse, rl, tl, "lse")
    want, tol = backward(host["dout"], *ops3, LENS, LENS, causal, d ** -0.5)
    for name, a, b, c in zip(("dq", "dk", "dv"), got, want, tol):
        assert_close(a, b, c, name)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("d", [64, 128, 40, 16])
@pytest.mark.parametrize("t", [45, 100])
def test_seen_key_without_weight(dev, dt, d, t):
    """A key whose scores are all -inf (its first channel is -inf, the queries' positive) has
    probability zero: its dk and dv are zeros, and the others' as if it were not there."""
    heads, kv, at = 4, 2, 20
    g = torch.Generator().manual_seed(5)
    q, k, v, do = (torch.randn(t, h, d, generator=g).to(dt) for h in (heads, kv, kv, heads))
    q[..., 0] = q[..., 0].abs() + 0.5
    k[at, :, 0] = -math.inf
    keep = [i for i in range(t) if i != at]
    qd, kd, vd = (x.to(dev) for x in (q, k, v))
    out, lse = ops.attention(qd, kd, vd, causal=False)
    _, dk, dv = ops.attention_backward(do.to(dev), qd, kd, vd, out, lse, causal=False)
    ro, rl, to, tl = forward(q, k[keep], v[keep], [t], [t - 1], False, d ** -0.5)
    assert_close(out, ro, to, "out")
    assert_close(lse, rl, tl, "lse")
    want, tol = backward(do, q, k[keep], v[keep], [t], [t - 1], False, d ** -0.5)
    assert_close(dk[keep], want[1], tol[1], "dk")
    assert_close(dv[keep], want[2], tol[2], "dv")
    assert (dk[at] == 0).all() and (dv[at] == 0).all()
