"""Outputs of the norms of heads that share memory with another operand: refused.  The allowed ones, and
operands between each other's places: taken."""
import ctypes
import itertools

import pytest
import torch

from katsu_amd import _abi, ops
from tests.test_lm_ends import _heads

L = _abi.lib()
BUF = (ctypes.c_float * 256)()
DIM, T = 4, 2


def _at(i):
    return ctypes.c_void_p(ctypes.addressof(BUF) + 4 * i)


def _forward(q, k, q_out, k_out, heads, k_heads, **kw):
    d = _heads(tokens=T, heads=heads, k_heads=k_heads, head_dim=DIM, rotary_dim=DIM, **kw)
    return L.katsu_hip_qk_norm_rotary_dev(d, _at(q), _at(k), None, None, _at(248), None, _at(q_out),
                                          _at(k_out), None)


def _backward(dq, dk, q, k, q_out, k_out, heads, k_heads, grads, **kw):
    d = _heads(tokens=T, heads=heads, k_heads=k_heads, head_dim=DIM, rotary_dim=DIM, **kw)
    return L.katsu_hip_qk_norm_rotary_bwd_dev(
        d, ctypes.byref(_abi.QkNormRotaryGrads(*grads)), _at(dq), _at(dk), _at(q), _at(k), None,
        None, _at(248), None, _at(q_out), _at(k_out), None, None, _at(240), 1 << 30, None)


# Two heads of q and k side by side in a token, or two tokens in a head, all 16 apart.
STRIDES = [dict.fromkeys(("q_stride", "k_stride", "q_out_stride", "k_out_stride"), s)
           for s in ((8, 4), (4, 8))]


@pytest.mark.parametrize("kw", STRIDES)
@pytest.mark.parametrize("by", [0, 4, 8, 12, -4, -12])
def test_refused(kw, by):
    """Without a GPU: only calls that are refused.  Each output at another operand, or a head or a
    token beside it; its own input's place (by 0) is allowed."""
    at = dict(q=16, k=48, q_out=80, k_out=112)
    for out, other in itertools.product(("q_out", "k_out"), at):
        if other == out or (by == 0 and other == out[0]):
            continue
        rc = _forward(**{**at, out: at[other] + by}, heads=2, k_heads=2, **kw)
        assert rc == _abi.E_INVALID, (out, other)
    at.update(dq=144, dk=176)
    grads = kw["q_stride"] * 2
    for out, other in itertools.product(("q_out", "k_out"), at):
        if other == out or (by == 0 and other in (out[0], "d" + out[0])):
            continue
        rc = _backward(**{**at, out: at[other] + by}, heads=2, k_heads=2, grads=grads, **kw)
        assert rc == _abi.E_INVALID, (out, other)


def test_refused_in_any_layout():
    """Heads with room between them, at one place."""
    kw = dict.fromkeys(("q_stride", "k_stride", "q_out_stride", "k_out_stride"), (24, 8))
    for out, other in (("q_out", "k"), ("k_out", "q"), ("q_out", "k_out")):
        at = dict(q=0, k=48, q_out=96, k_out=144)
        at[out] = at[other]
        assert _forward(**at, heads=2, k_heads=2, **kw) == _abi.E_INVALID
        assert _backward(192, 216, **at, heads=2, k_heads=2, grads=(24, 8, 24, 8),
                         **kw) == _abi.E_INVALID


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["tokens", "heads", "each"])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_taken(dev, dt, layout):
    """In place, with everything in one buffer: heads of all side by side in a token, head after head,
    or q, k and the outputs in turn within each head."""
    g = torch.Generator().manual_seed(1)
    t, h, d = 5, 3, 8
    table = ops.rotary_table(t, d, device=dev)
    base = torch.randn(t, 6 * h, d, generator=g).to(dt).to(dev)

    def parts():
        if layout == "tokens":
            return base.clone().view(t, 6, h, d).unbind(1)
        if layout == "heads":
            return base.clone().view(6, h, t, d).transpose(1, 2).unbind(0)
        return base.clone().view(t, h, 6, d).unbind(2)
    q, k = (v.contiguous() for v in parts()[:2])
    dq, dk = (v.contiguous() for v in parts()[4:])
    want = ops.qk_norm_rotary(q, k, table)
    back = ops.qk_norm_rotary_backward(dq, dk, q, k, table)[:2]
    rest = [v.clone() for v in parts()]
    for out in ((2, 3), (0, 1), (0, 3), (2, 1)):
        p = parts()
        got = ops.qk_norm_rotary(p[0], p[1], table, out_q=p[out[0]], out_k=p[out[1]])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(torch.equal(p[i], rest[i]) for i in range(6) if i not in out)
    for out in ((2, 3), (0, 1), (4, 5), (0, 5), (4, 1), (2, 5)):
        p = parts()
        got = ops.qk_norm_rotary_backward(p[4], p[5], p[0], p[1], table, out_q=p[out[0]],
                                          out_k=p[out[1]])[:2]
        assert all(torch.equal(a, b) for a, b in zip(got, back))
        assert all(torch.equal(p[i], rest[i]) for i in range(6) if i not in out)
    p = parts()
    for bad in ((p[1], p[3]), (p[2], p[0]), (p[2], p[2])):
        with pytest.raises(_abi.KatsuError):
            ops.qk_norm_rotary(p[0], p[1], table, out_q=bad[0], out_k=bad[1])
        with pytest.raises(_abi.KatsuError):
            ops.qk_norm_rotary_backward(p[4], p[5], p[0], p[1], table, out_q=bad[0], out_k=bad[1])
    # The same tensor as q and k, with outputs of their own.
    a, b = ops.qk_norm_rotary(q, q, table)
    assert torch.equal(a, want[0]) and torch.equal(b, want[0])
    with pytest.raises(_abi.KatsuError):
        ops.qk_norm_rotary(q, q, table, out_q=q)
