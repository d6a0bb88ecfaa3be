"""Strides that the language-model operators refuse, and odd ones that they take."""
import ctypes

import pytest
import torch

from katsu_amd import _abi, ops

L = _abi.lib()
BUF = (ctypes.c_float * 64)()
P = ctypes.c_void_p(ctypes.addressof(BUF))
Q = ctypes.c_void_p(ctypes.addressof(BUF) + 128)


def _rotary(q_in=P, q_out=Q, k_in=P, k_out=Q, **kw):
    d = dict(dtype=_abi.F32, interleaved=0, inverse=0, tokens=2, heads=2, k_heads=2, head_dim=4,
             rotary_dim=4, length=4, q_stride=(8, 4), k_stride=(8, 4), q_out_stride=(8, 4),
             k_out_stride=(8, 4))
    d.update(kw)
    return L.katsu_hip_rotary_dev(ctypes.byref(_abi.Rotary(**d)), q_in, k_in, P, None, q_out,
                                  k_out, None)


@pytest.mark.parametrize("which", ["q_out", "k_out"])
@pytest.mark.parametrize("stride", [(0, 4), (8, 0), (-8, 4), (8, -4)])
def test_rotary_refuses_outputs(which, stride):
    """Without a GPU: places that two values share, or lie before the tensor."""
    assert _rotary(**{which + "_stride": stride}) == _abi.E_INVALID


def test_rotary_refuses_inputs():
    for name in ("q_stride", "k_stride"):
        assert _rotary(**{name: (-8, 4)}) == _abi.E_INVALID
    # The input's memory in another order.
    assert _rotary(q_out=P, q_out_stride=(4, 8)) == _abi.E_INVALID
    assert _rotary(k_out=P, k_out_stride=(4, 8)) == _abi.E_INVALID


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_rotary_single_places(dev, dt):
    """Strides of a single token or head do not matter, in place or not; a broadcast input is one."""
    table = ops.rotary_table(8, 8, device=dev)
    x = torch.randn(1, 1, 24, device=dev).to(dt)
    want, _ = ops.rotary(x, None, table)
    flat = x.clone().flatten()
    view = flat.as_strided((1, 1, 24), (0, 0, 1))
    got, _ = ops.rotary(view, None, table, out_q=flat.as_strided((1, 1, 24), (24, 7, 1)))
    assert torch.equal(got, want)
    q = torch.randn(5, 1, 24, device=dev).to(dt).expand(5, 3, 24)
    a, b = ops.rotary(q, x.expand(5, 2, 24), table)
    c, d = ops.rotary(q.contiguous(), x.expand(5, 2, 24).contiguous(), table)
    assert torch.equal(a, c) and torch.equal(b, d)
    with pytest.raises(_abi.KatsuError):
        ops.rotary(q, None, table, out_q=x.expand(5, 3, 24))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 20])
def test_attention_far_tokens(dev, dt, d):
    """Tokens more than 2^31 values apart: all operands and outputs in one buffer of long rows."""
    t, heads, kv = 3, 4, 2
    step = (1 << 31) + 1024
    n = {"q": heads, "k": kv, "v": kv, "do": heads, "out": heads, "dq": heads, "dk": kv, "dv": kv}
    flat = torch.empty((t - 1) * step + sum(n.values()) * d, dtype=dt, device=dev)
    far, at = {}, 0
    for name, h in n.items():
        far[name] = flat.as_strided((t, h, d), (step, d, 1), at)
        at += h * d
    g = torch.Generator().manual_seed(1)
    near = {}
    for name in ("q", "k", "v", "do"):
        near[name] = torch.randn(t, n[name], d, generator=g).to(dt).to(dev)
        far[name].copy_(near[name])
    out, lse = ops.attention(near["q"], near["k"], near["v"])
    want = ops.attention_backward(near["do"], near["q"], near["k"], near["v"], out, lse)
    _, far_lse = ops.attention(far["q"], far["k"], far["v"], out=far["out"])
    got = ops.attention_backward(far["do"], far["q"], far["k"], far["v"], far["out"], far_lse,
                                 dq=far["dq"], dk=far["dk"], dv=far["dv"])
    # The copy to LDS is another one, and with it the blocks of 32 channels and the order of the
    # sums of at most 64 products: a few roundings. Rows of 40 bytes take the same copy near and far.
    tol = 0 if d == 20 and dt is torch.bfloat16 else 64 * 2.0 ** -24 + (
        0 if dt is torch.float32 else 2.0 ** -7)
    for a, b in zip((far["out"], far_lse, *got), (out, lse, *want)):
        assert ((a - b).abs() <= tol * (b.abs() + 1)).all()


@pytest.mark.gpu
def test_no_channels(dev):
    """A refusal of ops' own, not a division by zero."""
    q = torch.empty(3, 2, 0, device=dev)
    with pytest.raises(ValueError):
        ops.attention(q, q, q)
    with pytest.raises(ValueError):
        ops.attention_workspace_bytes(q, q, q)
