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
