"""Outputs of rotary and of the norms of heads whose heads share memory: refused, and no others."""
import ctypes
import itertools

import pytest
import torch

from katsu_amd import _abi, ops
from tests.test_lm_ends import _heads
from tests.test_lm_strides import L, P, Q, _rotary

DIM = 4
# tokens, heads, their strides
LAYOUTS = [(n, h, s, t) for n, h in ((1, 3), (3, 1), (2, 2), (3, 2), (2, 3), (3, 3))
           for s, t in itertools.product((1, 3, 4, 5, 7, 8, 9, 11, 12, 13, 16, 20), repeat=2)]


def _overlap(n, h, s, t):
    """Place by place."""
    at = [i * s + j * t + c for i in range(n) for j in range(h) for c in range(DIM)]
    return len(set(at)) < len(at)


def test_layouts():
    """Of each kind: side by side, tokens within heads, and some that are neither."""
    free = [v for v in LAYOUTS if not _overlap(*v)]
    assert (3, 2, 8, 4) in free and (3, 2, 4, 12) in free and (3, 2, 8, 12) in free
    assert 100 < len(free) < len(LAYOUTS) - 100


def test_refused():
    """Without a GPU: only calls that are refused."""
    for n, h, s, t in (v for v in LAYOUTS if _overlap(*v)):
        out = dict(tokens=n, heads=h, k_heads=h, head_dim=DIM, rotary_dim=DIM)
        for which in ("q", "k"):
            other = {"q_out_stride": (16, 4), "k_out_stride": (16, 4), which + "_out_stride": (s, t)}
            assert _rotary(**out, **other) == _abi.E_INVALID, (n, h, s, t)
            d = _heads(**out, **other)
            assert L.katsu_hip_qk_norm_rotary_dev(d, P, P, None, None, P, None, Q, Q,
                                                  None) == _abi.E_INVALID, (n, h, s, t)
            g = ctypes.byref(_abi.QkNormRotaryGrads(16, 4, 16, 4))
            assert L.katsu_hip_qk_norm_rotary_bwd_dev(
                d, g, P, P, P, P, None, None, P, None, Q, Q, None, None, P, 1 << 30,
                None) == _abi.E_INVALID, (n, h, s, t)


@pytest.mark.gpu
@pytest.mark.parametrize("far", [0, 1 << 31])
def test_taken(dev, far):
    """All others, with the results of a contiguous output, also where strides pass 2^31."""
    table = ops.rotary_table(8, DIM, device=dev)
    x = torch.randn(3, 3, DIM, device=dev)
    buf = torch.empty((2 * far or 0) + 200, device=dev)
    layouts = [v for v in LAYOUTS if not _overlap(*v)]
    if far:
        layouts = [(3, h, s + far, t) for n, h, s, t in layouts if n == 3]
    for n, h, s, t in layouts:
        q = x[:n, :h]
        want = (ops.rotary(q, None, table)[0], ops.qk_norm_rotary(q, None, table)[0],
                ops.qk_norm_rotary_backward(q, None, q, None, table)[0])
        out = buf.as_strided((n, h, DIM), (s, t, 1))
        for i in range(3):
            out.fill_(7.0)
            if i == 0:
                ops.rotary(q, None, table, out_q=out)
            elif i == 1:
                ops.qk_norm_rotary(q, None, table, out_q=out)
            else:
                ops.qk_norm_rotary_backward(q, None, q, None, table, out_q=out)
            assert torch.equal(out, want[i]), (n, h, s, t, i)
