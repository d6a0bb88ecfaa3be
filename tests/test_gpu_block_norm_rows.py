"""The norms around a block with the most rows, and with none, where the gradients of the weights and of
a gate for each channel are zeros, whatever operands are left out."""
import ctypes

import pytest
import torch

from katsu_amd import _abi, ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("post,pre", [(False, False), (True, False), (False, True), (True, True)])
def test_no_rows(dev, dt, post, pre):
    """No operand but the weights is there, the gate neither: dgate is what gate_rows asks for, and
    a weight that is not there has no gradient, wherever its pointer leads."""
    cols = 70
    dgate, dpost, dpre = (torch.full((cols,), 7.0, dtype=dt, device=dev) for _ in range(3))
    w = torch.ones(cols, dtype=dt, device=dev)
    d = _abi.BlockNorm(_abi.F32 if dt is torch.float32 else _abi.BF16, 1, 0, cols, 1.0, 0.0)
    assert _abi.lib().katsu_hip_block_norm_bwd_dev(
        ctypes.byref(d), None, None, None, None, None, None, w.data_ptr() if post else None,
        w.data_ptr() if pre else None, None, None, dgate.data_ptr(),
        dpost.data_ptr(), dpre.data_ptr(), None, 0,
        torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert (dgate == 0).all()
    assert (dpost == (0 if post else 7)).all() and (dpre == (0 if pre else 7)).all()


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_many_rows(dev, dt):
    """More rows than one launch's threads along its first axis cover: norms of one head's one
    channel, which are its sign (but for eps)."""
    rows = (1 << 26) + 5
    o = torch.ones(rows, 1, dtype=dt, device=dev)
    o[1::2] = -2
    x = torch.full_like(o, 0.5)
    w = torch.full((1,), 3.0, dtype=dt, device=dev)
    y, h, stats = ops.block_norm(x, o, w_post=w, w_pre=w, eps=0.0)
    # y = 0.5 + 3 or 0.5 - 3 and h = 3 or -3, within the roundings of 1/sqrt and three products.
    for got, even, odd in ((y, 3.5, -2.5), (h, 3.0, -3.0), (stats[0, :, None], 1.0, 0.5),
                           (stats[1, :, None], 1 / 3.5, 1 / 2.5)):
        unit = 8 * 2.0 ** -24 + (2.0 ** -8 if got.dtype is torch.bfloat16 else 0)
        assert ((got[::2] - even).abs() <= unit * abs(even)).all()
        assert ((got[1::2] - odd).abs() <= unit * abs(odd)).all()
