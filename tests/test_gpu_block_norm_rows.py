"""The norms around a block at their ends of the rows: none, where the gradients of the weights and of
a gate for each channel are zeros, whatever operands are left out."""
import ctypes

import pytest
import torch

from katsu_amd import _abi

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
