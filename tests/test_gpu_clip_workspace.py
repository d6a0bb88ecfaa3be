"""Gradient clipping with the caller's workspace: the same bits as with the library's, the partial
sums in the caller's memory and nothing in the library's, refusals."""
import ctypes

import pytest
import torch

from katsu_amd import _abi, ops


def test_workspace_sizes():
    """Without a GPU: sizes, and what is refused before any launch."""
    L, n = _abi.lib(), ctypes.c_size_t(0)
    assert L.katsu_hip_clip_grad_norm_workspace(3, None) == _abi.E_INVALID
    assert L.katsu_hip_clip_grad_norm_workspace(1 << 40, ctypes.byref(n)) == _abi.E_INVALID
    assert ops.clip_workspace_bytes(0) == 0
    assert 0 < ops.clip_workspace_bytes(1) == ops.clip_workspace_bytes(128)
    assert ops.clip_workspace_bytes(129) == 2 * ops.clip_workspace_bytes(1)
    buf = (ctypes.c_double * 4)()
    p = ctypes.cast(buf, ctypes.c_void_p)
    kinds, counts = (ctypes.c_int32 * 1)(_abi.F32), (ctypes.c_size_t * 1)(4)
    ptr = (ctypes.c_void_p * 1)(p.value)
    assert L.katsu_hip_clip_grad_norm_ws_dev(
        kinds, ptr, ptr, counts, 1, 1.0, p, p, ops.clip_workspace_bytes(1) - 1,
        None) == _abi.E_INVALID


@pytest.mark.gpu
@pytest.mark.parametrize("counts", [[5], [40000, 3, 70001], [(37 * i) % 3000 for i in range(300)]])
def test_own_workspace(dev, counts):
    g = torch.Generator().manual_seed(1)
    grads = [torch.randn(n, generator=g).to([torch.float32, torch.bfloat16][i % 2]).to(dev)
             for i, n in enumerate(counts)]
    a, b = ([torch.empty_like(t) for t in grads] for _ in range(2))
    norm = ops.clip_grad_norm(grads, 1.0, out=a)
    ws = torch.zeros(ops.clip_workspace_bytes(len(grads)) // 8, dtype=torch.float64, device=dev)
    own = ops.clip_grad_norm(grads, 1.0, out=b, workspace=ws)
    assert torch.equal(norm, own) and all(torch.equal(x, y) for x, y in zip(a, b))
    # The sums of squares are there, one for each block: their total is the norm's square, within
    # both sums' rounding in any order (2 n 2^-53, n below 2^19).
    total = sum(t.double().square().sum() for t in grads)
    assert (ws.sum() - total).abs() <= 2.0 ** -33 * total
    with pytest.raises(_abi.KatsuError) as e:
        ops.clip_grad_norm(grads, 1.0, out=b, workspace=ws[:-1])
    assert e.value.status == _abi.E_INVALID
