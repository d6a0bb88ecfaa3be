"""Workspaces that the language-model operators refuse: memory that is not their device's, tensors with
fewer bytes than they show, addresses inside a 16-byte piece.  Nothing is launched with them."""
import ctypes

import pytest
import torch

from katsu_amd import _abi, ops


def test_alignment():
    """Without a GPU: each entry refuses an unaligned workspace before any launch."""
    L = _abi.lib()
    buf = (ctypes.c_char * 65536)()
    base = (ctypes.addressof(buf) + 15) // 16 * 16
    p = ctypes.c_void_p(base)
    s = ((64, 64), (64, 64), (64, 64), (64, 64))
    d = _abi.Attention(_abi.F32, 1, 1, 1, 64, 1, 1, 4096, *s, 0.125)
    g = _abi.AttentionGrads(*s)
    n = _abi.BlockNorm(_abi.F32, 0, 2, 4, 1.0, 0.0)
    kinds, counts = (ctypes.c_int32 * 1)(_abi.F32), (ctypes.c_size_t * 1)(4)
    ptr = (ctypes.c_void_p * 1)(base)
    for off in (1, 2, 4, 8):
        w = ctypes.c_void_p(base + off)
        for rc in (
                L.katsu_hip_attention_fwd_dev(ctypes.byref(d), p, p, p, None, None, None, p, p, w,
                                              1 << 40, None),
                L.katsu_hip_attention_bwd_dev(ctypes.byref(d), ctypes.byref(g), p, p, p, p, p, p,
                                              None, None, p, p, p, w, 1 << 40, None),
                L.katsu_hip_block_norm_bwd_dev(ctypes.byref(n), *[p] * 13, w, 1 << 40, None),
                L.katsu_hip_clip_grad_norm_ws_dev(kinds, ptr, ptr, counts, 1, 1.0, p, w, 1 << 40,
                                                  None)):
            assert rc == _abi.E_INVALID, off


@pytest.mark.gpu
def test_memory(dev):
    q = torch.randn(100, 2, 64, device=dev)
    out, lse = ops.attention(q, q, q)
    x = torch.randn(20, 64, device=dev)
    w = torch.ones(64, device=dev)
    _, h, stats = ops.block_norm(x, x, w_pre=w)
    size = 1 << 24
    for ws in (torch.empty(size, dtype=torch.uint8),
               torch.empty(1, dtype=torch.uint8, device=dev).expand(size),
               torch.empty(2 * size, dtype=torch.uint8, device=dev)[::2]):
        for call in (lambda: ops.attention(q, q, q, workspace=ws),
                     lambda: ops.attention_backward(q, q, q, q, out, lse, workspace=ws),
                     lambda: ops.block_norm_backward(x, h, x, x, stats, w_pre=w, workspace=ws),
                     lambda: ops.clip_grad_norm([x], 1.0, workspace=ws)):
            with pytest.raises(ValueError):
                call()
