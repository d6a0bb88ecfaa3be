"""The language-model operators' C entry points without a GPU: arguments that they refuse before any
launch, empty problems, and workspace sizes.  No kernel is launched here."""
import ctypes

import pytest

from katsu_amd import _abi

L = _abi.lib()
BUF = (ctypes.c_float * 16)()
P = ctypes.cast(BUF, ctypes.c_void_p)
SZ = ctypes.c_size_t


def _attention(**kw):
    d = dict(dtype=_abi.F32, causal=1, heads=4, kv_heads=2, head_dim=64, seqs=1, tokens_q=8,
             tokens_k=8, q_stride=(256, 64), k_stride=(128, 64), v_stride=(128, 64),
             out_stride=(256, 64), scale=0.125)
    d.update(kw)
    return _abi.Attention(**d)


@pytest.mark.parametrize("kw", [
    dict(dtype=2), dict(heads=0), dict(kv_heads=0), dict(kv_heads=3), dict(head_dim=0),
    dict(head_dim=129), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
    dict(scale=float("inf")), dict(tokens_q=1 << 31), dict(tokens_k=1 << 31), dict(seqs=1 << 31),
    dict(q_stride=(-1, 64)), dict(k_stride=(128, -64)), dict(heads=1 << 20, kv_heads=1 << 20),
    dict(tokens_q=(1 << 31) - 1, heads=65535, kv_heads=1)])
def test_attention_refuses(kw):
    d = _attention(**kw)
    n = SZ(0)
    g = _abi.AttentionGrads((256, 64), (256, 64), (128, 64), (128, 64))
    for rc in (L.katsu_hip_attention_fwd_workspace(ctypes.byref(d), ctypes.byref(n)),
               L.katsu_hip_attention_bwd_workspace(ctypes.byref(d), ctypes.byref(n)),
               L.katsu_hip_attention_fwd_dev(ctypes.byref(d), P, P, P, None, None, None, P, P, P, 0,
                                             None),
               L.katsu_hip_attention_bwd_dev(ctypes.byref(d), ctypes.byref(g), P, P, P, P, P, P,
                                             None, None, P, P, P, P, 0, None)):
        assert rc == _abi.E_INVALID


def test_attention_pointers_and_starts():
    d, g = _attention(), _abi.AttentionGrads((256, 64), (256, 64), (128, 64), (128, 64))

    def fwd(d, q=P, k=P, v=P, cu_q=None, cu_k=None, out=P):
        return L.katsu_hip_attention_fwd_dev(ctypes.byref(d), q, k, v, cu_q, cu_k, None, out, None,
                                             P, 0, None)
    for kw in (dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(cu_q=P),
               dict(cu_k=P)):
        assert fwd(d, **kw) == _abi.E_INVALID
    assert fwd(_attention(seqs=2)) == _abi.E_INVALID  # starts are needed
    assert L.katsu_hip_attention_fwd_dev(None, P, P, P, None, None, None, P, P, P, 0,
                                         None) == _abi.E_INVALID
    bad = _abi.AttentionGrads((256, 64), (-1, 64), (128, 64), (128, 64))
    for gg, ptrs in ((bad, (P,) * 6), (g, (None,) + (P,) * 5), (g, (P,) * 5 + (None,))):
        assert L.katsu_hip_attention_bwd_dev(ctypes.byref(d), ctypes.byref(gg), *ptrs, None, None, P,
                                             P, P, P, 0, None) == _abi.E_INVALID
    # Outputs whose places are not their own.
    for kw in (dict(out_stride=(256, 0)), dict(out_stride=(0, 64))):
        assert fwd(_attention(**kw)) == _abi.E_INVALID
    for f in ("dq_stride", "dk_stride", "dv_stride"):
        gg = _abi.AttentionGrads((256, 64), (256, 64), (128, 64), (128, 64))
        setattr(gg, f, (ctypes.c_int64 * 2)(256, 0))
        assert L.katsu_hip_attention_bwd_dev(ctypes.byref(d), ctypes.byref(gg), *(P,) * 6, None,
                                             None, P, P, P, P, 0, None) == _abi.E_INVALID
    # A workspace that is too small.
    n = SZ(0)
    assert L.katsu_hip_attention_bwd_workspace(ctypes.byref(d), ctypes.byref(n)) == _abi.OK
    assert n.value > 0
    assert L.katsu_hip_attention_bwd_dev(ctypes.byref(d), ctypes.byref(g), P, P, P, P, P, P, None,
                                         None, P, P, P, P, n.value - 1, None) == _abi.E_INVALID
    # No queries or no sequences: nothing to do.
    assert fwd(_attention(tokens_q=0), q=None, out=None) == _abi.OK
    assert fwd(_attention(seqs=0), q=None, out=None) == _abi.OK


def test_rotary_refuses():
    ok = dict(dtype=_abi.F32, interleaved=0, inverse=0, tokens=2, heads=2, k_heads=0, head_dim=8,
              rotary_dim=8, length=4, q_stride=(16, 8), q_out_stride=(16, 8))

    def call(q=P, table=P, out=P, **kw):
        d = _abi.Rotary(**{**ok, **kw})
        return L.katsu_hip_rotary_dev(ctypes.byref(d), q, None, table, None, out, None, None)
    for kw in (dict(dtype=7), dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=10),
               dict(head_dim=0), dict(length=0), dict(length=1 << 31), dict(tokens=1 << 31),
               dict(heads=65536), dict(heads=60000, head_dim=128, rotary_dim=2), dict(q=None),
               dict(table=None), dict(out=None), dict(k_heads=1)):
        assert call(**kw) == _abi.E_INVALID, kw
    assert call(tokens=0, q=None) == _abi.OK
    t = L.katsu_hip_rotary_table_f32_dev
    for args in ((P, 4, 7, 1e4, 1.0, 0), (P, 4, 0, 1e4, 1.0, 0), (P, 4, 8, 0.0, 1.0, 0),
                 (P, 4, 8, 1e4, 0.9, 0), (None, 4, 8, 1e4, 1.0, 0), (P, 1 << 31, 8, 1e4, 1.0, 0)):
        assert t(*args, None) == _abi.E_INVALID, args
    assert t(None, 0, 8, 1e4, 1.0, 0, None) == _abi.OK


def test_block_norm_refuses():
    def fwd(x=P, o=P, gate=None, w_pre=None, y=P, h=None, **kw):
        d = _abi.BlockNorm(**{**dict(dtype=_abi.F32, gate_rows=0, rows=2, cols=4, alpha=1.0,
                                     eps=1e-6), **kw})
        return L.katsu_hip_block_norm_dev(ctypes.byref(d), x, o, gate, None, w_pre, y, h, None, None)
    for kw in (dict(dtype=3), dict(gate_rows=3), dict(gate_rows=-1), dict(cols=0),
               dict(cols=16385), dict(rows=1 << 31), dict(alpha=float("nan")), dict(eps=-1.0),
               dict(x=None), dict(o=None), dict(y=None), dict(w_pre=P), dict(gate_rows=1)):
        assert fwd(**kw) == _abi.E_INVALID, kw
    assert fwd(rows=0, x=None) == _abi.OK
    d = _abi.BlockNorm(_abi.BF16, 1, 100, 64, 1.0, 0.0)
    n = SZ(0)
    assert L.katsu_hip_block_norm_bwd_workspace(ctypes.byref(d), ctypes.byref(n)) == _abi.OK
    ptrs = [P] * 14
    assert L.katsu_hip_block_norm_bwd_dev(ctypes.byref(d), *ptrs, n.value - 1,
                                          None) == _abi.E_INVALID
    for i in (0, 1, 2, 3, 4, 5, 8, 9, 10, 11, 12):
        some = [None if j == i else P for j in range(14)]
        assert L.katsu_hip_block_norm_bwd_dev(ctypes.byref(d), *some, n.value,
                                              None) == _abi.E_INVALID, i


def test_clip_refuses():
    kinds, counts = (ctypes.c_int32 * 1)(_abi.F32), (SZ * 1)(4)
    ptr, null = (ctypes.c_void_p * 1)(P.value), (ctypes.c_void_p * 1)(None)

    def call(kinds=kinds, src=ptr, dst=ptr, counts=counts, norm=P, max_norm=1.0):
        return L.katsu_hip_clip_grad_norm_dev(kinds, src, dst, counts, 1, max_norm, norm, None)
    for kw in (dict(kinds=(ctypes.c_int32 * 1)(5)), dict(src=null), dict(dst=null), dict(src=None),
               dict(counts=None), dict(norm=None), dict(max_norm=-1.0),
               dict(max_norm=float("nan")), dict(counts=(SZ * 1)((1 << 38) + 1))):
        assert call(**kw) == _abi.E_INVALID, kw
