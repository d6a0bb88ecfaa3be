"""Embedding, the norm of heads with their turn, and distillation: what their entry points refuse before
any launch, empty problems, and workspace sizes.  The C entry points need no GPU; no kernel is launched
with refused arguments."""
import ctypes

import pytest
import torch

from katsu_amd import _abi, ops

L = _abi.lib()
BUF = (ctypes.c_float * 64)()
P = ctypes.c_void_p((ctypes.addressof(BUF) + 15) // 16 * 16)
SZ = ctypes.c_size_t
NAN, INF, BIG = float("nan"), float("inf"), 1 << 41


def _embed(**kw):
    d = dict(dtype=_abi.F32, accumulate=0, tokens=4, vocab=8, cols=16, table_stride=16,
             out_stride=16, scale=1.0)
    return ctypes.byref(_abi.Embedding(**{**d, **kw}))


@pytest.mark.parametrize("kw", [
    dict(dtype=2), dict(accumulate=2), dict(accumulate=-1), dict(tokens=1 << 31),
    dict(vocab=1 << 31), dict(cols=0), dict(cols=1 << 31), dict(table_stride=-1),
    dict(out_stride=-16), dict(table_stride=BIG), dict(out_stride=BIG), dict(scale=NAN),
    dict(scale=INF)])
def test_embedding_refuses(kw):
    n = SZ(0)
    assert L.katsu_hip_embedding_dev(_embed(**kw), P, P, P, None) == _abi.E_INVALID
    assert L.katsu_hip_embedding_bwd_workspace(_embed(**kw), ctypes.byref(n)) == _abi.E_INVALID
    assert L.katsu_hip_embedding_bwd_dev(_embed(**kw), P, P, P, P, 1 << 30,
                                         None) == _abi.E_INVALID


def test_embedding_pointers():
    fwd, bwd = L.katsu_hip_embedding_dev, L.katsu_hip_embedding_bwd_dev
    n = SZ(0)
    assert fwd(None, P, P, P, None) == _abi.E_INVALID
    assert bwd(None, P, P, P, P, 1 << 30, None) == _abi.E_INVALID
    assert L.katsu_hip_embedding_bwd_workspace(_embed(), None) == _abi.E_INVALID
    for i in range(3):
        some = [None if j == i else P for j in range(3)]
        assert fwd(_embed(), *some, None) == _abi.E_INVALID
        assert bwd(_embed(), *some, P, 1 << 30, None) == _abi.E_INVALID
    # Rows that share memory can be read, not written.
    assert fwd(_embed(out_stride=15), P, P, P, None) == _abi.E_INVALID
    assert fwd(_embed(out_stride=0), P, P, P, None) == _abi.E_INVALID
    assert bwd(_embed(table_stride=15), P, P, P, P, 1 << 30, None) == _abi.E_INVALID
    # Nothing to do.
    assert fwd(_embed(tokens=0), None, None, None, None) == _abi.OK
    assert bwd(_embed(vocab=0), P, P, None, None, 0, None) == _abi.OK
    assert bwd(_embed(tokens=0, accumulate=1), None, None, P, None, 0, None) == _abi.OK
    # A workspace that is too small, or not aligned.
    d = dict(tokens=100000, vocab=50000)
    assert L.katsu_hip_embedding_bwd_workspace(_embed(**d), ctypes.byref(n)) == _abi.OK
    if n.value:
        assert bwd(_embed(**d), P, P, P, P, n.value - 1, None) == _abi.E_INVALID
        for off in (1, 2, 4, 8):
            assert bwd(_embed(**d), P, P, P, ctypes.c_void_p(P.value + off), 1 << 40,
                       None) == _abi.E_INVALID


def _heads(**kw):
    d = dict(dtype=_abi.F32, interleaved=0, tokens=2, heads=2, k_heads=0, head_dim=8, rotary_dim=8,
             length=4, q_stride=(16, 8), q_out_stride=(16, 8), k_stride=(8, 8),
             k_out_stride=(8, 8), eps=1e-6)
    flat = {}
    for name, v in {**d, **kw}.items():
        flat.update({name + "0": v[0], name + "1": v[1]} if isinstance(v, tuple) else {name: v})
    return ctypes.byref(_abi.QkNormRotary(**flat))


GRADS = ctypes.byref(_abi.QkNormRotaryGrads(16, 8, 8, 8))


@pytest.mark.parametrize("kw", [
    dict(dtype=7), dict(heads=65536), dict(k_heads=65536), dict(head_dim=0), dict(head_dim=513),
    dict(rotary_dim=7), dict(rotary_dim=10), dict(tokens=1 << 31), dict(length=0),
    dict(length=1 << 31), dict(q_stride=(-1, 8)), dict(k_stride=(8, -8)),
    dict(q_out_stride=(BIG, 8)), dict(eps=-1.0), dict(eps=NAN), dict(eps=INF)])
def test_heads_refuse(kw):
    n = SZ(0)
    assert L.katsu_hip_qk_norm_rotary_dev(_heads(**kw), P, P, P, P, P, None, P, P,
                                          None) == _abi.E_INVALID
    assert L.katsu_hip_qk_norm_rotary_bwd_workspace(_heads(**kw), ctypes.byref(n)) \
        == _abi.E_INVALID
    assert L.katsu_hip_qk_norm_rotary_bwd_dev(_heads(**kw), GRADS, *[P] * 7, None, *[P] * 5,
                                              1 << 30, None) == _abi.E_INVALID


def test_heads_pointers():
    def fwd(q=P, k=None, w_q=None, w_k=None, table=P, pos=None, out_q=P, out_k=None, **kw):
        return L.katsu_hip_qk_norm_rotary_dev(_heads(**kw), q, k, w_q, w_k, table, pos, out_q,
                                              out_k, None)

    def bwd(dq=P, dk=P, q=P, k=P, w_q=P, w_k=P, table=P, dx_q=P, dx_k=P, dw_q=P, dw_k=P, ws=P,
            size=1 << 30, grads=GRADS, **kw):
        d = _heads(**{**dict(k_heads=1), **kw})
        return L.katsu_hip_qk_norm_rotary_bwd_dev(d, grads, dq, dk, q, k, w_q, w_k, table, None,
                                                  dx_q, dx_k, dw_q, dw_k, ws, size, None)
    other = ctypes.c_void_p(P.value + 64)
    for kw in (dict(q=None), dict(out_q=None), dict(table=None), dict(k_heads=1),
               dict(out_q=other, q_out_stride=(16, 0)), dict(out_q=other, q_out_stride=(0, 8)),
               dict(q_stride=(32, 8))):  # the last: in place with other strides
        assert fwd(**kw) == _abi.E_INVALID, kw
    assert fwd(tokens=0, q=None, out_q=None) == _abi.OK
    assert fwd(heads=0, q=None, out_q=None) == _abi.OK
    for name in ("dq", "dk", "q", "k", "table", "dx_q", "dx_k", "dw_q", "dw_k"):
        assert bwd(**{name: None}) == _abi.E_INVALID, name
    assert bwd(grads=None) == _abi.E_INVALID
    assert bwd(grads=ctypes.byref(_abi.QkNormRotaryGrads(32, 8, 8, 8))) == _abi.E_INVALID
    assert bwd(grads=ctypes.byref(_abi.QkNormRotaryGrads(-16, 8, 8, 8))) == _abi.E_INVALID
    n = SZ(0)
    assert L.katsu_hip_qk_norm_rotary_bwd_workspace(_heads(k_heads=1),
                                                    ctypes.byref(n)) == _abi.OK
    assert n.value > 0
    assert bwd(size=n.value - 1) == _abi.E_INVALID
    for off in (1, 2, 4, 8):
        assert bwd(ws=ctypes.c_void_p(P.value + off)) == _abi.E_INVALID


def _distill(**kw):
    d = dict(dtype=_abi.F32, teacher_dtype=_abi.F32, rows=2, vocab=8, top=2, stride=8,
             out_stride=8, dloss_stride=1, temperature=1.0)
    return ctypes.byref(_abi.Distillation(**{**d, **kw}))


@pytest.mark.parametrize("kw", [
    dict(dtype=2), dict(teacher_dtype=-1), dict(rows=1 << 31), dict(vocab=1 << 31),
    dict(top=1025), dict(stride=-1), dict(out_stride=-8), dict(dloss_stride=-1), dict(stride=BIG),
    dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=NAN), dict(temperature=INF),
    dict(temperature=1e-42)])
def test_distillation_refuses(kw):
    for rc in (L.katsu_hip_distillation_dev(_distill(**kw), *[P] * 5, None),
               L.katsu_hip_distillation_bwd_dev(_distill(**kw), *[P] * 6, None),
               L.katsu_hip_distillation_step_dev(_distill(**kw), *[P] * 6, None)):
        assert rc == _abi.E_INVALID


def test_distillation_pointers():
    fwd, bwd, step = (L.katsu_hip_distillation_dev, L.katsu_hip_distillation_bwd_dev,
                      L.katsu_hip_distillation_step_dev)
    for i in range(4):  # logits, ids, teacher, loss; stats may be missing
        some = [None if j == i else P for j in range(4)]
        assert fwd(_distill(), *some, P, None) == _abi.E_INVALID
    for i in range(6):
        some = [None if j == i else P for j in range(6)]
        assert bwd(_distill(), *some, None) == _abi.E_INVALID
        assert step(_distill(), *some, None) == _abi.E_INVALID
    # Rows that share memory; in place with another stride.
    other = ctypes.c_void_p(P.value + 64)
    for kw, out in ((dict(out_stride=7), other), (dict(stride=16), P)):
        assert bwd(_distill(**kw), P, P, P, P, P, out, None) == _abi.E_INVALID
        assert step(_distill(**kw), P, P, P, P, P, out, None) == _abi.E_INVALID
    for fn in (fwd, bwd, step):
        assert fn(None, *[P] * (5 if fn is fwd else 6), None) == _abi.E_INVALID
    assert fwd(_distill(rows=0), *[None] * 5, None) == _abi.OK
    assert bwd(_distill(rows=0), *[None] * 6, None) == _abi.OK
    assert bwd(_distill(vocab=0), *[None] * 6, None) == _abi.OK
    assert step(_distill(rows=0), *[None] * 6, None) == _abi.OK


def _bad(*calls):
    for i, call in enumerate(calls):
        with pytest.raises(ValueError):
            print(i, flush=True)
            call()


def test_host_tensors():
    """Nothing here runs on host memory."""
    x, i = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int32)
    q = torch.zeros(4, 2, 8)
    _bad(lambda: ops.embedding(i, x), lambda: ops.embedding_backward(x, i, 4),
         lambda: ops.qk_norm_rotary(q, q), lambda: ops.qk_norm_rotary_backward(q, q, q, q),
         lambda: ops.distillation(x, i[:, None], x[:, :1]),
         lambda: ops.distillation_step(x, i[:, None], x[:, :1], x[:, 0]),
         lambda: ops.distillation_backward(x[:, 0], x, i[:, None], x[:, :1], x[:2]))


@pytest.mark.gpu
def test_embedding_operands(dev):
    x, ids = torch.zeros(9, 8, device=dev), torch.zeros(9, dtype=torch.int32, device=dev)
    h = x.half()
    _bad(lambda: ops.embedding(ids.long(), x), lambda: ops.embedding(ids.cpu(), x),
         lambda: ops.embedding(ids[::2], x), lambda: ops.embedding(ids, h),
         lambda: ops.embedding(ids, x.t()), lambda: ops.embedding(ids, x[:, :0]),
         lambda: ops.embedding(ids, x, out=x[:, :4]), lambda: ops.embedding(ids[:4], x, out=x),
         lambda: ops.embedding(ids, x, out=x.bfloat16()),
         lambda: ops.embedding_backward(x, ids[:3], 9),
         lambda: ops.embedding_backward(x, ids, 8, out=x),
         lambda: ops.embedding_backward(x, ids, 9, beta=1.0),
         lambda: ops.embedding_backward(x, ids, 9, out=x.clone(), beta=0.5))
    with pytest.raises(_abi.KatsuError):
        ops.embedding(ids, x, out=x[:1].expand(9, 8))


@pytest.mark.gpu
def test_heads_operands(dev):
    q, k = torch.zeros(5, 4, 8, device=dev), torch.zeros(5, 2, 8, device=dev)
    table, w = torch.zeros(6, 8, device=dev), torch.ones(8, device=dev)
    pos = torch.zeros(5, dtype=torch.int32, device=dev)
    f, b = ops.qk_norm_rotary, ops.qk_norm_rotary_backward
    _bad(lambda: f(q, k[:4]), lambda: f(q, k[..., :4]), lambda: f(q[0], None),
         lambda: f(q, k.bfloat16()), lambda: f(q.transpose(1, 2), None),
         lambda: f(q, k, w_q=w[:4]), lambda: f(q, k, w_q=w.bfloat16()),
         lambda: f(q, None, w_k=w), lambda: f(q, k, table.bfloat16()), lambda: f(q, k, table[0]),
         lambda: f(q, k, table[:, :0]), lambda: f(q, k, None, pos),
         lambda: f(q, k, table, pos.long()), lambda: f(q, k, table, pos[:4]),
         lambda: f(q, k, out_q=k), lambda: f(q, None, out_k=k),
         lambda: b(k, k, q, k), lambda: b(q, None, q, k), lambda: b(q, k, q, None),
         lambda: b(q.bfloat16(), k, q, k))
    for call in (lambda: f(q, k, torch.zeros(6, 10, device=dev)),
                 lambda: f(q, k, table[:, :3].contiguous()), lambda: f(q, k, eps=-1.0),
                 lambda: f(q, k, out_q=q[:, :1].expand(5, 4, 8))):
        with pytest.raises(_abi.KatsuError):
            call()


@pytest.mark.gpu
def test_distillation_operands(dev):
    z, ids = torch.zeros(5, 30, device=dev), torch.zeros(5, 3, dtype=torch.int32, device=dev)
    t, g, s = torch.zeros(5, 3, device=dev), torch.zeros(5, device=dev), torch.zeros(2, 5,
                                                                                     device=dev)
    f, b, step = ops.distillation, ops.distillation_backward, ops.distillation_step
    _bad(lambda: f(z[0], ids, t), lambda: f(z.half(), ids, t), lambda: f(z.t(), ids, t),
         lambda: f(z, ids.long(), t), lambda: f(z, ids[:4], t[:4]), lambda: f(z, ids, t[:, :2]),
         lambda: f(z, ids, t.half()), lambda: f(z, ids.cpu(), t), lambda: f(z, ids, t.cpu()),
         lambda: f(z, ids.t().contiguous().t(), t),
         lambda: b(g[:4], z, ids, t, s), lambda: b(g.double(), z, ids, t, s),
         lambda: b(g, z, ids, t, s[:1]), lambda: b(g, z, ids, t, s.t().contiguous().t()),
         lambda: b(g, z, ids, t, s, out=z[:4]), lambda: b(g, z, ids, t, s, out=z.bfloat16()),
         lambda: step(z, ids, t, g[:, None]), lambda: step(z, ids, t, g.cpu()))
    for call in (lambda: f(z, ids, t, 0.0), lambda: f(z, ids, t, NAN),
                 lambda: step(z, ids, t, g, out=z[:1].expand(5, 30))):
        with pytest.raises(_abi.KatsuError):
            call()


@pytest.mark.gpu
def test_memory(dev):
    """Workspaces and devices that are not the operands'."""
    g, size = torch.Generator().manual_seed(1), 1 << 22
    x, ids = torch.zeros(6000, 8, device=dev), torch.zeros(6000, dtype=torch.int32, device=dev)
    q, w = torch.zeros(50, 2, 64, device=dev), torch.ones(64, device=dev)
    z, i, t = (torch.zeros(2, 50, device=dev), torch.zeros(2, 1, dtype=torch.int32, device=dev),
               torch.zeros(2, 1, device=dev))
    calls = (lambda ws: ops.embedding_backward(x, ids, 6000, workspace=ws),
             lambda ws: ops.qk_norm_rotary_backward(q, None, q, None, w_q=w, workspace=ws))
    for ws in (torch.empty(size, dtype=torch.uint8),
               torch.empty(1, dtype=torch.uint8, device=dev).expand(size),
               torch.empty(2 * size, dtype=torch.uint8, device=dev)[::2]):
        _bad(*(lambda c=c: c(ws) for c in calls))
    ok = torch.empty(size, dtype=torch.uint8, device=dev)
    for c in calls:
        c(ok)
    now = torch._C._cuda_getDevice
    torch._C._cuda_getDevice = lambda: 1  # as if another device were the current one
    try:
        _bad(lambda: ops.embedding(ids, x), lambda: ops.qk_norm_rotary(q, None),
             lambda: ops.distillation(z, i, t), lambda: ops.distillation_step(z, i, t, t[:, 0]),
             *(lambda c=c: c(None) for c in calls))
    finally:
        torch._C._cuda_getDevice = now
