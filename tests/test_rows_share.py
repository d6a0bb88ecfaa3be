"""Outputs of the embedding, its gradient and distillation that share memory with an input whose rows other
waves still read: refused, and no others."""
import ctypes
import random

import pytest
import torch

from katsu_amd import _abi, ops
from tests.test_lm_ends import L, P, _distill, _embed

ROOM = 64
BUF = (ctypes.c_float * ROOM)()


def _at(i):
    return ctypes.c_void_p(ctypes.addressof(BUF) + 4 * i)


def _places(at, rows, cols, stride):
    return {at + r * stride + c for r in range(rows) for c in range(cols)}


def _cases(n, seed, same_rows):
    """(place, rows, stride) of an input and an output, their columns, whether they share a place."""
    g = random.Random(seed)
    for _ in range(n):
        cols, rows = g.randint(1, 6), g.randint(1, 6)
        out_rows = rows if same_rows else g.randint(1, 6)
        stride = g.choice([g.randint(0, 12), g.randint(cols, 16)])
        out_stride = stride if stride >= cols and g.random() < 0.4 else g.randint(cols, 16)
        a, b = g.randint(0, ROOM // 2), g.randint(0, ROOM // 2)
        x, y = _places(a, rows, cols, stride), _places(b, out_rows, cols, out_stride)
        if max(x | y) < ROOM:
            yield (a, rows, stride), (b, out_rows, out_stride), cols, bool(x & y)


def test_cases():
    """Both kinds, and among those that share nothing some whose rows lie between each other's."""
    for same in (False, True):
        cases = list(_cases(4000, 1, same))
        free = [c for c in cases if not c[3]]
        between = [c for c in free if c[0][0] < c[1][0] < c[0][0] + (c[0][1] - 1) * c[0][2]]
        assert len(cases) - len(free) > 500 and len(free) > 300 and len(between) > 30
        assert any(c[0][2] != c[1][2] for c in between)


def test_embedding_refuses():
    """Without a GPU: only calls that are refused."""
    for (a, rows, s), (b, n, t), cols, share in _cases(4000, 1, False):
        if share:
            d = _embed(vocab=rows, tokens=n, cols=cols, table_stride=s, out_stride=t)
            assert L.katsu_hip_embedding_dev(d, P, _at(a), _at(b), None) == _abi.E_INVALID
            for beta in (0, 1):
                d = _embed(tokens=rows, vocab=n, cols=cols, out_stride=s, table_stride=t,
                           accumulate=beta)
                assert L.katsu_hip_embedding_bwd_dev(d, _at(a), P, _at(b), P, 1 << 30,
                                                     None) == _abi.E_INVALID


@pytest.mark.gpu
def test_embedding_operands(dev):
    """As many tokens as rows, in the table's own place, or half a row beside it."""
    ids = torch.zeros(9, dtype=torch.int32, device=dev)
    for dt in (torch.float32, torch.bfloat16):
        x = torch.zeros(10, 8, dtype=dt, device=dev)
        flat = x.flatten()
        for a, b in ((x[:9], x[:9]), (x[:9], x[1:]), (flat[:72].view(9, 8), flat[4:76].view(9, 8)),
                     (x[:9, :5], x[:9, 4:8].as_strided((9, 5), (8, 1), 4))):
            with pytest.raises(_abi.KatsuError):
                ops.embedding(ids, a, out=b)
            for beta in (0.0, 1.0):
                with pytest.raises(_abi.KatsuError):
                    ops.embedding_backward(a, ids, 9, out=b, beta=beta)


@pytest.mark.gpu
def test_embedding_taken(dev):
    """Rows between each other's, with the same stride and with others: the results of rows apart."""
    base = torch.arange(1.0, ROOM + 1, device=dev)
    done = 0
    for (a, rows, s), (b, n, t), cols, share in _cases(1500, 2, False):
        if share:
            continue
        done += 1
        for call in (lambda i, o: ops.embedding(torch.arange(n, device=dev).int() % (rows + 1), i,
                                                2.0, out=o),
                     lambda i, o: ops.embedding_backward(i, torch.arange(rows, device=dev).int()
                                                         % (n + 1), n, 2.0, out=o)):
            buf = base.clone()
            i, o = buf.as_strided((rows, cols), (s, 1), a), buf.as_strided((n, cols), (t, 1), b)
            want = base.clone()
            view = want.as_strided((n, cols), (t, 1), b)
            apart = i.clone(memory_format=torch.contiguous_format)
            view.copy_(call(apart, torch.empty(n, cols, device=dev)))
            call(i, o)
            assert torch.equal(buf, want), ((a, rows, s), (b, n, t), cols)
    assert done > 100


def test_distillation_refuses():
    """Without a GPU: only calls that are refused; the logits' own place is another test's."""
    for (a, rows, s), (b, _, t), cols, share in _cases(4000, 1, True):
        if share and a != b:
            d = _distill(rows=rows, vocab=cols, top=1, stride=s, out_stride=t)
            assert L.katsu_hip_distillation_bwd_dev(d, P, _at(a), P, P, P, _at(b),
                                                    None) == _abi.E_INVALID
            assert L.katsu_hip_distillation_step_dev(d, _at(a), P, P, P, P, _at(b),
                                                     None) == _abi.E_INVALID


@pytest.mark.gpu
def test_distillation_taken(dev):
    """Rows between each other's, and the logits' own place: the results of rows apart."""
    g = torch.Generator().manual_seed(3)
    base = torch.randn(ROOM, generator=g).to(dev)
    done = 0
    for (a, rows, s), (b, _, t), cols, share in _cases(1500, 2, True):
        if share and ((a, s) != (b, t) or s < cols):
            continue
        done += 1
        ids = (torch.arange(rows, device=dev).int() % cols)[:, None].contiguous()
        t_, dloss = torch.zeros(rows, 1, device=dev), torch.ones(rows, device=dev)
        for call in (lambda z, o: ops.distillation_step(z, ids, t_, dloss, out=o)[1],
                     lambda z, o: ops.distillation_backward(
                         dloss, z, ids, t_, ops.distillation(z, ids, t_)[1], out=o)):
            buf, want = base.clone(), base.clone()
            i, o = buf.as_strided((rows, cols), (s, 1), a), buf.as_strided((rows, cols), (t, 1), b)
            apart = call(i.clone(memory_format=torch.contiguous_format),
                         torch.empty(rows, cols, device=dev))
            want.as_strided((rows, cols), (t, 1), b).copy_(apart)
            call(i, o)
            # The order of at most six terms' sum may be another one.
            assert ((buf - want).abs() <= 32 * 2.0 ** -24).all(), ((a, rows, s), (b, t), cols)
            o.copy_(want.as_strided((rows, cols), (t, 1), b))
            assert torch.equal(buf, want)
    assert done > 100
