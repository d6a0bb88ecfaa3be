"""Attention over some of a batch's sequences, by a slice of its starts: tokens before the first and
after the last belong to none.  What lies around lse and the outputs stays as it was."""
import ctypes

import pytest
import torch

from katsu_amd import _abi, ops
from tests.attention_ref import assert_close, backward, forward, starts

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16]
GUARD = 4096


def _guarded(shape, dt, dev):
    """A tensor in the middle of a buffer of sevens, and the buffer."""
    n = torch.Size(shape).numel()
    flat = torch.full((n + 2 * GUARD,), 7.0, dtype=dt, device=dev)
    return flat[GUARD:GUARD + n].view(shape), flat


def _untouched(flats):
    return all((f[:GUARD] == 7).all() and (f[-GUARD:] == 7).all() for f in flats)


CASES = [  # query lengths, key lengths, the sequences taken
    ([128, 128], [128, 128], (1, 2)),
    ([3, 1, 1, 2], [900, 20, 700, 5], (1, 3)),          # few rows, the key axis split
    ([700, 3, 1200, 40, 9], [700, 3, 1200, 40, 9], (1, 4)),
    ([5] * 150, [7] * 150, (40, 120)),                  # more than 64 sequences
    ([300, 10], [10, 400], (1, 2)),
    ([50, 60], [50, 60], (1, 1)),                       # none
]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("d", [64, 40])
@pytest.mark.parametrize("heads,kv", [(8, 2), (3, 3)])
@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("causal", [True, False])
def test_slice_of_starts(dev, dt, d, heads, kv, case, causal):
    q_lens, k_lens, (first, last) = CASES[case]
    tq, tk = sum(q_lens), sum(k_lens)
    g = torch.Generator().manual_seed(6)
    q, k, v, do = (torch.randn(t, h, d, generator=g).to(dt)
                   for t, h in ((tq, heads), (tk, kv), (tk, kv), (tq, heads)))
    print(dt, d, heads, kv, CASES[case], causal, flush=True)
    qd, kd, vd, dod = (x.to(dev) for x in (q, k, v, do))
    cq, ck = (torch.tensor(starts(x), dtype=torch.int32)[first:last + 1].to(dev)
              for x in (q_lens, k_lens))
    out, flat_out = _guarded((tq, heads, d), dt, dev)
    lse, flat_lse = _guarded((heads, tq), torch.float32, dev)
    grads = [_guarded(x.shape, dt, dev) for x in (q, k, v)]
    desc = _abi.Attention(_abi.F32 if dt is torch.float32 else _abi.BF16, causal, heads, kv, d,
                          last - first, tq, tk, qd.stride()[:2], kd.stride()[:2],
                          vd.stride()[:2], out.stride()[:2], d ** -0.5)
    assert _abi.lib().katsu_hip_attention_fwd_dev(
        ctypes.byref(desc), qd.data_ptr(), kd.data_ptr(), vd.data_ptr(), cq.data_ptr(),
        ck.data_ptr(), None, out.data_ptr(), lse.data_ptr(), None, 0,
        torch.cuda.current_stream().cuda_stream) == 0
    (dq, _), (dk, _), (dv, _) = grads
    ops.attention_backward(dod, qd, kd, vd, out, lse, cu_q=cq, cu_k=ck, causal=causal, dq=dq,
                           dk=dk, dv=dv)
    torch.cuda.synchronize()
    assert _untouched([flat_out, flat_lse] + [f for _, f in grads])
    qs, ks = (slice(starts(x)[first], starts(x)[last]) for x in (q_lens, k_lens))
    lens = q_lens[first:last], k_lens[first:last]
    args = (q[qs], k[ks], v[ks], *lens, causal, d ** -0.5)
    ro, rl, to, tl = forward(*args)
    assert_close(out[qs], ro, to, "out")
    assert_close(lse[:, qs], rl, tl, "lse")
    want, tol = backward(do[qs], *args)
    for name, a, b, c in zip(("dq", "dk", "dv"), (dq[qs], dk[ks], dv[ks]), want, tol):
        assert_close(a, b, c, name)


@pytest.mark.parametrize("dt", TYPES)
def test_most_sequences(dev, dt):
    """So many sequences that a launch's first axis does not cover their tiles; most are empty."""
    heads, d, n = 4, 16, (1 << 22) + 70
    lens = torch.zeros(n, dtype=torch.int32)
    lens[::1 << 17] = 3
    some = [3] * int((lens > 0).sum())
    cu = torch.cat([torch.zeros(1, dtype=torch.int32), lens.cumsum(0, dtype=torch.int32)]).to(dev)
    t = sum(some)
    g = torch.Generator().manual_seed(7)
    q, k, v, do = (torch.randn(t, heads, d, generator=g).to(dt) for _ in range(4))
    card = [x.to(dev) for x in (q, k, v)]
    nan = [torch.full_like(x, float("nan")) for x in card]
    out, lse = ops.attention(*card, cu, cu, out=nan[0].clone())
    got = ops.attention_backward(do.to(dev), *card, out, lse, cu, cu, dq=nan[0], dk=nan[1],
                                 dv=nan[2])
    ro, rl, to, tl = forward(q, k, v, some, some, True, d ** -0.5)
    assert_close(out, ro, to, "out")
    assert_close(lse, rl, tl, "lse")
    want, tol = backward(do, q, k, v, some, some, True, d ** -0.5)
    for name, a, b, c in zip(("dq", "dk", "dv"), got, want, tol):
        assert_close(a, b, c, name)
