"""Attention over packed sequences against its float64 definition: both types, head widths with and
without whole 16-byte rows, shared key heads, lengths of zero and one, rows that see no key, caches
with slots, strides, non-finite values in masked places, and the variants for few and many rows."""
import math

import pytest
import torch

from katsu_amd import _abi, ops
from tests.attention_ref import assert_close, forward, starts

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16]


def _cu(lens, dev):
    return torch.tensor(starts(lens), dtype=torch.int32, device=dev)


def _inputs(tq, tk, heads, kv, d, dt, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(*s, generator=g).to(dt) for s in ((tq, heads, d), (tk, kv, d), (tk, kv, d))]


def _check(dev, q_lens, k_lens, heads, kv, d, dt, causal=True, scale=None):
    q, k, v = _inputs(sum(q_lens), sum(k_lens), heads, kv, d, dt)
    print(q_lens, k_lens, heads, kv, d, dt, causal, flush=True)
    out, lse = ops.attention(q.to(dev), k.to(dev), v.to(dev), _cu(q_lens, dev), _cu(k_lens, dev),
                             causal=causal, scale=scale)
    torch.cuda.synchronize()
    ro, rl, to, tl = forward(q, k, v, q_lens, k_lens, causal, scale or d ** -0.5)
    assert_close(out, ro, to, "out")
    assert_close(lse, rl, tl, "lse")


LENGTHS = [
    ([1], [1]),
    ([1], [0]),                            # nothing to see
    ([1, 1, 1], [5, 700, 64]),             # single tokens, the key axis split and joined
    ([37, 0, 130, 1], [37, 0, 130, 300]),
    ([200, 70, 33], [100, 20, 1]),         # first rows that see nothing
    ([129], [129]),
    ([40], [1500]),
]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("d", [64, 128, 80, 33, 1])
@pytest.mark.parametrize("heads,kv", [(4, 1), (6, 2), (3, 3)])
def test_lengths(dev, dt, d, heads, kv):
    for q_lens, k_lens in LENGTHS:
        _check(dev, q_lens, k_lens, heads, kv, d, dt)


@pytest.mark.parametrize("dt", TYPES)
def test_not_causal_and_scale(dev, dt):
    _check(dev, [65, 300, 0], [129, 64, 7], 4, 2, 64, dt, causal=False)
    _check(dev, [1, 1], [400, 1], 8, 1, 128, dt, causal=False, scale=0.31)


def test_many_sequences(dev):
    """More sequences than one step of the search for a tile's sequence looks at."""
    lens = [(7 * i) % 5 for i in range(200)]
    _check(dev, lens, lens, 2, 2, 64, torch.float32)
    _check(dev, [1] * 130, [(13 * i) % 40 for i in range(130)], 2, 1, 64, torch.bfloat16)


def test_one_sequence_without_starts(dev):
    q, k, v = _inputs(70, 90, 2, 1, 64, torch.float32)
    out, lse = ops.attention(q.to(dev), k.to(dev), v.to(dev))
    ro, rl, to, tl = forward(q, k, v, [70], [90], True, 0.125)
    assert_close(out, ro, to, "out")
    assert_close(lse, rl, tl, "lse")


@pytest.mark.parametrize("dt", TYPES)
def test_cache_slots(dev, dt):
    """k_lens keys of each slot are used; what lies behind them, NaN here, is not."""
    used, slot, q_lens = [3, 0, 64, 41], 64, [1, 1, 1, 5]
    q, k, v = _inputs(8, 4 * slot, 4, 2, 64, dt)
    for s, n in enumerate(used):
        k[s * slot + n:(s + 1) * slot] = math.nan
        v[s * slot + n:(s + 1) * slot] = math.nan
    out, lse = ops.attention(q.to(dev), k.to(dev), v.to(dev), _cu(q_lens, dev),
                             _cu([slot] * 4, dev),
                             torch.tensor(used, dtype=torch.int32, device=dev))
    ro, rl, to, tl = forward(q, k, v, q_lens, used, True, 0.125, slots=[slot] * 4)
    assert_close(out, ro, to, "out")
    assert_close(lse, rl, tl, "lse")


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("offset", [0, 1])
def test_strides(dev, dt, offset):
    """q, k and v as views of one projection's output, heads before tokens in the output, and
    (offset 1) addresses that are not multiples of 16 bytes."""
    t, heads, kv, d = 75, 4, 2, 64
    g = torch.Generator().manual_seed(3)
    flat = torch.randn(t * (heads + 2 * kv) * d + offset, generator=g).to(dt)
    host = flat[offset:].view(t, heads + 2 * kv, d)
    x = flat.to(dev)[offset:].view(t, heads + 2 * kv, d)
    out = torch.full((heads, t, d), 7.0, dtype=dt, device=dev).transpose(0, 1)
    q, k, v = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
    got, lse = ops.attention(q, k, v, out=out)
    assert got is out
    ro, rl, to, tl = forward(host[:, :heads], host[:, heads:heads + kv], host[:, heads + kv:], [t],
                             [t], True, 0.125)
    assert_close(out, ro, to, "out")
    assert_close(lse, rl, tl, "lse")


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("d", [64, 40])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_masked_nonfinite(dev, dt, d, bad):
    """The last key and value are visible to the last query only: every other row is as if they
    were not there.  A non-finite value that a row does see gives what the formula gives."""
    t = 100
    q, k, v = _inputs(t, t, 2, 1, d, dt)
    k[-1], v[-1] = bad, bad
    out, lse = ops.attention(q.to(dev), k.to(dev), v.to(dev))
    ro, rl, to, tl = forward(q[:-1], k[:-1], v[:-1], [t - 1], [t - 1], True, d ** -0.5)
    assert_close(out[:-1], ro, to, "out")
    assert_close(lse[:, :-1], rl, tl, "lse")
    q, k, v = _inputs(t, t, 2, 1, d, dt)
    v[50] = bad
    out, _ = ops.attention(q.to(dev), k.to(dev), v.to(dev))
    ro, _, to, _ = forward(q[:50], k[:50], v[:50], [50], [50], True, d ** -0.5)
    assert_close(out[:50], ro, to, "out")
    want = torch.full_like(out[50:], bad)
    assert torch.equal(out[50:].isnan(), want.isnan()) and (
        math.isnan(bad) or torch.equal(out[50:], want))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("lq,lk,d", [(3, 70, 64), (3, 3000, 128), (2, 40, 33), (300, 700, 128)])
def test_masked_nonfinite_few_rows_and_runs(dev, dt, lq, lk, d):
    """The same where few rows' waves share the keys, and where these are split into runs."""
    for bad in (math.nan, math.inf):
        q, k, v = _inputs(lq, lk, 2, 1, d, dt)
        k[-1], v[-1] = bad, bad
        out, lse = ops.attention(q.to(dev), k.to(dev), v.to(dev))
        ro, rl, to, tl = forward(q[:-1], k[:-1], v[:-1], [lq - 1], [lk - 1], True, d ** -0.5)
        assert_close(out[:-1], ro, to, "out")
        assert_close(lse[:, :-1], rl, tl, "lse")
        q, k, v = _inputs(lq, lk, 2, 1, d, dt)
        v[lk - lq] = bad  # the last key that the first query sees: all see it
        out, lse = ops.attention(q.to(dev), k.to(dev), v.to(dev))
        want = torch.full_like(out, bad)
        assert torch.equal(out.isnan(), want.isnan()) and (
            math.isnan(bad) or torch.equal(out, want))
        _, rl, _, tl = forward(q, k, torch.zeros_like(v), [lq], [lk], True, d ** -0.5)
        assert_close(lse, rl, tl, "lse")


def test_scores_that_are_all_minus_infinity(dev):
    """A row that sees keys, whose scores are all -inf: 0/0, as the formula has it."""
    q = torch.full((2, 1, 64), math.inf)
    k = torch.full((2, 1, 64), -1.0)
    out, lse = ops.attention(q.to(dev), k.to(dev), torch.ones_like(k).to(dev))
    assert out.isnan().all() and (lse == -math.inf).all()


@pytest.mark.parametrize("dt", TYPES)
def test_large_scores(dev, dt):
    """Scores of some hundreds, rising along the keys: the running maximum moves at every tile."""
    t = 300
    q, k, v = _inputs(t, t, 1, 1, 64, dt)
    q, k = q.abs() * 4, (k.abs() * torch.linspace(0, 8, t)[:, None, None]).to(dt)
    out, lse = ops.attention(q.to(dev), k.to(dev), v.to(dev))
    ro, rl, to, tl = forward(q, k, v, [t], [t], True, 0.125)
    assert_close(out, ro, to, "out")
    assert_close(lse, rl, tl, "lse")


def test_same_bits_and_workspace(dev):
    """The same call gives the same bits, on the library's scratch or the caller's."""
    q, k, v = [x.to(dev) for x in _inputs(3, 3000, 8, 2, 128, torch.bfloat16)]
    need = ops.attention_workspace_bytes(q, k, v)
    assert need > 0  # the key axis is split
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    a, b, c = (ops.attention(q, k, v)[0], ops.attention(q, k, v)[0],
               ops.attention(q, k, v, workspace=ws)[0])
    assert torch.equal(a, b) and torch.equal(a, c)
    with pytest.raises(_abi.KatsuError):
        ops.attention(q, k, v, workspace=ws[:-256])


def test_other_stream_and_graph(dev):
    """The call runs on torch's current stream and in a captured graph, replayed on new inputs."""
    q, k, v = [x.to(dev) for x in _inputs(130, 130, 4, 2, 64, torch.float32)]
    want = ops.attention(q, k, v)[0].clone()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = ops.attention(q, k, v)[0]
    s.synchronize()
    assert torch.equal(got, want)
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attention(q, k, v, out=out)
    for seed in (5, 6, 7):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.attention(q, k, v)[0])


def test_starts_outside_the_tensors(dev):
    """Starts that point outside are taken as the tensors' ends: no access outside them."""
    q, k, v = [x.to(dev) for x in _inputs(20, 30, 2, 1, 64, torch.float32)]
    cu = torch.tensor([0, 1 << 30], dtype=torch.int32, device=dev)
    a = ops.attention(q, k, v, cu, cu)[0]
    assert torch.equal(a, ops.attention(q, k, v)[0])


def test_long_cache_offsets(dev):
    """A cache beyond 2^32 bytes: the last sequence lies behind them."""
    slot, n, d = 1 << 18, 66, 128
    k = torch.zeros(n * slot, 1, d, dtype=torch.bfloat16, device=dev)
    v = torch.zeros_like(k)
    assert k.numel() * 2 > 1 << 32
    g = torch.Generator().manual_seed(4)
    used = 300
    tail = torch.randn(2, used, 1, d, generator=g).to(torch.bfloat16)
    at = (n - 1) * slot
    k[at:at + used], v[at:at + used] = tail[0].to(dev), tail[1].to(dev)
    q = torch.randn(n, 2, d, generator=g).to(torch.bfloat16)
    lens = torch.full((n,), used, dtype=torch.int32, device=dev)
    out, _ = ops.attention(q.to(dev), k, v, _cu([1] * n, dev), _cu([slot] * n, dev), lens)
    ro, _, to, _ = forward(q[-1:], tail[0], tail[1], [1], [used], True, d ** -0.5)
    assert_close(out[-1:], ro, to, "out")
    assert (out[:-1] == 0).all()


def test_refusals(dev):
    q, k, v = [x.to(dev) for x in _inputs(8, 8, 4, 2, 64, torch.float32)]
    cu = _cu([8], dev)
    for args, kw in (
            ((q.half(), k.half(), v.half()), {}),
            ((q, k.bfloat16(), v), {}),
            ((q.cpu(), k.cpu(), v.cpu()), {}),
            ((q, k, v[:4]), {}),
            ((q, k[..., :32], v[..., :32]), {}),
            ((q[..., ::2], k[..., ::2], v[..., ::2]), {}),
            ((q[:, :3], k, v), {}),
            ((q[0], k, v), {}),
            ((q, k, v), dict(cu_q=cu)),
            ((q, k, v), dict(cu_q=cu.long(), cu_k=cu.long())),
            ((q, k, v), dict(cu_q=cu, cu_k=_cu([4, 4], dev))),
            ((q, k, v), dict(cu_q=cu, cu_k=cu, k_lens=cu)),
            ((q, k, v), dict(out=torch.empty(8, 4, 32, device=dev)))):
        with pytest.raises(ValueError):
            ops.attention(*args, **kw)
    wide = torch.zeros(4, 1, 129, device=dev)
    for args, kw in (((wide, wide, wide), {}), ((q, k, v), dict(scale=0.0)),
                     ((q, k, v), dict(scale=-1.0)), ((q, k, v), dict(scale=math.inf))):
        with pytest.raises(_abi.KatsuError) as e:
            ops.attention(*args, **kw)
        assert e.value.status == _abi.E_INVALID


def test_empty(dev):
    z = torch.zeros(0, 4, 64, device=dev)
    out, lse = ops.attention(z, z, z)
    assert out.shape == z.shape and lse.shape == (4, 0)
