"""The gradient of attention against its float64 formula and against differences: both types, head
widths with and without whole 16-byte rows, shared key heads, rows that see nothing, strides, and
non-finite values in masked places."""
import math

import pytest
import torch

from katsu_amd import _abi, ops
from tests.attention_ref import assert_close, backward, forward, starts

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16]


def _cu(lens, dev):
    return torch.tensor(starts(lens), dtype=torch.int32, device=dev)


def _inputs(tq, tk, heads, kv, d, dt, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(*s, generator=g).to(dt)
            for s in ((tq, heads, d), (tk, kv, d), (tk, kv, d), (tq, heads, d))]


def _grads(dev, q, k, v, do, q_lens, k_lens, **kw):
    q, k, v, do = (t.to(dev) for t in (q, k, v, do))
    cu = dict(cu_q=_cu(q_lens, dev), cu_k=_cu(k_lens, dev), **kw)
    out, lse = ops.attention(q, k, v, **cu)
    got = ops.attention_backward(do, q, k, v, out, lse, **cu)
    torch.cuda.synchronize()
    return got


def _check(dev, q_lens, k_lens, heads, kv, d, dt, causal=True, scale=None):
    q, k, v, do = _inputs(sum(q_lens), sum(k_lens), heads, kv, d, dt)
    print(q_lens, k_lens, heads, kv, d, dt, causal, flush=True)
    got = _grads(dev, q, k, v, do, q_lens, k_lens, causal=causal, scale=scale)
    want, tol = backward(do, q, k, v, q_lens, k_lens, causal, scale or d ** -0.5)
    for name, a, b, t in zip(("dq", "dk", "dv"), got, want, tol):
        assert_close(a, b, t, name)


LENGTHS = [
    ([1], [1]),
    ([3], [0]),
    ([0, 2], [5, 2]),                      # keys that no query sees: zeros
    ([37, 0, 130, 1], [37, 0, 130, 300]),
    ([200, 70, 33], [100, 20, 1]),         # first rows that see nothing
    ([129, 64], [129, 64]),
    ([20], [500]),
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
    _check(dev, [90], [100], 4, 1, 128, dt, causal=False, scale=0.31)


@pytest.mark.parametrize("dt", TYPES)
def test_group_in_one_block(dev, dt):
    """Enough key tiles that a block adds up its group's heads itself."""
    lens = [40] * 300
    _check(dev, lens, lens, 8, 4, 64, dt)


@pytest.mark.parametrize("dt", TYPES)
def test_differences(dev, dt):
    """Along a random direction, against central differences of the float64 forward pass."""
    t, heads, kv, d = 90, 4, 2, 64
    q, k, v, do = _inputs(t, t, heads, kv, d, dt, seed=7)
    got = _grads(dev, q, k, v, do, [t], [t])
    _, tol = backward(do, q, k, v, [t], [t], True, 0.125)
    g = torch.Generator().manual_seed(8)
    for i in range(3):
        u = torch.randn(got[i].shape, generator=g, dtype=torch.float64)
        eps, loss = 1e-4, []
        for sign in (1, -1):
            x = [q.double(), k.double(), v.double()]
            x[i] = x[i] + sign * eps * u
            out = forward(*x, [t], [t], True, 0.125)[0]
            loss.append((out * do.double()).sum().item())
        want = (loss[0] - loss[1]) / (2 * eps)
        have = (got[i].double().cpu() * u).sum().item()
        # The differences' own error: the third derivative's term, eps^2 of a smooth function
        # of the size of the gradient's, and rounding, 2^-52 / eps of the loss.
        bound = (tol[i] * u.abs()).sum().item() + 1e-5 * (got[i].double().cpu() * u).abs().sum()
        assert abs(have - want) <= bound, (i, have, want, bound)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("offset", [0, 1])
def test_strides(dev, dt, offset):
    """Operands and gradients as views of one projection's output and its gradient."""
    t, heads, kv, d = 75, 4, 2, 64
    g = torch.Generator().manual_seed(3)
    n = heads + 2 * kv
    flat = torch.randn(t * n * d + offset, generator=g).to(dt)
    host = flat[offset:].view(t, n, d)
    x = flat.to(dev)[offset:].view(t, n, d)
    dx = torch.empty(t * n * d + offset, dtype=dt, device=dev)[offset:].view(t, n, d)
    do = torch.randn(heads, t, d, generator=g).to(dt).transpose(0, 1)

    def parts(y):
        return y[:, :heads], y[:, heads:heads + kv], y[:, heads + kv:]
    q, k, v = parts(x)
    out, lse = ops.attention(q, k, v)
    dq, dk, dv = parts(dx)
    got = ops.attention_backward(do.to(dev), q, k, v, out, lse, dq=dq, dk=dk, dv=dv)
    assert got[0] is dq and got[1] is dk and got[2] is dv
    want, tol = backward(do, *parts(host), [t], [t], True, 0.125)
    for a, b, c in zip(got, want, tol):
        assert_close(a, b, c, "gradient")


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("d", [64, 40])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_masked_nonfinite(dev, dt, d, bad):
    """Non-finite values of the last token's key and value reach the last query's gradient only;
    those of the first rows' queries, which see no key, reach nothing."""
    t = 100
    q, k, v, do = _inputs(t, t, 2, 1, d, dt)
    k[-1], v[-1], do[-1] = bad, bad, 0
    got = _grads(dev, q, k, v, do, [t], [t])
    cut = [x[:-1] for x in (q, k, v)]
    want, tol = backward(do[:-1], *cut, [t - 1], [t - 1], True, d ** -0.5)
    assert_close(got[0][:-1], want[0], tol[0], "dq")
    q, k, v, do = _inputs(t, 60, 2, 1, d, dt)
    q[:40], do[:40] = bad, bad
    got = _grads(dev, q, k, v, do, [t], [60])
    want, tol = backward(do[40:], q[40:], k, v, [60], [60], True, d ** -0.5)
    assert (got[0][:40] == 0).all()
    assert_close(got[0][40:], want[0], tol[0], "dq")
    assert_close(got[1], want[1], tol[1], "dk")
    assert_close(got[2], want[2], tol[2], "dv")
    # A row's values reach the keys that it sees and no others.
    q, k, v, do = _inputs(t, t, 2, 1, d, dt)
    do[50] = bad
    got = _grads(dev, q, k, v, do, [t], [t])
    keep = [i for i in range(t) if i != 50]
    # dk and dv of the keys behind row 50 take nothing from the rows up to it.
    want, tol = backward(do[51:], q[51:], k, v, [49], [t], True, d ** -0.5)
    assert_close(got[1][51:], want[1][51:], tol[1][51:], "dk")
    assert_close(got[2][51:], want[2][51:], tol[2][51:], "dv")
    assert not got[2][:51].isfinite().any()
    want, tol = backward(torch.where(do.isfinite(), do, 0), q, k, v, [t], [t], True, d ** -0.5)
    assert_close(got[0][keep], want[0][keep], tol[0][keep], "dq")


@pytest.mark.parametrize("dt", TYPES)
def test_masked_nonfinite_runs(dev, dt):
    """The same where the other axis is split into runs."""
    t, d = 600, 128
    q, k, v, do = _inputs(t, t, 2, 1, d, dt)
    k[-1], v[-1], do[-1] = math.nan, math.nan, 0
    got = _grads(dev, q, k, v, do, [t], [t])
    want, tol = backward(do[:-1], q[:-1], k[:-1], v[:-1], [t - 1], [t - 1], True, d ** -0.5)
    assert_close(got[0][:-1], want[0], tol[0], "dq")
    q, k, v, do = _inputs(t, t, 2, 1, d, dt)
    do[290] = math.nan
    got = _grads(dev, q, k, v, do, [t], [t])
    want, tol = backward(do[291:], q[291:], k, v, [t - 291], [t], True, d ** -0.5)
    assert_close(got[1][291:], want[1][291:], tol[1][291:], "dk")
    assert_close(got[2][291:], want[2][291:], tol[2][291:], "dv")
    assert got[2][:291].isnan().all()


@pytest.mark.parametrize("dt", TYPES)
def test_many_sequences(dev, dt):
    """More than 64 sequences, of all lengths from none; and a long one among short ones."""
    lens = [(7 * i) % 5 for i in range(200)]
    _check(dev, lens, lens, 2, 2, 64, dt)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("lens", [[3, 700, 0, 64, 1500], [3, 1500, 0, 64, 130, 1400]])
def test_orders_of_tiles(dev, dt, lens):
    """Tiles enough that they go in pairs (256 to 512 of them), and by work (more): two
    heads against the reference."""
    t, heads, d = sum(lens), 24, 64
    q, k, v, do = _inputs(t, t, heads, heads, d, dt)
    out, lse = ops.attention(*(x.to(dev) for x in (q, k, v)), _cu(lens, dev), _cu(lens, dev))
    got = _grads(dev, q, k, v, do, lens, lens)
    for h in (0, 23):
        one = [x[:, h:h + 1] for x in (q, k, v, do)]
        ro, rl, to, tl = forward(*one[:3], lens, lens, True, d ** -0.5)
        assert_close(out[:, h:h + 1], ro, to, "out")
        assert_close(lse[h:h + 1], rl, tl, "lse")
        want, tol = backward(one[3], *one[:3], lens, lens, True, d ** -0.5)
        for a, b, c in zip(got, want, tol):
            assert_close(a[:, h:h + 1], b, c, "gradient")
    assert all(x.isfinite().all() for x in got) and out.isfinite().all()


@pytest.mark.parametrize("kv", [1, 4])
def test_same_bits_and_workspace(dev, kv):
    q, k, v, do = [x.to(dev) for x in _inputs(500, 500, 4, kv, 128, torch.bfloat16)]
    out, lse = ops.attention(q, k, v)
    need = ops.attention_workspace_bytes(q, k, v, backward=True)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    a = ops.attention_backward(do, q, k, v, out, lse)
    b = ops.attention_backward(do, q, k, v, out, lse, workspace=ws)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    with pytest.raises(_abi.KatsuError):
        ops.attention_backward(do, q, k, v, out, lse, workspace=ws[:-256])


def test_graph(dev):
    """Forward and backward in one captured graph, replayed on new inputs."""
    q, k, v, do = [x.to(dev) for x in _inputs(130, 130, 4, 2, 64, torch.float32)]
    dq, dk, dv = (torch.empty_like(t) for t in (q, k, v))

    def step():
        out, lse = ops.attention(q, k, v)
        ops.attention_backward(do, q, k, v, out, lse, dq=dq, dk=dk, dv=dv)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in (5, 6, 7):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (dq, dk, dv)]
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (dq, dk, dv)))


def test_refusals(dev):
    q, k, v, do = [x.to(dev) for x in _inputs(8, 8, 4, 2, 64, torch.float32)]
    out, lse = ops.attention(q, k, v)
    for args, kw in (
            ((do[:4], q, k, v, out, lse), {}),
            ((do.bfloat16(), q, k, v, out, lse), {}),
            ((do, q, k, v, out, lse[:2]), {}),
            ((do, q, k, v, out, lse.double()), {}),
            ((do, q, k, v, out, lse), dict(dk=torch.empty_like(q))),
            ((do, q, k, v, out[..., ::2], lse), {})):
        with pytest.raises(ValueError):
            ops.attention_backward(*args, **kw)
    with pytest.raises(_abi.KatsuError):
        ops.attention_backward(do, q, k, v, out, lse, scale=0.0)
