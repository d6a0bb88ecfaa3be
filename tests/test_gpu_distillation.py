"""The loss against a teacher's top logits and its gradient against their float64 definition: sizes,
types, strides, in place, rows without an entry, repeated ids, masked, huge and non-finite logits."""
import math

import pytest
import torch

from katsu_amd import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16]


def _gamma(n):
    return n * U / (1 - n * U)


def _softmax(x, mask):
    """(probabilities, x - max, log of the total) over the mask's places; zeros where it has none."""
    some = mask.any(1, keepdim=True)
    x = x.masked_fill(~mask, -math.inf)
    top = torch.where(some, x.amax(1, keepdim=True), 0.0)
    d = (x - top).masked_fill(~mask, -math.inf)
    total = d.exp().sum(1, keepdim=True)
    p = torch.where(some, d.exp() / torch.where(some, total, 1.0), 0.0)
    return p, torch.where(mask, d, 0.0), torch.where(some, total.log(), 0.0)


def _ref(z, ids, t, tau, dloss):
    """(loss, gradient, their bounds) in float64; finite logits but for -inf.

    A difference from the largest, over tau, has an error of 4 u of itself, its exponential that and
    2^-22 more.  A total adds gamma(n) of n terms, and for each time that its reference moves the
    error of one more exponential (at most 64 a thread); a logarithm and a sum of few terms round
    once each.  A probability's error is its exponential's and its total's."""
    rows, v = z.shape
    if ids.shape[1] == 0:  # no entries: as one that is no column
        ids, t = torch.full((rows, 1), -1), torch.zeros(rows, 1)
    real = (ids >= 0) & (ids < v)
    td = t.double().masked_fill(~real, -math.inf)
    some = (real & (td > -math.inf)).any(1)
    mask = real & some[:, None] & (td > -math.inf)
    p, dt, lt = _softmax(td / tau, mask)
    all_p, dz, lz = _softmax(z.double() / tau, z.double() > -math.inf)
    at = ids.long().clamp(0, max(v - 1, 0))
    zk = torch.where(mask, dz.gather(1, at), 0.0)
    gone = mask & (z.double().gather(1, at) == -math.inf) & (p > 0)
    terms = torch.where(p > 0, (dt - zk) - lt + lz, 0.0)
    loss = (p * terms).sum(1) * tau ** 2
    loss = torch.where(gone.any(1), math.inf, loss)

    far = dz.abs().amax(1, keepdim=True)
    rel_l = _gamma(v) + 4 * U * far + 66 * 2.0 ** -22
    rel_t = _gamma(ids.shape[1]) + 2.0 ** -21 + 4 * U * dt.abs().amax(1, keepdim=True)
    rel_p = rel_t + 4 * U * dt.abs() + 2.0 ** -21
    each = 6 * U * (dt.abs() + zk.abs() + lt.abs() + lz.abs()) + rel_l + rel_t
    ltol = (p * (each + (rel_p + _gamma(ids.shape[1])) * terms.abs())).sum(1) * tau ** 2
    ltol = ltol + 6 * U * loss.abs().nan_to_num(posinf=0.0) + 1e-30

    want = torch.zeros_like(dz).scatter_add_(1, at, p)
    wtol = torch.zeros_like(dz).scatter_add_(1, at, p * (rel_p + _gamma(ids.shape[1])))
    g = (tau * dloss.double())[:, None]
    grad = torch.where(some[:, None], (all_p - want) * g, 0.0)
    gtol = (all_p * (4 * U * dz.abs() + 2.0 ** -21 + rel_l) + wtol + 2.0 ** -120) * g.abs()
    gtol = torch.where(some[:, None], gtol + (torch.finfo(z.dtype).eps / 2 + 2 * U)
                       * (grad.abs() + gtol), 0.0)
    return torch.where(some, loss, 0.0), grad, torch.where(some, ltol, 0.0), gtol


def _close(got, want, tol):
    got = got.double().cpu()
    same = got == want
    err = (got - want).abs()
    assert (same | (err <= tol)).all(), (err - tol)[~same].max()


def _inputs(rows, vocab, top, dt, seed=1, std=2.5, pad=True):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(rows, vocab, generator=g) * std).to(dt)
    ids = torch.randint(0, vocab, (rows, top), generator=g, dtype=torch.int32)
    t = (torch.randn(rows, top, generator=g) * 2).to(dt)
    if pad and rows > 2 and top > 0:
        ids[1] = -1                               # a row that says nothing
        t[1] = float("nan")
        ids[2, top // 2:] = vocab                 # one with fewer entries (or none)
        t[2, top // 2:] = float("inf")
    dloss = torch.randn(rows, generator=g)
    return z, ids, t, dloss


def _all(dev, z, ids, t, dloss, tau, out=None):
    """The three entry points' results: loss, stats, gradient; step's loss, step's gradient."""
    z, ids, t, dloss = (v.to(dev) for v in (z, ids, t, dloss))
    loss, stats = ops.distillation(z, ids, t, tau)
    grad = ops.distillation_backward(dloss, z, ids, t, stats, tau)
    return (loss, stats, grad) + ops.distillation_step(z, ids, t, dloss, tau)


def _test(dev, z, ids, t, dloss, tau):
    loss, stats, grad, loss2, grad2 = _all(dev, z, ids, t, dloss, tau)
    want, dz, ltol, gtol = _ref(z, ids, t, tau, dloss)
    for got in (loss, loss2):
        _close(got, want, ltol)
    for got in (grad, grad2):
        assert got.dtype is z.dtype
        _close(got, dz, gtol)
    return stats


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("tau", [1.0, 0.5, 3.0])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 5, 2), (3, 8, 8), (5, 1001, 8),
                                            (300, 129, 17), (37, 4099, 64), (2, 70001, 100),
                                            (600, 1000, 1), (4, 3000, 1024), (9, 64, 0),
                                            (260, 9001, 300), (1, 131071, 3), (3, 131073, 20),
                                            (1100, 20, 3)])
def test_sizes(dev, dt, tau, rows, vocab, top):
    print(dt, tau, rows, vocab, top, flush=True)
    z, ids, t, dloss = _inputs(rows, vocab, top, dt)
    stats = _test(dev, z, ids, t, dloss, tau).double().cpu()
    # What stats hold, as documented.
    real = ((ids >= 0) & (ids < vocab)).any(1)
    m = z.double().amax(1)
    inv = 1 / ((z.double() - m[:, None]) / tau).exp().sum(1)
    assert torch.equal(stats[0], torch.where(real, m, 0.0))
    far = (z.double() - m[:, None]).abs().amax(1) / tau
    rel = _gamma(vocab) + 4 * U * far + 67 * 2.0 ** -22
    assert ((stats[1] - torch.where(real, inv, 0.0)).abs() <= rel * inv).all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("other", TYPES)
def test_teacher_type(dev, dt, other):
    z, ids, t, dloss = _inputs(20, 333, 12, dt)
    _test(dev, z, ids, t.to(other), dloss, 2.0)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows", [4, 400])
def test_strides_in_place_broadcast(dev, dt, rows):
    """Logits that are a part of wider rows, at an odd place; the gradient in the logits' place and
    what lies beside it untouched; one dloss for all rows; logits that all rows share."""
    vocab = 1037
    z, ids, t, _ = _inputs(rows, vocab, 9, dt)
    one = torch.tensor([0.75])
    want, dz, ltol, gtol = _ref(z, ids, t, 1.5, one.expand(rows))
    buf = torch.full((rows, vocab + 22), 5.0, dtype=dt)
    buf[:, 3:3 + vocab] = z
    a, b = buf.to(dev), buf.to(dev)
    i, s, g = ids.to(dev), t.to(dev), one.to(dev).expand(rows)
    loss, stats = ops.distillation(a[:, 3:3 + vocab], i, s, 1.5)
    _close(loss, want, ltol)
    out = ops.distillation_backward(g, a[:, 3:3 + vocab], i, s, stats, 1.5, out=a[:, 3:3 + vocab])
    loss, out2 = ops.distillation_step(b[:, 3:3 + vocab], i, s, g, 1.5, out=b[:, 3:3 + vocab])
    _close(loss, want, ltol)
    for o, full in ((out, a), (out2, b)):
        _close(o, dz, gtol)
        _close(full[:, 3:3 + vocab], dz, gtol)
        assert (full[:, :3] == 5).all() and (full[:, 3 + vocab:] == 5).all()
    shared = z[:1].expand(rows, vocab)
    want, dz, ltol, gtol = _ref(shared, ids, t, 1.0, one.expand(rows))
    loss, out = ops.distillation_step(z[:1].to(dev).expand(rows, vocab), i, s, g)
    _close(loss, want, ltol)
    _close(out, dz, gtol)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows", [3, 300])
def test_repeated_ids(dev, dt, rows):
    """The same column twice, all entries at one column, and each of them once."""
    z, ids, t, dloss = _inputs(rows, 500, 40, dt, pad=False)
    ids[0] = 7
    ids[1] = torch.arange(40) % 3 + 250
    ids[2] = torch.arange(40)
    _test(dev, z, ids, t, dloss, 1.0)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows", [6, 280])
def test_masked_logits(dev, dt, rows):
    """Columns at -inf, columns at the type's lowest value, rows of the lowest value alone, a row
    with one column left; teacher entries at -inf, at the lowest value, all of them at -inf."""
    low = torch.finfo(dt).min
    z, ids, t, dloss = _inputs(rows, 900, 10, dt, pad=False)
    ids[:] = torch.arange(10) * 7
    z[0, 100:] = -math.inf
    z[1, 100:] = low
    z[2] = low
    z[3, :63] = z[3, 64:] = -math.inf
    z[3, 63] = 4.0
    t[3, :9], t[3, 9] = -math.inf, 1.0          # whose column is 63
    t[4, 3:] = -math.inf
    t[5] = -math.inf
    t[0, 4] = low
    for tau in (1.0, 0.25, 4.0):
        _test(dev, z, ids, t, dloss, tau)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows", [4, 270])
def test_extremes(dev, dt, rows):
    """A teacher's column at -inf: an infinite loss, and a gradient all the same.  Logits of 1e4 and
    more, where a logarithm of the total taken by itself would lose the loss.  NaN and +inf in a row
    make it NaN and no other, and none where the teacher says nothing."""
    z, ids, t, dloss = _inputs(rows, 700, 5, dt, pad=False)
    ids[:] = torch.arange(5) * 31
    z[0, 31] = -math.inf
    z[1] = z[1] * 3e4
    z[2] += 1e4
    _test(dev, z, ids, t, dloss, 1.0)
    clean = [v.clone() for v in _all(dev, z, ids, t, dloss, 1.0)]
    z[1, 5], z[2, 699] = float("nan"), math.inf
    ids[3] = -1
    z[3] = float("nan")
    dloss[3] = float("nan")
    loss, _, grad, loss2, grad2 = _all(dev, z, ids, t, dloss, 1.0)
    for a, b, base, gbase in ((loss, grad, clean[0], clean[2]), (loss2, grad2, clean[3], clean[4])):
        assert a[1:3].isnan().all() and a[3] == 0 and a[0] == math.inf
        assert b[1:3].isnan().all() and (b[3] == 0).all()
        assert torch.equal(b[0], gbase[0]) and torch.equal(b[4:], gbase[4:])
        assert torch.equal(a[4:], base[4:])


@pytest.mark.parametrize("rows", [4, 400])
def test_row_of_minus_infinity(dev, rows):
    """Logits of nothing but -inf, as the formula has it: NaN where a teacher speaks, else zeros."""
    z, ids, t, dloss = _inputs(rows, 300, 4, torch.float32, pad=False)
    clean = _all(dev, z, ids, t, dloss, 1.0)
    z[1:3], ids[2] = -math.inf, -1
    loss, _, grad, loss2, grad2 = _all(dev, z, ids, t, dloss, 1.0)
    for a, b, was, gwas in ((loss, grad, clean[0], clean[2]), (loss2, grad2, clean[3], clean[4])):
        assert a[1].isnan() and b[1].isnan().all() and a[2] == 0 and not b[2].any()
        assert torch.equal(a[3:], was[3:]) and torch.equal(b[3:], gwas[3:])


@pytest.mark.parametrize("dt", TYPES)
def test_many_long_rows(dev, dt):
    """Rows that no block's registers hold, more than 1024 of them: one row of logits, read by all."""
    rows, vocab = 1030, 140001
    g = torch.Generator().manual_seed(7)
    z = (torch.randn(1, vocab, generator=g) * 2.5).to(dt)
    ids = torch.randint(0, vocab, (4, 6), generator=g, dtype=torch.int32)
    t = torch.randn(4, 6, generator=g).to(dt)
    want, dz, ltol, gtol = _ref(z.expand(4, vocab), ids, t, 2.0, torch.ones(4))
    loss, grad = ops.distillation_step(
        z.to(dev).expand(rows, vocab), ids.repeat(258, 1)[:rows].to(dev),
        t.repeat(258, 1)[:rows].to(dev), torch.ones(1, device=dev).expand(rows), 2.0)
    _close(loss[:4], want, ltol)
    _close(grad[:4], dz, gtol)
    for i in range(4, rows, 4):
        n = min(4, rows - i)
        assert torch.equal(loss[i:i + n], loss[:n]) and torch.equal(grad[i:i + n], grad[:n]), i


def test_cross_entropy(dev):
    """One entry at temperature 1 is the cross entropy with labels, -1 for rows that do not count."""
    g = torch.Generator().manual_seed(3)
    z, labels = torch.randn(50, 333, generator=g), torch.randint(0, 333, (50,), generator=g)
    labels[::7] = -1
    loss, _ = ops.distillation(z.to(dev), labels.int()[:, None].to(dev),
                               torch.zeros(50, 1, device=dev))
    want = torch.nn.functional.cross_entropy(z.double(), labels, ignore_index=-1,
                                             reduction="none")
    # Logits up to 4 and totals of 333 terms: within 400 u of a value below 10.
    assert ((loss.double().cpu() - want).abs() <= 4000 * U).all()


def test_gradient_by_differences(dev):
    """Along a direction, the loss's differences in float64 against the gradient."""
    z, ids, t, dloss = _inputs(6, 200, 12, torch.float32, 4)
    g = torch.Generator().manual_seed(5)
    e, h = torch.randn(z.shape, generator=g).double(), 1e-4
    f = [(_ref(z.double() + s * h * e, ids, t, 2.0, dloss)[0] * dloss.double()).sum()
         for s in (1, -1)]
    _, grad = ops.distillation_step(*(v.to(dev) for v in (z, ids, t, dloss)), 2.0)
    grad = grad.double().cpu()
    # h^2 of third derivatives of order one, float32 results of order one.
    assert abs((grad * e).sum() - (f[0] - f[1]) / (2 * h)) <= 1e-5 * (grad * e).abs().sum()


@pytest.mark.parametrize("rows,vocab", [(3, 40000), (500, 2000)])
def test_same_bits(dev, rows, vocab):
    """Calls, replays of a graph with other logits between, another stream."""
    z, ids, t, dloss = (v.to(dev) for v in _inputs(rows, vocab, 33, torch.bfloat16))
    other = torch.randn_like(z)
    want = [_all(dev, v, ids, t, dloss, 2.0) for v in (z, other)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        own = ops.distillation(z, ids, t, 2.0)
        step = ops.distillation_step(z, ids, t, dloss, 2.0)
        side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(own + step, want[0][:2] + want[0][3:]))
    x = z.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _all(dev, x, ids, t, dloss, 2.0)
    for i in (0, 1, 0, 1):
        x.copy_((z, other)[i])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[i]))
        assert torch.equal(ops.distillation(other, ids, t, 2.0)[0], want[1][0])


def test_large_offsets(dev):
    """Rows beyond 2^31 elements."""
    rows, vocab = 33000, 70000
    z = torch.zeros(rows, vocab, dtype=torch.bfloat16, device=dev)
    ids = torch.full((rows, 1), -1, dtype=torch.int32, device=dev)
    t, dloss = torch.zeros(rows, 1, device=dev), torch.ones(rows, device=dev)
    ids[-1], ids[31000] = 69999, 5
    z[-1, 69999] = 3.0
    loss, stats = ops.distillation(z, ids, t)
    grad = ops.distillation_backward(dloss, z, ids, t, stats)
    loss2, z = ops.distillation_step(z, ids, t, dloss, out=z)
    for a, b in ((loss, grad), (loss2, z)):
        assert abs(a[-1].item() - (math.log(69999 + math.exp(3)) - 3)) <= 1e-5
        assert abs(a[31000].item() - math.log(70000)) <= 1e-5
        assert not a[:31000].any() and not a[31001:-1].any()
        assert not b[:31000].any() and not b[31001:-1].any()
        assert abs(b[-1, 69999].item() + 1) < 0.01 and b[-1, 0] > 0
        assert abs(b[31000, 5].item() + 1) < 0.01 and b[31000, 6] > 0
