"""Distillation's totals to their last logit: rows of one value, whose totals are whole numbers, and rows with
one logit far above the others at every place where a row, a thread's run or a 16-byte access begins or
ends, for rows that begin at every place within 16 bytes."""
import math

import pytest
import torch

from katsu_amd import ops
from tests.test_gpu_distillation import TYPES

U = 2.0 ** -24
PEAK = 30.0


def _edges(dt):
    """Columns around the numbers of 16-byte pieces at which the launches change, and odd ones."""
    e = 16 // (torch.finfo(dt).bits // 8)
    some = {1, 2, e, e + 1, 37, 1001}
    for pieces in (128, 512, 1024, 2048, 4096, 8192, 16384):
        some |= {pieces * e + d for d in (-e, 1 - e, -1, 0, 1)}
    return sorted(some)


def _rows(rows, vocab, dt, dev, at):
    """[rows, vocab] with a place of its own within 16 bytes for each row, and for the first `at` values
    after a boundary; room behind the last row."""
    stride = (vocab // 8 + 1) * 8 + 1
    buf = torch.full((rows * stride + 64,), math.nan, dtype=dt, device=dev)
    return buf[at:at + rows * stride].view(rows, stride)[:, :vocab]


def _calls(z, ids, t, dloss, tau=1.0):
    loss, stats = ops.distillation(z, ids, t, tau)
    grad = ops.distillation_backward(dloss, z, ids, t, stats, tau)
    loss2, grad2 = ops.distillation_step(z, ids, t, dloss, tau)
    return loss, stats, grad, loss2, grad2


def _near(got, want, tol):
    assert ((got.double() - want).abs() <= tol).all(), ((got.double() - want).abs().max(), tol)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows", [9, 270, 1100])
def test_rows_of_one_value(dev, dt, rows):
    """L = V exactly: exp2(0) is 1, and float32 holds whole numbers below 2^24.  So 1/L is off by half a
    step; loss = tau^2 log V by the logarithm's two steps, a product's half each for tau twice, which
    together are below what one logit is; P = 1/V by a product's half step more than 1/L, then the
    products with dloss tau and the type's rounding."""
    top = 2
    for vocab in _edges(dt):
        if rows * vocab > 1 << 26:
            continue
        tau = 2.0 if vocab % 2 else 1.0
        print(dt, rows, vocab, tau, flush=True)
        z = _rows(rows, vocab, dt, dev, vocab % 5).fill_(-3.25)
        ids = torch.zeros(rows, top, dtype=torch.int32, device=dev)
        ids[:, 0] = torch.arange(rows, device=dev).int() % vocab
        ids[:, 1] = -1
        t = torch.ones(rows, top, device=dev)
        dloss = torch.full((rows,), 0.5, device=dev)
        loss, stats, grad, loss2, grad2 = _calls(z, ids, t, dloss, tau)
        want = math.log(vocab)
        ltol = 6 * U * want * tau * tau
        assert vocab == 1 or ltol < (want - math.log(vocab - 1) if vocab > 1 else 1) * tau * tau
        assert (stats[0] == -3.25).all()
        _near(stats[1], 1 / vocab, 2 * U / vocab)
        assert vocab == 1 or 2 * U / vocab < 1 / (vocab - 1) - 1 / vocab
        for a in (loss, loss2):
            _near(a, want * tau * tau, ltol)
        half = torch.finfo(dt).eps / 2
        label = torch.arange(vocab, device=dev) == ids[:, :1]
        g = 0.5 * tau
        for b in (grad, grad2):
            assert b.dtype is dt
            p = 1.0 / vocab
            _near(b.masked_fill(label, p * g), p * g, (half + 6 * U) * p * g)
            one = b.gather(1, ids[:, :1].long())
            _near(one, (p - 1) * g, (half + 4 * U) * (1 - p) * g + 4 * U * g)


def _places(vocab, dt):
    """Around multiples of the runs of pieces: a block's of 128 to 1024 threads, one or four a thread,
    and the gradient's runs of columns, each also a row's start within 16 bytes before it."""
    e = 16 // (torch.finfo(dt).bits // 8)
    some = set(range(min(2 * e + 1, vocab))) | set(range(max(vocab - 2 * e - 1, 0), vocab))
    for step in (64 * e, 128 * e, 256 * e, 512 * e, 1024 * e, 4096 * e, 2048):
        for n in (1, 2, vocab // step):
            some |= {n * step + d for d in (-e - 1, -e, -1, 0, 1, e)}
    return sorted(j for j in some if 0 <= j < vocab)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("vocab", [2, 9, 129, 515, 1023, 2049, 4097, 8197, 16391, 32771, 65539, 131079])
@pytest.mark.parametrize("times", [1, 7])
def test_largest_logit_anywhere(dev, dt, vocab, times):
    """z = 30 at column j, else 0; the teacher's column is another.  M = 30, L = 1 + (V - 1) e^-30, loss
    30 + log L, P[j] = 1 / L; without column j they were 0, V - 1 and log(V - 1).  L - 1 is below a
    fourth of u, so that a total is 1 to a step or two.  Each column is that of a row of every start
    within 16 bytes."""
    e = 16 // (torch.finfo(dt).bits // 8)
    j = torch.tensor(_places(vocab, dt), device=dev).repeat_interleave(e)
    if times > 1:  # as many rows as take the launches of many
        j = j.repeat(times)[:max(1100, len(j))]
    rows = len(j)
    if rows * vocab > 1 << 28:
        pytest.skip("as large as the case of one time")
    print(dt, vocab, rows, flush=True)
    z = _rows(rows, vocab, dt, dev, 3).zero_()
    z.scatter_(1, j[:, None], PEAK)
    other = (j + 1 + vocab // 2) % vocab
    other = torch.where(other == j, (j + 1) % vocab, other)
    ids = other.int()[:, None].contiguous()
    t, dloss = torch.zeros(rows, 1, device=dev), torch.ones(rows, device=dev)
    rest = math.exp(-PEAK)
    assert (vocab - 1) * rest < U / 4
    loss, stats, grad, loss2, grad2 = _calls(z, ids, t, dloss)
    assert (stats[0] == PEAK).all()
    _near(stats[1], 1.0, 4 * U)
    for a in (loss, loss2):
        _near(a, PEAK + (vocab - 1) * rest, 8 * U * PEAK)
    half = torch.finfo(dt).eps / 2
    # exp(-30): an exponent of 43.3 rounded, its exp2 and a product.
    small = rest * (half + 2.0 ** -21 + 4 * U * PEAK * 1.5)
    for b in (grad, grad2):
        rows_ = torch.arange(rows, device=dev)
        _near(b[rows_, j], 1.0, half + 8 * U)
        _near(b[rows_, other], rest - 1, half + 8 * U)
        b[rows_, j], b[rows_, other] = rest, rest
        assert ((b.float() - rest).abs() <= small).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
def test_rows_that_no_registers_hold(dev, dt):
    """Loss and gradient in one call, rows beyond 256 KB, few and many of them.  The loss is log V, between
    8 and 16, where two steps of the logarithm are less than a logit."""
    vocab = 131079 if dt is torch.bfloat16 else 65539
    vocab = 2 * vocab + 1
    for rows in (5, 260):
        z = _rows(rows, vocab, dt, dev, 1).fill_(1.5)
        ids = (torch.arange(rows, device=dev).int() * 997 % vocab)[:, None].contiguous()
        t, dloss = torch.zeros(rows, 1, device=dev), torch.ones(rows, device=dev)
        for a in _calls(z, ids, t, dloss)[0::3]:
            _near(a, math.log(vocab), 2 * 2.0 ** -20)
        assert 8 < math.log(vocab) < 16 and 2 * 2.0 ** -20 < 1 / vocab


def test_a_logit_is_seen():
    """What the comparisons' bounds tell apart, without a GPU: totals without one logit."""
    for dt in TYPES:
        for vocab in _edges(dt):
            if vocab > 1:
                assert abs(1 / vocab - 1 / (vocab - 1)) > 2 * U / vocab
                assert math.log(vocab) - math.log(vocab - 1) > 6 * U * math.log(vocab)
