"""Distillation at both ends of its ranges: a teacher's column that the student masks with the type's
lowest value, and the smallest and largest temperatures."""
import math

import pytest
import torch

from katsu_amd import ops
from tests.distill_ref import close, reference
from tests.test_gpu_distillation import TYPES, _all, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("tau", [0.125, 0.5, 0.9, 1.0, 1.5])
@pytest.mark.parametrize("rows", [3, 280])
def test_lowest_column_of_the_teacher(dev, dt, tau, rows):
    """tau p times the lowest value is a number that float32 holds; the lowest value over tau is not."""
    z, ids, t, dloss = _inputs(rows, 900, 10, dt, pad=False)
    ids[:] = torch.arange(10) * 7
    z[:, 14] = torch.finfo(dt).min        # the third entry's
    t[:, 2] = torch.cat([t[:, :2], t[:, 3:]], 1).amax(1) - 0.4      # below half of the total
    want, dz, ltol, gtol = reference(z, ids, t, tau, dloss)
    assert (want > 1e33).all() and (want < 3e38).all() and (ltol < 1e-5 * want).all()
    assert (gtol < 1e-2 * dloss.abs()[:, None]).all()
    loss, _, grad, loss2, grad2 = _all(dev, z, ids, t, dloss, tau)
    for a, b in ((loss, grad), (loss2, grad2)):
        close(a, want, ltol)
        close(b, dz, gtol)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("tau", [4.3e-39, 1e-30, 1e-20, 1e-3, 1e3, 1e15])
@pytest.mark.parametrize("rows", [3, 280])
def test_temperatures(dev, dt, tau, rows):
    """Down to where 1.44 / tau is the largest float32, and tau^2 none at all.  A difference of logits
    beyond tau leaves a probability of zero, as the formula does."""
    tau = torch.tensor(tau).item()  # as the call takes it
    z, ids, t, dloss = _inputs(rows, 300, 8, dt, pad=False)
    t[:, 0] = 9.0                         # one entry is the largest
    want, dz, ltol, gtol = reference(z, ids, t, tau, dloss)
    if tau < 1:                           # what is left are differences of logits, times tau
        assert (ltol <= 1e-5 * (want + tau) + 2.0 ** -140).all()
    loss, _, grad, loss2, grad2 = _all(dev, z, ids, t, dloss, tau)
    for a, b in ((loss, grad), (loss2, grad2)):
        close(a, want, ltol)
        close(b, dz, gtol)


@pytest.mark.parametrize("rows", [2, 280])
def test_infinite_and_zero_losses(dev, rows):
    """A teacher's column at -inf is an infinite loss whatever the temperature; a row of one column has
    none."""
    z, ids, t, dloss = _inputs(rows, 50, 2, torch.float32, pad=False)
    ids[:, 0], ids[:, 1], t[:] = 3, 9, 0.0
    z[:, 9] = -math.inf
    one = (z[:, :1], torch.zeros_like(ids[:, :1]), t[:, :1], dloss)
    for tau in (1e-30, 1e-3, 1.0, 1e3, 1e25):
        loss, _, _, loss2, _ = _all(dev, z, ids, t, dloss, tau)
        assert (loss == math.inf).all() and (loss2 == math.inf).all(), tau
        loss, _, grad, loss2, grad2 = _all(dev, *one, tau)
        assert not loss.any() and not loss2.any(), tau
        assert not grad.any() and not grad2.any(), tau


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("tau", [0.125, 0.3, 0.49])
@pytest.mark.parametrize("rows", [3, 280])
def test_all_of_the_teacher_masked(dev, dt, tau, rows):
    """Every column that the teacher names at the lowest value, so that a sum of the differences, weighted
    with probabilities whose sum may be above 1, is no float32 before it is multiplied by tau; and with
    a logit near the largest value, as one difference is none."""
    low = torch.finfo(dt).min
    z, ids, t, dloss = _inputs(rows, 400, 9, dt, pad=False)
    ids[:] = torch.arange(9) * 7
    z[:, :100] = low
    z[1::3, 300] = -low * 0.9
    want, dz, ltol, gtol = reference(z, ids, t, tau, dloss)
    assert (want > 1e37).all() and (want < 3.39e38).all() and (ltol < 1e-5 * want).all()
    loss, _, grad, loss2, grad2 = _all(dev, z, ids, t, dloss, tau)
    for a, b in ((loss, grad), (loss2, grad2)):
        close(a, want, ltol)
        close(b, dz, gtol)
