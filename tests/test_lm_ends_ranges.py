"""The largest and smallest values that the embedding, the norms of heads and distillation take, and what
lies beyond them.  No kernel is launched."""
import ctypes

import pytest

from katsu_amd import _abi
from tests.test_lm_ends import L, P, _distill

NONE = [None] * 6


@pytest.mark.parametrize("tau", [2.94e-39, 3e-39, 4.2e-39, 4.23e-39])
def test_temperature_too_small(tau):
    """log2(e) / tau is infinite, 1 / tau is not: a difference of zero times it is NaN."""
    tau = ctypes.c_float(tau).value
    assert 1 / tau < 3.4028235e38 < 1.4426950408889634 / tau
    for rows in (0, 2):
        d = _distill(temperature=tau, rows=rows)
        assert L.katsu_hip_distillation_dev(d, *[P] * 5, None) == _abi.E_INVALID
        assert L.katsu_hip_distillation_bwd_dev(d, *[P] * 6, None) == _abi.E_INVALID
        assert L.katsu_hip_distillation_step_dev(d, *[P] * 6, None) == _abi.E_INVALID


@pytest.mark.parametrize("tau", [4.24e-39, 1e-30, 1.0, 3.4e38])
def test_temperature(tau):
    d = _distill(temperature=tau, rows=0)
    assert L.katsu_hip_distillation_dev(d, *NONE[:5], None) == _abi.OK
    assert L.katsu_hip_distillation_bwd_dev(d, *NONE, None) == _abi.OK
    assert L.katsu_hip_distillation_step_dev(d, *NONE, None) == _abi.OK
