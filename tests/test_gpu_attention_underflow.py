"""A key that a query sees with a score so low that its probability is zero in float32: its value is
multiplied by that zero all the same, so a NaN or an infinity there reaches the output as it does
in the formula, wherever the key lies."""
import math

import pytest
import torch

from katsu_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128, 40])
@pytest.mark.parametrize("lq", [1, 5, 200])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_value_without_weight(dev, dt, d, lq, bad):
    """One of every four tiles of 32 keys has scores 400 below the others'; keys of the first such
    tile and of the last hold `bad` in a channel each, which every query sees (not causal)."""
    t = 1100
    g = torch.Generator().manual_seed(1)
    q = torch.zeros(lq, 4, d)
    q[..., 0] = 1
    k = torch.zeros(t, 2, d)
    low = (torch.arange(t) // 32) % 4 == 1
    k[low, :, 0] = -400
    v = torch.randn(t, 2, d, generator=g)
    first, last = int(low.nonzero()[0]), int(low.nonzero()[-1])
    v[first, :, 3] = bad
    v[last, :, 7] = -bad
    out, lse = ops.attention(*(x.to(dt).to(dev) for x in (q, k, v)), causal=False, scale=1.0)
    want = torch.softmax((q[:, 0] @ k[:, 0].T), 1)[..., None] * v[:, 0]  # 0 * bad is NaN
    want = want.sum(1).isnan()  # [lq, d]
    assert want.sum() == 2 * lq
    assert torch.equal(out[:, 0].isnan().cpu(), want) and torch.equal(out[:, 3].isnan().cpu(), want)
    assert lse.isfinite().all()
