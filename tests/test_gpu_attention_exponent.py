"""The probabilities that attention's gradient computes again from lse: as exact as the scores are,
whatever the size of lse / scale."""
import pytest
import torch

from katsu_amd import ops
from tests.attention_ref import U, assert_close, backward, forward

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [128, 64, 40, 20])
@pytest.mark.parametrize("heads,kv", [(4, 2), (2, 2)])
def test_probabilities(dev, d, heads, kv):
    """Scores that are whole numbers, sums of products up to 64 d / 2 on the way, and an lse that is
    none: with one row's dout all ones and the others zero, dv is that row's probabilities.

    Bound: the exponent log2(e) (s / 8 - lse) is one fused multiply-add (u of itself) of scale
    log2(e) (u: the constant; 1/8 is exact) and log2(e) lse (2 u: the constant and the product);
    ln 2 of its error is the probability's, and 2^-22 for the hardware's 2^x; the sum over a
    group's heads adds u each."""
    t, row, lse = 300, 37, 8.1
    g = torch.Generator().manual_seed(2)
    q = torch.full((t, heads, d), 8.0)
    q[..., d // 2:] = -8.0
    k = torch.full((t, kv, d), 8.0)
    k[..., d // 2:] += torch.randint(-1, 2, (t, kv, d // 2), generator=g)
    v = torch.randn(t, kv, d, generator=g)
    do = torch.zeros(t, heads, d)
    do[row] = 1.0
    stats = torch.full((heads, t), lse)
    out = torch.zeros_like(q)
    _, _, dv = ops.attention_backward(*(x.to(dev) for x in (do, q, k, v, out, stats)),
                                      causal=False, scale=0.125)
    lse64 = stats[0, 0].double()
    # The heads of a group have the same q, so the same row of probabilities.
    s = (q[row, 0].double() * k.double()).sum(-1)  # [t, kv]
    want = (s / 8 - lse64).exp()
    e = U * (s.abs() / 8 + 2 * lse64 + (s / 8 - lse64).abs()) + 2.0 ** -22 + (heads // kv) * U
    want = want * (heads // kv)
    assert_close(dv, want[..., None].expand(t, kv, d), (e * want)[..., None].expand(t, kv, d), "dv")


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128, 40])
def test_smallest_scale(dev, dt, d):
    """A scale next to the smallest normal number: lse / scale is beyond float32."""
    t, scale = 100, 2.0 ** -126
    g = torch.Generator().manual_seed(3)
    q, k, v, do = (torch.randn(t, 2, d, generator=g).to(dt) for _ in range(4))
    card = [x.to(dev) for x in (q, k, v)]
    out, lse = ops.attention(*card, scale=scale)
    ro, rl, to, tl = forward(q, k, v, [t], [t], True, scale)
    assert_close(out, ro, to, "out")
    assert_close(lse, rl, tl, "lse")
    _, _, dv = ops.attention_backward(do.to(dev), *card, out, lse, scale=scale)
    want, tol = backward(do, q, k, v, [t], [t], True, scale)
    assert_close(dv, want[2], tol[2], "dv")
