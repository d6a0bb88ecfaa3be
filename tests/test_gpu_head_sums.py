"""The norms of heads: the weights' gradient, a sum over all tokens and heads, where float32's roundings can
be counted."""
import pytest
import torch

from katsu_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", ["q", "k"])
@pytest.mark.parametrize("part", [0x155555, 0x0aaaab, 0x1fffff])
def test_equal_terms(dev, which, part):
    """512 heads of ones, whose gradients are all 1 + part 2^-21: a block's 16 heads and sums in pairs of
    the blocks' are powers of two, or three powers of two, times it, which float32 holds.  Added one
    after the other the 32 sums of blocks are off by up to 4 u of the whole."""
    c = 1 + part * 2.0 ** -21
    x, w = torch.ones(512, 1, 128, device=dev), torch.ones(128, device=dev)
    g = torch.full_like(x, c)
    if which == "q":
        _, _, dw, _ = ops.qk_norm_rotary_backward(g, None, x, None, w_q=w, eps=0.0)
    else:
        _, _, _, dw = ops.qk_norm_rotary_backward(g[:, :0], g, x[:, :0], x, w_k=w, eps=0.0)
    assert (dw == 512 * c).all()
