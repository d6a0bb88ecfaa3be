"""The global gradient norm and clipping against float64: both types in one call, tensors of zero and
one value, more of them than one launch takes, in place and not, sums that would overflow."""
import math

import pytest
import torch

from katsu_amd import _abi, ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _grads(counts, dev, seed=1, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * std).to([torch.float32, torch.bfloat16][i % 2]).to(dev)
            for i, n in enumerate(counts)]


def _check(grads, max_norm, out, norm):
    """The norm within 2 u (float64 sums, one rounding); an output within 2 u (the factor's
    rounding and the product's) and its type's rounding."""
    total = math.sqrt(math.fsum(g.double().square().sum().item() for g in grads))
    assert abs(norm.item() - total) <= 2 * U * total
    coef = min(1.0, max_norm / (total + 1e-6))
    for g, o in zip(grads, out):
        want = g.double() * coef
        unit = 2.0 ** -8 if g.dtype is torch.bfloat16 else U
        # 2^-134: half the smallest bfloat16 and float32 step.
        assert ((o.double() - want).abs() <= (2 * U + unit) * want.abs() + 2.0 ** -134).all()


COUNTS = [[1], [0, 5, 0], [16384], [16385, 3, 100000, 1, 7],
          [(37 * i) % 3000 for i in range(300)], [3 << 20, 5, 1 << 20]]


@pytest.mark.parametrize("counts", COUNTS)
@pytest.mark.parametrize("max_norm", [1.0, 1e9, 0.0])
def test_clip(dev, counts, max_norm):
    print(len(counts), sum(counts), max_norm, flush=True)
    grads = _grads(counts, dev)
    out = [torch.empty_like(g) for g in grads]
    keep = [g.clone() for g in grads]
    norm = ops.clip_grad_norm(grads, max_norm, out=out)
    assert all(torch.equal(a, b) for a, b in zip(grads, keep))
    _check(keep, max_norm, out, norm)
    norm2 = ops.clip_grad_norm(grads, max_norm)
    assert torch.equal(norm, norm2)
    assert all(torch.equal(a, b) for a, b in zip(grads, out))


def test_odd_addresses_and_shapes(dev):
    base = _grads([1001, 1001], dev)
    grads = [base[0][1:], base[1][1:].view(8, 125)]
    keep = [g.clone() for g in grads]
    norm = ops.clip_grad_norm(grads, 0.5)
    _check(keep, 0.5, grads, norm)


@pytest.mark.parametrize("std", [1e-30, 1e30])
def test_squares_outside_float32(dev, std):
    grads = _grads([1000, 1000], dev, std=std)
    out = [torch.empty_like(g) for g in grads]
    _check(grads, 1.0, out, ops.clip_grad_norm(grads, 1.0, out=out))


def test_nonfinite(dev):
    """A NaN norm makes everything NaN; an infinite one zeros, NaN at the infinite value."""
    grads = _grads([100, 100], dev)
    grads[0][3] = math.nan
    assert ops.clip_grad_norm(grads, 1.0).isnan().all()
    assert all(g.isnan().all() for g in grads)
    grads = _grads([100, 100], dev)
    grads[0][3] = math.inf
    assert ops.clip_grad_norm(grads, 1.0).isinf().all()
    assert grads[0][3].isnan() and (grads[0][:3] == 0).all() and (grads[1] == 0).all()


def test_empty_tensors_only(dev):
    assert ops.clip_grad_norm([torch.zeros(0, device=dev)], 1.0).item() == 0


def test_graph(dev):
    grads = _grads([70000, 300], dev)
    out = [torch.empty_like(g) for g in grads]
    ops.clip_grad_norm(grads, 1.0, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = ops.clip_grad_norm(grads, 1.0, out=out)
    for seed in (1, 2, 3):
        for g, n in zip(grads, _grads([70000, 300], dev, seed)):
            g.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in out]
        want = ops.clip_grad_norm(grads, 1.0, out=out)
        torch.cuda.synchronize()
        assert torch.equal(norm, want) and all(torch.equal(a, b) for a, b in zip(got, out))


def test_refusals(dev):
    g = torch.zeros(4, 6, device=dev)
    for args, kw in ((([], 1.0), {}), (([g.half()], 1.0), {}), (([g.cpu()], 1.0), {}),
                     (([g.t()], 1.0), {}), (([g, g], 1.0), dict(out=[g])),
                     (([g], 1.0), dict(out=[g.bfloat16()])), (([g], 1.0), dict(out=[g[:2]]))):
        with pytest.raises(ValueError):
            ops.clip_grad_norm(*args, **kw)
    for m in (-1.0, math.nan):
        with pytest.raises(_abi.KatsuError) as e:
            ops.clip_grad_norm([g], m)
        assert e.value.status == _abi.E_INVALID
