"""Rotary positions against their float64 definition: both layouts, parts of a head, odd widths,
strides, in place, the inverse as transpose, and the table's scaling."""
import math

import numpy as np
import pytest
import torch

from katsu_amd import _abi, ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16]


def _ref(x, table, pos, interleaved, inverse):
    """The turned x, and the bound of a float32 evaluation rounded once: two products and a sum
    (3 u of sum|a||b|), and half a unit in the last place of the output's type."""
    r = table.shape[1]
    half = r // 2
    y, mag = x.double().clone(), x.double().abs()
    t = table.double()[pos]
    c, s = t[:, None, :half], t[:, None, half:] * (-1 if inverse else 1)
    ia = torch.arange(half) * 2 if interleaved else torch.arange(half)
    ib = ia + 1 if interleaved else ia + half
    a, b = x.double()[..., ia], x.double()[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    mag[..., ia] = mag[..., ib] = a.abs() * c.abs() + b.abs() * s.abs() + a.abs() * s.abs() + \
        b.abs() * c.abs()
    turned = torch.zeros(x.shape[-1], dtype=torch.bool)
    turned[:r] = True
    tol = torch.where(turned, 3 * U * mag + (2.0 ** -8 if x.dtype is torch.bfloat16 else U)
                      * y.abs(), 0.0)
    return y, tol


def _check(got, want, tol):
    assert ((got.double().cpu() - want).abs() <= tol).all()


def _inputs(tokens, heads, kv, d, dt, length, seed=1):
    g = torch.Generator().manual_seed(seed)
    q, k = (torch.randn(tokens, h, d, generator=g).to(dt) for h in (heads, kv))
    pos = torch.randint(0, length, (tokens,), generator=g, dtype=torch.int32)
    return q, k, pos


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot", [(128, 128), (128, 64), (72, 36), (40, 20), (64, 2), (5, 4),
                                   (80, 80), (96, 48)])
def test_layouts(dev, dt, interleaved, d, rot):
    table = ops.rotary_table(50, rot, device=dev)
    for tokens, heads, kv in ((1, 1, 1), (7, 5, 2), (300, 8, 2)):
        q, k, pos = _inputs(tokens, heads, kv, d, dt, 50)
        for inverse in (False, True):
            print(dt, interleaved, d, rot, tokens, heads, kv, inverse, flush=True)
            a, b = ops.rotary(q.to(dev), k.to(dev), table, pos.to(dev), interleaved, inverse)
            for x, y in ((q, a), (k, b)):
                _check(y, *_ref(x, table.cpu(), pos.long(), interleaved, inverse))


@pytest.mark.parametrize("dt", TYPES)
def test_one_operand_positions_strides_in_place(dev, dt):
    """k absent; positions 0, 1, ..; q and k as views of one projection, turned in place, the rest
    of the buffer untouched."""
    t, heads, kv, d, rot = 33, 4, 2, 64, 32
    table = ops.rotary_table(64, rot, device=dev)
    g = torch.Generator().manual_seed(2)
    host = torch.randn(t, heads + 2 * kv, d, generator=g).to(dt)
    x = host.to(dev)
    q, k = x[:, :heads], x[:, heads:heads + kv]
    ops.rotary(q, k, table, out_q=q, out_k=k)
    want, tol = _ref(host, table.cpu(), torch.arange(t), False, False)
    want[:, heads + kv:], tol[:, heads + kv:] = host[:, heads + kv:].double(), 0
    _check(x, want, tol)
    a, b = ops.rotary(host.to(dev), None, table)
    assert b is None
    _check(a, *_ref(host, table.cpu(), torch.arange(t), False, False))
    odd = torch.randn(t * 3 * 7 + 1, generator=g).to(dt)  # rows at odd addresses
    y, _ = ops.rotary(odd.to(dev)[1:].view(t, 3, 7), None, ops.rotary_table(40, 6, device=dev))
    _check(y, *_ref(odd[1:].view(t, 3, 7), ops.rotary_table(40, 6, device=dev).cpu(),
                    torch.arange(t), False, False))


@pytest.mark.parametrize("interleaved", [False, True])
def test_inverse_is_the_gradient(dev, interleaved):
    """<turn(x), y> = <x, turn back(y)>: the gradient; and central differences of the float64
    turn along a direction (linear, so exact but for rounding, 1e-16 / 1e-4)."""
    t, h, d = 20, 3, 64
    table = ops.rotary_table(100, d, device=dev)
    x, y, pos = _inputs(t, h, h, d, torch.float32, 100)
    back = ops.rotary(y.to(dev), None, table, pos.to(dev), interleaved, True)[0].double().cpu()
    _, tol = _ref(y, table.cpu(), pos.long(), interleaved, True)

    def loss(z):
        return (_ref(z, table.cpu(), pos.long(), interleaved, False)[0] * y.double()).sum()
    u = torch.randn(x.shape, dtype=torch.float64)
    want = (loss(x.double() + 1e-4 * u) - loss(x.double() - 1e-4 * u)) / 2e-4
    assert abs(want - (back * u).sum()) <= (tol * u.abs()).sum() + 1e-9


def test_positions_outside_the_table(dev):
    """Taken as its ends: no access outside it."""
    table = ops.rotary_table(10, 8, device=dev)
    x = torch.randn(4, 1, 8)
    pos = torch.tensor([-5, 1 << 30, 0, 9], dtype=torch.int32)
    y, _ = ops.rotary(x.to(dev), None, table, pos.to(dev))
    _check(y, *_ref(x, table.cpu(), torch.tensor([0, 9, 0, 9]), False, False))


@pytest.mark.parametrize("factor,by_wavelength", [(1.0, True), (4.0, False), (4.0, True)])
def test_table(dev, factor, by_wavelength):
    """Against numpy in float64: an angle's error is some units of 2^-53 of it (its power and
    product), the result's a unit of 2^-24."""
    n, r, base = 70000, 64, 10000.0
    t = ops.rotary_table(n, r, base, factor, by_wavelength, device=dev).double().cpu().numpy()
    f = base ** (-2.0 * np.arange(r // 2) / r)
    amp = 1.0
    if factor != 1 and by_wavelength:
        keep = np.clip((n / factor * f / (2 * math.pi) - 1) / 31, 0, 1)
        f, amp = f * (keep + (1 - keep) / factor), 0.1 * math.log(factor) + 1
    else:
        f = f / factor
    angle = np.arange(n)[:, None] * f
    tol = amp * (2.0 ** -24 + 8 * 2.0 ** -53 * angle) + 1e-14
    assert (np.abs(t[:, :r // 2] - amp * np.cos(angle)) <= tol).all()
    assert (np.abs(t[:, r // 2:] - amp * np.sin(angle)) <= tol).all()


def test_refusals(dev):
    table = ops.rotary_table(10, 8, device=dev)
    q = torch.zeros(4, 2, 16, device=dev)
    pos = torch.zeros(4, dtype=torch.int32, device=dev)
    for args, kw in (((q.double(), None, table), {}), ((q, q.bfloat16(), table), {}),
                     ((q.cpu(), None, table), {}), ((q, q[:2], table), {}),
                     ((q, q[..., :8], table), {}), ((q[..., ::2], None, table), {}),
                     ((q, None, table.bfloat16()), {}), ((q, None, table[:, ::2]), {}),
                     ((q, None, table, pos.long()), {}), ((q, None, table, pos[:3]), {}),
                     ((q[0], None, table), {}), ((q, None, table), dict(out_q=q[:2]))):
        with pytest.raises(ValueError):
            ops.rotary(*args, **kw)
    for t in (torch.zeros(10, 7, device=dev), torch.zeros(10, 18, device=dev),
              torch.zeros(0, 8, device=dev)):
        with pytest.raises(_abi.KatsuError) as e:
            ops.rotary(q, None, t)
        assert e.value.status == _abi.E_INVALID
    for args in ((10, 7), (10, 8, 0.0), (10, 8, 1e4, 0.5), (10, 8, math.nan)):
        with pytest.raises(_abi.KatsuError):
            ops.rotary_table(*args, device=dev)
    assert ops.rotary(q[:0], q[:0], table)[0].shape == (0, 2, 16)
