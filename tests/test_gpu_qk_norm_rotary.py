"""The norm of query and key heads with their turn, and its gradient, against the float64 definition:
widths, parts that turn, layouts, strides, in place; the gradient also against differences."""
import pytest
import torch

from katsu_amd import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16]
EPS = 1e-6
SHAPES = [(128, 128), (128, 64), (72, 36), (40, 20), (64, 2), (5, 4), (80, 80), (96, 48), (1, 0),
          (7, 0), (64, 0), (16, 16), (256, 256), (512, 512), (510, 510), (511, 2), (300, 100),
          (130, 26)]


def _half(dt):
    return torch.finfo(dt).eps / 2


def _gamma(n):
    return n * U / (1 - n * U)


def _pairs(rot, interleaved):
    half = rot // 2
    a = torch.arange(half) * 2 if interleaved else torch.arange(half)
    return a, a + (1 if interleaved else half)


def _turn(x, table, pos, interleaved, back=False, size=False):
    """x's heads turned in float64; size: |a||cos| + |b||sin| in the places of the sums."""
    if table is None:
        return x.clone()
    half = table.shape[1] // 2
    t = table.double()[pos.long().clamp(0, len(table) - 1)][:, None]
    c, s = t[..., :half], t[..., half:] * (-1 if back else 1)
    i, j = _pairs(table.shape[1], interleaved)
    y, a, b = x.clone(), x[..., i], x[..., j]
    if size:
        a, b, c, s = a.abs(), b.abs(), c.abs(), s.abs()
    y[..., i], y[..., j] = a * c + (1 if size else -1) * b * s, a * s + b * c
    return y


def _forward(x, w, table, pos, interleaved):
    """(y, bound).  The sum of D squares, its mean, eps and the hardware's root: gamma(D + 8) of a
    norm; two products and a sum of the turn: 4 u; and the output's rounding."""
    d = x.shape[2]
    n = x.double() / (x.double().square().mean(-1, keepdim=True) + EPS).sqrt()
    n = n if w is None else n * w.double()
    y, mag = (_turn(n, table, pos, interleaved, size=s) for s in (False, True))
    tol = (_gamma(d + 8) + 4 * U) * mag.abs()
    return y, tol + _half(x.dtype) * (y.abs() + tol)


def _backward(dy, x, w, table, pos, interleaved):
    """(dx, dw, their bounds).  r's relative error counts three times in dx, its two sums of D
    products once: gamma(3 D + 40) of the terms' sizes; dw is a sum over tokens and heads."""
    t, h, d = x.shape
    xd, g = x.double(), _turn(dy.double(), table, pos, interleaved, True)
    mag = _turn(dy.double(), table, pos, interleaved, True, True).abs()
    r = 1 / (xd.square().mean(-1, keepdim=True) + EPS).sqrt()
    dw, dwt = (g * xd * r).sum((0, 1)), (mag * xd.abs() * r).sum((0, 1))
    wd = torch.ones(d, dtype=torch.float64) if w is None else w.double()
    g, mag = g * wd, mag * wd.abs()
    dx = r * g - xd * r ** 3 * (g * xd).mean(-1, keepdim=True)
    tol = r * mag + xd.abs() * r ** 3 * (mag * xd.abs()).mean(-1, keepdim=True)
    tol = _gamma(3 * d + 40) * tol
    dwt = _gamma(t * h + d + 16) * dwt
    half = _half(x.dtype)
    return dx, dw, tol + half * (dx.abs() + tol), dwt + half * (dw.abs() + dwt)


def _inputs(tokens, heads, kv, d, dt, length, seed=1):
    g = torch.Generator().manual_seed(seed)
    q, k, dq, dk = (torch.randn(tokens, h, d, generator=g).to(dt) for h in (heads, kv) * 2)
    w_q, w_k = (1 + 0.3 * torch.randn(d, generator=g)).to(dt), torch.randn(d, generator=g).to(dt)
    pos = torch.randint(-2, length + 3, (tokens,), generator=g, dtype=torch.int32)
    return q, k, dq, dk, w_q, w_k, pos


def _close(got, want, tol):
    err = (got.double().cpu() - want).abs()
    assert (err <= tol).all(), (err - tol).max()


def _on(dev, *ts):
    return [None if t is None else t.to(dev) for t in ts]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot", SHAPES)
def test_both_ways(dev, dt, interleaved, d, rot):
    """Positions outside the table are taken as its ends."""
    table = ops.rotary_table(50, rot, device=dev) if rot else None
    for tokens, heads, kv in ((1, 1, 1), (7, 5, 2), (90, 3, 1)):
        print(dt, interleaved, d, rot, tokens, heads, kv, flush=True)
        q, k, dq, dk, w_q, w_k, pos = _inputs(tokens, heads, kv, d, dt, 50)
        pos = pos if rot else None
        cpu = None if table is None else table.cpu()
        how = dict(table=table, positions=None if pos is None else pos.to(dev), w_q=w_q.to(dev),
                   w_k=w_k.to(dev), eps=EPS, interleaved=interleaved)
        x, g = _on(dev, q, k), _on(dev, dq, dk)
        for got, t, w in zip(ops.qk_norm_rotary(*x, **how), (q, k), (w_q, w_k)):
            _close(got, *_forward(t, w, cpu, pos, interleaved))
        got = ops.qk_norm_rotary_backward(*g, *x, **how)
        for i, (t, w, dy) in enumerate(((q, w_q, dq), (k, w_k, dk))):
            dx, dw, xt, wt = _backward(dy, t, w, cpu, pos, interleaved)
            _close(got[i], dx, xt)
            _close(got[i + 2], dw, wt)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("tokens,heads,kv", [(2000, 8, 2), (3, 64, 64), (1, 300, 3), (4097, 1, 1)])
def test_sizes(dev, dt, tokens, heads, kv):
    q, k, dq, dk, w_q, w_k, pos = _inputs(tokens, heads, kv, 64, dt, 999)
    table = ops.rotary_table(999, 64, device=dev)
    how = dict(table=table, positions=pos.to(dev), w_q=w_q.to(dev), w_k=w_k.to(dev), eps=EPS)
    x, g = _on(dev, q, k), _on(dev, dq, dk)
    for got, t, w in zip(ops.qk_norm_rotary(*x, **how), (q, k), (w_q, w_k)):
        _close(got, *_forward(t, w, table.cpu(), pos, False))
    got = ops.qk_norm_rotary_backward(*g, *x, **how)
    for i, (t, w, dy) in enumerate(((q, w_q, dq), (k, w_k, dk))):
        dx, dw, xt, wt = _backward(dy, t, w, table.cpu(), pos, False)
        _close(got[i], dx, xt)
        _close(got[i + 2], dw, wt)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("d", [64, 33])
def test_views_in_place_and_absent_operands(dev, dt, d):
    """q and k as parts of one projection, in place, the values beside them untouched; positions
    0, 1, ..; gradients in place; no weights, no k."""
    t, heads, kv, rot = 37, 4, 2, d // 4 * 2
    table = ops.rotary_table(64, rot, device=dev)
    g = torch.Generator().manual_seed(2)
    host = torch.randn(t, heads + 2 * kv, d, generator=g).to(dt)
    grad = torch.randn(t, heads + 2 * kv, d, generator=g).to(dt)
    pos = torch.arange(t)
    parts = slice(0, heads), slice(heads, heads + kv)
    x, dy = host.to(dev), grad.to(dev)
    gq, gk = dy[:, parts[0]], dy[:, parts[1]]
    a, b, dwa, dwb = ops.qk_norm_rotary_backward(gq, gk, x[:, parts[0]], x[:, parts[1]], table,
                                                 out_q=gq, out_k=gk, eps=EPS)
    assert dwa is None and dwb is None and a is gq and b is gk
    for p, got in zip(parts, (a, b)):
        dx, _, tol, _ = _backward(grad[:, p], host[:, p], None, table.cpu(), pos, False)
        _close(got, dx, tol)
    assert torch.equal(dy[:, heads + kv:].cpu(), grad[:, heads + kv:])
    w = torch.randn(d, generator=g).to(dt)
    ops.qk_norm_rotary(x[:, parts[0]], x[:, parts[1]], table, w_k=w.to(dev), eps=EPS,
                       out_q=x[:, parts[0]], out_k=x[:, parts[1]])
    for p, wt in zip(parts, (None, w)):
        _close(x[:, p], *_forward(host[:, p], wt, table.cpu(), pos, False))
    assert torch.equal(x[:, heads + kv:].cpu(), host[:, heads + kv:])
    a, b = ops.qk_norm_rotary(host.to(dev), None, table, eps=EPS)
    assert b is None
    _close(a, *_forward(host, None, table.cpu(), pos, False))
    a, b, dw, none = ops.qk_norm_rotary_backward(grad.to(dev), None, host.to(dev), None, table,
                                                 w_q=w.to(dev), eps=EPS)
    dx, want, tol, wtol = _backward(grad, host, w, table.cpu(), pos, False)
    _close(a, dx, tol)
    _close(dw, want, wtol)
    assert b is None and none is None


@pytest.mark.parametrize("dt", TYPES)
def test_heads_first_and_shared(dev, dt):
    """[heads, tokens, channels] memory; a gradient and an operand that all heads share."""
    g = torch.Generator().manual_seed(3)
    host = torch.randn(6, 50, 48, generator=g).to(dt)
    x = host.to(dev).transpose(0, 1)
    one = torch.randn(50, 1, 48, generator=g).to(dt)
    w = torch.randn(48, generator=g).to(dt)
    table = ops.rotary_table(50, 48, device=dev)
    how = dict(table=table, w_q=w.to(dev), eps=EPS, interleaved=True)
    a, _ = ops.qk_norm_rotary(x, None, **how)
    pos = torch.arange(50)
    _close(a, *_forward(host.transpose(0, 1), w, table.cpu(), pos, True))
    for xs, xh in ((x, host.transpose(0, 1)), (one.to(dev).expand(50, 6, 48),
                                               one.expand(50, 6, 48))):
        a, _, dw, _ = ops.qk_norm_rotary_backward(one.to(dev).expand(50, 6, 48), None, xs, None,
                                                  **how)
        dx, want, tol, wtol = _backward(one.expand(50, 6, 48), xh, w, table.cpu(), pos, True)
        _close(a, dx, tol)
        _close(dw, want, wtol)


def test_gradient_by_differences(dev):
    """<dy, y(x + h e) - y(x - h e)> / 2h in float64 against <dx, e>, and so for the weights: the
    differences' own error is h^2 / 6 of the third derivative, 1e-7 of the value at h = 1e-4."""
    q, _, dq, _, w, _, pos = _inputs(9, 2, 1, 32, torch.float32, 40, 4)
    table = ops.rotary_table(40, 16, device=dev)
    g = torch.Generator().manual_seed(5)
    e, ew = torch.randn(q.shape, generator=g).double(), torch.randn(32, generator=g).double()

    def y(x, wt):
        n = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * wt
        return (_turn(n, table.cpu(), pos, False) * dq.double()).sum()
    h = 1e-4
    by_x = (y(q + h * e, w.double()) - y(q - h * e, w.double())) / (2 * h)
    by_w = (y(q.double(), w + h * ew) - y(q.double(), w - h * ew)) / (2 * h)
    dx, _, dw, _ = ops.qk_norm_rotary_backward(dq.to(dev), None, q.to(dev), None, table,
                                               pos.to(dev), w_q=w.to(dev), eps=EPS)
    # 576 products of values of order one, each within 1e-5.
    for got, want, v in ((dx, by_x, e), (dw, by_w, ew)):
        got = got.double().cpu()
        assert abs((got * v).sum() - want) <= 1e-5 * (got * v).abs().sum()


@pytest.mark.parametrize("dt", TYPES)
def test_zeros_and_non_finite(dev, dt):
    """A head of zeros gives zeros (eps > 0); NaN and infinities stay in their head."""
    q, _, dq, _, w, _, pos = _inputs(12, 3, 1, 64, dt, 30, 6)
    q[2, 1] = 0
    q[5, 0, 7], q[6, 2, 63] = float("nan"), float("inf")
    table = ops.rotary_table(30, 32, device=dev)
    how = dict(table=table, positions=pos.to(dev), w_q=w.to(dev), eps=EPS)
    y, _ = ops.qk_norm_rotary(q.to(dev), None, **how)
    y = y.cpu()
    assert (y[2, 1] == 0).all() and y[5, 0].isnan().all()
    want, tol = _forward(q, w, table.cpu(), pos, False)
    ok = torch.ones(12, 3, dtype=torch.bool)
    ok[5, 0] = ok[6, 2] = False
    _close(y[ok], want[ok], tol[ok])
    dx, _, dw, _ = ops.qk_norm_rotary_backward(dq.to(dev), None, q.to(dev), None, **how)
    want, _, tol, _ = _backward(dq, q, w, table.cpu(), pos, False)
    _close(dx.cpu()[ok], want[ok], tol[ok])
    assert dw.isnan().any()


def test_same_bits(dev):
    """Calls, replays of a graph, another stream, an own workspace."""
    q, k, dq, dk, w_q, w_k, pos = _on(dev, *_inputs(1500, 6, 2, 80, torch.float32, 1500))
    table = ops.rotary_table(1500, 40, device=dev)
    how = dict(table=table, positions=pos, w_q=w_q, w_k=w_k)
    want = ops.qk_norm_rotary(q, k, **how) + ops.qk_norm_rotary_backward(dq, dk, q, k, **how)
    ws = torch.empty(ops.qk_norm_rotary_workspace_bytes(q, k), dtype=torch.uint8, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        own = ops.qk_norm_rotary_backward(dq, dk, q, k, workspace=ws, **how)
        side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(own, want[2:]))
    x, other = q.clone(), torch.randn_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.qk_norm_rotary(x, k, **how) + ops.qk_norm_rotary_backward(dq, dk, x, k, **how)
    for src in (q, other, q):
        x.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        now = ops.qk_norm_rotary(src, k, **how) + ops.qk_norm_rotary_backward(dq, dk, src, k,
                                                                              **how)
        assert all(torch.equal(a, b) for a, b in zip(got, now))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_no_tokens_and_no_heads(dev):
    """Nothing to turn: the weights' gradients are zeros."""
    w = torch.ones(16, device=dev)
    for q, k in ((torch.zeros(0, 3, 16, device=dev), torch.zeros(0, 1, 16, device=dev)),
                 (torch.zeros(5, 0, 16, device=dev), torch.ones(5, 2, 16, device=dev))):
        a, b = ops.qk_norm_rotary(q, k, w_q=w, w_k=w)
        assert a.shape == q.shape and b.shape == k.shape
        dq, dk, dw_q, dw_k = ops.qk_norm_rotary_backward(q, k, q, k, w_q=w, w_k=w)
        assert dq.shape == q.shape and dk.shape == k.shape and not dw_q.any()
        assert dw_k.any() == (k.numel() > 0)


def test_large_offsets(dev):
    """Heads beyond 2^31 elements."""
    tokens, heads, d = 70_000, 248, 128
    x = torch.zeros(tokens, heads, d, dtype=torch.bfloat16, device=dev)
    g = torch.Generator().manual_seed(8)
    host, grad = (torch.randn(2, heads, d, generator=g).bfloat16() for _ in range(2))
    x[-2:] = host.to(dev)
    dy = torch.zeros_like(x)
    dy[-2:] = grad.to(dev)
    table = ops.rotary_table(tokens, 64, device=dev)
    w = torch.randn(d, generator=g).bfloat16()
    pos = torch.arange(tokens - 2, tokens)
    y, _ = ops.qk_norm_rotary(x, None, table, w_q=w.to(dev), eps=EPS)
    _close(y[-2:], *_forward(host, w, table.cpu(), pos, False))
    assert not y[:-2].any()
    dx, _, dw, _ = ops.qk_norm_rotary_backward(dy, None, x, None, table, w_q=w.to(dev), eps=EPS,
                                               out_q=dy)
    want, dwant, tol, wtol = _backward(grad, host, w, table.cpu(), pos, False)
    _close(dx[-2:], want, tol)
    # The sum runs over all tokens, of which the others add zeros.
    _close(dw, dwant, wtol)
    assert not dx[:-2].any()
