"""The norms, gate and residual between two blocks and their gradient against float64: both types,
every set of operands, widths from one to the largest, one row to many."""
import math

import pytest
import torch

from katsu_amd import _abi, ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16]
EPS = 1e-6


def _unit(dt):
    return 2.0 ** -8 if dt is torch.bfloat16 else U


def _gamma(n):
    return n * U / (1 - n * U)


def _inputs(rows, cols, dt, gate, post, pre, seed=1):
    g = torch.Generator().manual_seed(seed)

    def r(*s, mean=0.0):
        return (torch.randn(*s, generator=g) + mean).to(dt)
    return dict(x=r(rows, cols), o=r(rows, cols),
                gate={"none": None, "channel": r(cols), "element": r(rows, cols)}[gate],
                w_post=r(cols, mean=1.0) if post else None,
                w_pre=r(cols, mean=1.0) if pre else None)


def _forward(x, o, gate, w_post, w_pre, alpha):
    """y, h, stats and their bounds.  A mean of n squares has relative error gamma(n + 2), its
    reciprocal root half of that and 2 u more; each further factor adds u, the residual sum u of
    the larger; a result u of its type."""
    x, o, gate, w_post, w_pre = (t.double() if t is not None else None
                                 for t in (x, o, gate, w_post, w_pre))
    cols = x.shape[1]
    er = _gamma(cols + 2) / 2 + 2 * U
    stats = torch.zeros(2, x.shape[0], dtype=torch.float64)
    n, en = o, 0.0
    if w_post is not None:
        stats[0] = (o.square().mean(1) + EPS).rsqrt()
        n, en = o * stats[0][:, None] * w_post, er + 2 * U
    if gate is not None:
        n, en = n * gate, en + U
    y = x + alpha * n
    ey = (en + 2 * U) * (alpha * n).abs() + U * y.abs()
    h = eh = None
    if w_pre is not None:
        stats[1] = (y.square().mean(1) + EPS).rsqrt()
        r = stats[1][:, None]
        # The root's relative error from y's: at most that of its norm.
        rel = ey.norm(dim=1, keepdim=True) / (y.norm(dim=1, keepdim=True) + 1e-300)
        h = y * r * w_pre
        eh = r * w_pre.abs() * ey + (er + rel + 2 * U) * h.abs()
    return y, h, stats, ey, eh, er


def _close(got, want, tol, dt, what):
    tol = tol + _unit(dt) * (want.abs() + tol)
    bad = ~((got.double().cpu() - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), bad.numel())


SETS = [("none", False, True), ("channel", True, True), ("element", True, True),
        ("element", False, False), ("none", True, False), ("channel", False, True)]
SIZES = [(1, 1), (1, 64), (5, 335), (3, 512), (300, 1030), (2, 2162), (17, 4096), (2, 8191),
         (1, 16384), (0, 64)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("gate,post,pre", SETS)
def test_forward(dev, dt, gate, post, pre):
    for rows, cols in SIZES:
        print(dt, gate, post, pre, rows, cols, flush=True)
        t = _inputs(rows, cols, dt, gate, post, pre)
        d = {k: v.to(dev) if v is not None else None for k, v in t.items()}
        y, h, stats = ops.block_norm(**d, alpha=0.7, eps=EPS)
        ry, rh, rs, ey, eh, er = _forward(**t, alpha=0.7)
        _close(y, ry, ey, dt, "y")
        assert (h is None) == (rh is None)
        if pre:
            _close(h, rh, eh, dt, "h")
        assert ((stats.double().cpu() - rs).abs() <= (er + 4 * U + (
            ey.norm(dim=1) / (ry.norm(dim=1) + 1e-300))) * rs).all()
        for out_y, out_h in ((d["x"], d["o"]),):  # in place, the same bits
            y2, h2, _ = ops.block_norm(**d, alpha=0.7, eps=EPS, out_y=out_y,
                                       out_h=out_h if pre else None)
            assert torch.equal(y2, y) and (h is None or torch.equal(h2, h))


def _backward(dy, dh, y, o, stats, gate, w_post, w_pre, alpha):
    """All gradients and bounds from the given y, o and stats.  gamma(cols + 8) of the absolute
    sums for a row's results, gamma(rows + 8) more for the sums over rows."""
    dy, dh, y, o, gate, w_post, w_pre, stats = (
        t.double() if t is not None else None
        for t in (dy, dh, y, o, gate, w_post, w_pre, stats))
    rows, cols = dy.shape
    e = _gamma(cols + 8)
    r_o, r_y = stats[0][:, None], stats[1][:, None]
    out, tol = {}, {}
    gx, ex = dy, U * dy.abs()
    if w_pre is not None:
        yn, g = y * r_y, dh * w_pre
        gx = dy + r_y * (g - yn * (g * yn).mean(1, keepdim=True))
        mag = dy.abs() + r_y * (g.abs() + yn.abs() * (g * yn).abs().mean(1, keepdim=True))
        ex = e * mag
        out["dw_pre"] = (dh * yn).sum(0)
        tol["dw_pre"] = _gamma(rows + 8) * (dh * yn).abs().sum(0)
    out["dx"], tol["dx"] = gx, ex
    on = o * r_o if w_post is not None else o
    n = on * w_post if w_post is not None else on
    if gate is not None:
        dg, eg = alpha * gx * n, alpha * n.abs() * (ex + 8 * U * gx.abs())
        channel = gate.dim() == 1
        out["dgate"] = dg.sum(0) if channel else dg
        tol["dgate"] = eg.sum(0) + _gamma(rows + 8) * dg.abs().sum(0) if channel else eg
    gt = gate if gate is not None else torch.ones(cols, dtype=torch.float64)
    db, eb = alpha * gx * gt, alpha * gt.abs() * (ex + 4 * U * gx.abs())
    if w_post is not None:
        out["dw_post"] = (db * on).sum(0)
        tol["dw_post"] = (eb * on.abs()).sum(0) + _gamma(rows + 8) * (db * on).abs().sum(0)
        g, eg = db * w_post, eb * w_post.abs()
        db = r_o * (g - on * (g * on).mean(1, keepdim=True))
        eb = r_o * (eg + on.abs() * (eg * on.abs()).mean(1, keepdim=True)) + e * r_o * (
            g.abs() + on.abs() * (g * on).abs().mean(1, keepdim=True))
    out["do"], tol["do"] = db, eb
    return out, tol


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("gate,post,pre", SETS)
def test_backward(dev, dt, gate, post, pre):
    for rows, cols in SIZES + [(3000, 96)]:
        print(dt, gate, post, pre, rows, cols, flush=True)
        t = _inputs(rows, cols, dt, gate, post, pre)
        x = t.pop("x")
        d = {k: v.to(dev) if v is not None else None for k, v in t.items()}
        y, _, stats = ops.block_norm(x.to(dev), **d, alpha=0.7)
        g = torch.Generator().manual_seed(9)
        dy, dh = (torch.randn(rows, cols, generator=g).to(dt) for _ in range(2))
        o = d.pop("o")
        got = dict(zip(("dx", "do", "dgate", "dw_post", "dw_pre"), ops.block_norm_backward(
            dy.to(dev), dh.to(dev) if pre else None, y, o, stats, **d, alpha=0.7)))
        t.pop("o")
        want, tol = _backward(dy, dh, y.cpu(), o.cpu(), stats.cpu(), **t, alpha=0.7)
        for k in ("dx", "do", "dgate", "dw_post", "dw_pre"):
            assert (got[k] is None) == (k not in want), k
            if k in want:
                _close(got[k], want[k], tol[k], dt, k)


def test_differences(dev):
    """All gradients along random directions against central differences of the float64 forward
    (third-derivative term eps^2 = 1e-10 of a smooth function, rounding 2^-52 / 1e-5)."""
    rows, cols, dt = 6, 200, torch.float32
    t = _inputs(rows, cols, dt, "channel", True, True, seed=3)
    d = {k: v.to(dev) for k, v in t.items()}
    y, h, stats = ops.block_norm(**d, alpha=0.7)
    g = torch.Generator().manual_seed(4)
    dy, dh = (torch.randn(rows, cols, generator=g) for _ in range(2))
    got = ops.block_norm_backward(dy.to(dev), dh.to(dev), y, d["o"], stats, d["gate"], d["w_post"],
                                  d["w_pre"], 0.7)
    for name, grad in zip(("x", "o", "gate", "w_post", "w_pre"), got):
        u = torch.randn(t[name].shape, generator=g, dtype=torch.float64)
        loss = []
        for s in (1e-5, -1e-5):
            w = {k: v.double() for k, v in t.items()}
            w[name] = w[name] + s * u
            a, b = _forward(**w, alpha=0.7)[:2]
            loss.append((a * dy + b * dh).sum().item())
        want = (loss[0] - loss[1]) / 2e-5
        terms = grad.double().cpu() * u
        # y in float32 instead of float64: U of it, through the norm's derivative; and the
        # gradient's own gamma(cols + rows) of its terms.
        assert abs(terms.sum().item() - want) <= 8 * _gamma(cols + rows) * terms.abs().sum() + 1e-6


def test_nonfinite_stays_in_its_row(dev):
    t = _inputs(3, 300, torch.float32, "channel", True, True)
    t["o"][1, 7] = math.nan
    d = {k: v.to(dev) for k, v in t.items()}
    y, h, _ = ops.block_norm(**d)
    assert y[[0, 2]].isfinite().all() and h[[0, 2]].isfinite().all()
    assert y[1].isnan().all() and h[1].isnan().all()


def test_same_bits_workspace_and_graph(dev):
    t = _inputs(700, 512, torch.bfloat16, "channel", True, True)
    d = {k: v.to(dev) for k, v in t.items()}
    y, h, stats = ops.block_norm(**d)
    args = (h, y, y, d["o"], stats, d["gate"], d["w_post"], d["w_pre"])
    a = ops.block_norm_backward(*args)
    ws = torch.empty(ops.block_norm_workspace_bytes(y), dtype=torch.uint8, device=dev)
    b = ops.block_norm_backward(*args, workspace=ws)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    with pytest.raises(_abi.KatsuError):
        ops.block_norm_backward(*args, workspace=ws[:-256])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c = ops.block_norm_backward(*args)
    for seed in (1, 2, 3):
        h.copy_(torch.randn(h.shape, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(c, ops.block_norm_backward(*args)))


def test_refusals(dev):
    x = torch.zeros(4, 32, device=dev)
    w = torch.ones(32, device=dev)
    for args, kw in (((x.double(), x.double()), {}), ((x, x.bfloat16()), {}), ((x, x[:2]), {}),
                     ((x.cpu(), x.cpu()), {}), ((x[0], x[0]), {}), ((x, x.t().t()[:, ::2]), {}),
                     ((x, x), dict(w_post=w[:3])), ((x, x), dict(gate=x[:2])),
                     ((x, x), dict(w_pre=w.bfloat16()))):
        with pytest.raises(ValueError):
            ops.block_norm(*args, **kw)
    wide = torch.zeros(1, 16385, device=dev)
    for args, kw in (((wide, wide), {}), ((x, x), dict(eps=-1.0)), ((x, x), dict(alpha=math.inf))):
        with pytest.raises(_abi.KatsuError) as e:
            ops.block_norm(*args, **kw)
        assert e.value.status == _abi.E_INVALID
    _, _, stats = ops.block_norm(x, x, w_pre=w)
    with pytest.raises(ValueError):
        ops.block_norm_backward(x, None, x, x, stats, w_pre=w)
    with pytest.raises(ValueError):
        ops.block_norm_backward(x, x, x, x, stats[:1], w_pre=w)
