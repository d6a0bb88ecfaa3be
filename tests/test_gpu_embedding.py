"""Embedding and its gradient against their float64 definition: sizes, strides, padding, repeated
tokens, accumulation; the same bits in every call, in replayed graphs and on other streams."""
import pytest
import torch

from katsu_amd import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16]


def _half(dt):
    return torch.finfo(dt).eps / 2


def _gamma(n):
    return n * U / (1 - n * U)


def _ids(n, vocab, seed, kind="mixed"):
    """mixed: some tokens far more frequent than others, some no row of the table."""
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, vocab, (n,), generator=g)
    if kind == "same":
        return torch.full((n,), vocab // 2, dtype=torch.int32)
    if kind == "mixed" and n > 1:
        often = torch.rand(n, generator=g)
        ids[often < 0.3] = vocab // 3
        ids[often > 0.9] = torch.tensor([-1, vocab, -2 ** 31, 2 ** 31 - 1])[
            torch.randint(0, 4, (int((often > 0.9).sum()),), generator=g)]
    return ids.int()


def _grad(dout, ids, vocab, scale, old=None):
    """(dtable, bound): a float32 sum of n terms in any order, its product with the scale, the sum
    with what was there, and the rounding to the type."""
    real = (ids >= 0) & (ids < vocab)
    at = ids[real].long()
    d = dout.double()[real]
    want = torch.zeros(vocab, dout.shape[1], dtype=torch.float64).index_add_(0, at, d) * scale
    mag = torch.zeros_like(want).index_add_(0, at, d.abs()) * abs(scale)
    n = torch.zeros(vocab, dtype=torch.float64).index_add_(0, at, torch.ones(len(at)).double())
    tol = (n + 2)[:, None] * U * 1.01 * mag
    if old is not None:
        tol = tol + U * (mag + old.double().abs())
        want = want + old.double()
    return want, torch.where(n[:, None] > 0, tol + _half(dout.dtype) * (want.abs() + tol), 0.0)


def _check(got, want, tol):
    err = (got.double().cpu() - want).abs()
    assert (err <= tol).all(), (err - tol).max()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("tokens,vocab,cols", [(1, 1, 1), (1, 7, 3), (5, 3, 8), (64, 100, 33),
                                               (65, 1001, 256), (200, 50, 2047), (3, 9, 4099),
                                               (700, 257, 130)])
def test_lookup(dev, dt, tokens, vocab, cols):
    g = torch.Generator().manual_seed(1)
    table, ids = torch.randn(vocab, cols, generator=g).to(dt), _ids(tokens, vocab, 2)
    for scale in (1.0, -2.75):
        print(dt, tokens, vocab, cols, scale, flush=True)
        got = ops.embedding(ids.to(dev), table.to(dev), scale).cpu()
        real = (ids >= 0) & (ids < vocab)
        want = torch.zeros(tokens, cols, dtype=torch.float64)
        want[real] = table.double()[ids[real].long()] * scale
        assert got.dtype is dt
        _check(got, want, (_half(dt) + 2 * U if scale != 1.0 else 0.0) * want.abs())


@pytest.mark.parametrize("dt", TYPES)
def test_lookup_strides(dev, dt):
    """A table and an output that are parts of wider ones, at odd places; what lies beside stays."""
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(40, 77, generator=g).to(dt).to(dev)
    ids = _ids(90, 40, 4).to(dev)
    buf = torch.full((91, 59), 7.0, dtype=dt, device=dev)
    out = ops.embedding(ids, wide[:, 3:48], out=buf[:90, 5:50])
    real = (ids >= 0) & (ids < 40)
    want = torch.where(real[:, None], wide[ids.long().clamp(0, 39), 3:48], 0)
    assert torch.equal(out, want) and torch.equal(buf[:90, 5:50], want)
    assert (buf[:, :5] == 7).all() and (buf[:, 50:] == 7).all() and (buf[90] == 7).all()
    row = torch.randn(1, 45, generator=g).to(dt).to(dev).expand(40, 45)  # one row for all
    assert torch.equal(ops.embedding(ids, row), torch.where(real[:, None], row[:1], 0))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("kind", ["mixed", "same", "spread"])
@pytest.mark.parametrize("tokens,vocab,cols", [(1, 1, 1), (0, 5, 16), (2, 9, 3), (64, 3, 40),
                                               (129, 1001, 256), (255, 70, 1030),
                                               (1000, 5000, 64), (1500, 31, 100),
                                               (5000, 3000, 72), (20000, 700, 33),
                                               (9000, 100000, 8), (150000, 100000, 8),
                                               (6000, 3000000, 3), (530000, 700, 5)])
def test_gradient(dev, dt, kind, tokens, vocab, cols):
    print(dt, kind, tokens, vocab, cols, flush=True)
    g = torch.Generator().manual_seed(5)
    ids = _ids(tokens, vocab, 6, kind)
    dout = torch.randn(tokens, cols, generator=g).to(dt)
    got = ops.embedding_backward(dout.to(dev), ids.to(dev), vocab, scale=1.5)
    _check(got, *_grad(dout, ids, vocab, 1.5))
    old = torch.randn(vocab, cols, generator=g).to(dt)
    into = old.to(dev)
    back = ops.embedding_backward(dout.to(dev), ids.to(dev), vocab, scale=1.5, out=into, beta=1.0)
    assert back is into
    want, tol = _grad(dout, ids, vocab, 1.5, old)
    _check(into, want, tol)  # rows without a token: no error at all


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("tokens", [40, 3000, 9000])
def test_gradient_strides(dev, dt, tokens):
    """dout and the gradient as parts of wider tensors, at odd places."""
    g = torch.Generator().manual_seed(7)
    ids = _ids(tokens, 45, 8)
    dout = torch.randn(tokens, 91, generator=g).to(dt)
    buf = torch.full((46, 80), 3.0, dtype=dt, device=dev)
    ops.embedding_backward(dout.to(dev)[:, 1:72], ids.to(dev), 45, out=buf[:45, 7:78])
    _check(buf[:45, 7:78], *_grad(dout[:, 1:72], ids, 45, 1.0))
    assert (buf[:, :7] == 3).all() and (buf[:, 78:] == 3).all() and (buf[45] == 3).all()
    one = torch.randn(1, 71, generator=g).to(dt)  # one gradient for all tokens
    got = ops.embedding_backward(one.to(dev).expand(tokens, 71), ids.to(dev), 45)
    _check(got, *_grad(one.expand(tokens, 71), ids, 45, 1.0))


@pytest.mark.parametrize("tokens", [100, 2500, 12345])
def test_padding_holds_anything(dev, tokens):
    """What the gradient of padding holds changes nothing, nor do NaN in one row the others."""
    g = torch.Generator().manual_seed(9)
    ids = torch.randint(0, 300, (tokens,), generator=g).int()
    dout = torch.randn(tokens, 64, generator=g)
    pad = torch.rand(tokens, generator=g) < 0.2
    ids[pad] = -1
    clean = ops.embedding_backward(dout.to(dev), ids.to(dev), 300)
    dout[pad] = float("nan")
    at = int(torch.nonzero(~pad)[3])
    assert torch.equal(ops.embedding_backward(dout.to(dev), ids.to(dev), 300), clean)
    dout[at] = float("inf")
    got = ops.embedding_backward(dout.to(dev), ids.to(dev), 300)
    v = int(ids[at])
    assert not got[v].isfinite().any()
    keep = torch.arange(300) != v
    assert torch.equal(got[keep.to(dev)], clean[keep.to(dev)])


@pytest.mark.parametrize("tokens", [200, 3000, 30000, 530000])
def test_same_bits(dev, tokens):
    """Calls, replays of a graph with other tokens between, another stream, an own workspace."""
    g = torch.Generator().manual_seed(10)
    dout = torch.randn(tokens, 36, generator=g).to(dev)
    a, b = (_ids(tokens, 2000, s).to(dev) for s in (11, 12))
    want = [ops.embedding_backward(dout, i, 2000, 0.5) for i in (a, b)]
    ws = torch.empty(ops.embedding_workspace_bytes(tokens, 2000, 36, torch.float32),
                     dtype=torch.uint8, device=dev)
    ids = a.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(ops.embedding_backward(dout, a, 2000, 0.5, workspace=ws), want[0])
        side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.embedding_backward(dout, ids, 2000, 0.5)
        rows = ops.embedding(ids, got, 2.0)
    for i in (0, 1, 0, 1):
        ids.copy_((a, b)[i])
        got.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want[i])
        assert torch.equal(rows, ops.embedding((a, b)[i], want[i], 2.0))
        assert torch.equal(ops.embedding_backward(dout, a, 2000, 0.5), want[0])


def test_two_streams_at_once(dev):
    """Calls that overlap, each with memory of its own."""
    g = torch.Generator().manual_seed(13)
    dout = torch.randn(5000, 300, generator=g).to(dev)
    ids = [_ids(5000, 900, s).to(dev) for s in (14, 15)]
    want = [ops.embedding_backward(dout, i, 900) for i in ids]
    streams = [torch.cuda.Stream() for _ in ids]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for n, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[n].append(ops.embedding_backward(dout, ids[n], 900))
    torch.cuda.synchronize()
    assert all(torch.equal(t, want[n]) for n in (0, 1) for t in got[n])


def test_large_offsets(dev):
    """Rows of a table and of its gradient that lie beyond 2^32 bytes and 2^31 elements."""
    vocab, cols = 1_100_000, 2048
    table = torch.empty(vocab, cols, dtype=torch.bfloat16, device=dev)
    ids = torch.tensor([vocab - 1, 0, 1_048_577, vocab - 1], dtype=torch.int32, device=dev)
    x = torch.randn(4, cols, device=dev).bfloat16()
    table[ids.long()[1:]] = x[1:]
    assert torch.equal(ops.embedding(ids, table), x[[3, 1, 2, 3]])
    ops.embedding_backward(x, ids, vocab, out=table)
    want, tol = _grad(x.cpu()[:, :8], torch.tensor([2, 0, 1, 2], dtype=torch.int32), 3, 1.0)
    _check(table[torch.tensor([0, 1_048_577, vocab - 1], device=dev), :8], want, tol)
    assert not table[1:1_048_577].any() and not table[1_048_578:vocab - 1].any()
