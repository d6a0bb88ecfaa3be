"""The embedding's gradient where it can be told exactly: gradients of small whole numbers, none of them
zero, whose sums float32 holds whatever their order.  A token that is left out, taken twice or given to
another row is off by one at least."""
import pytest
import torch

from katsu_amd import ops
from tests.test_gpu_embedding import TYPES, _ids


def _whole(rows, cols, gen):
    """-3..3 without 0."""
    x = torch.randint(1, 4, (rows, cols), generator=gen)
    return torch.where(torch.rand(rows, cols, generator=gen) < 0.5, -x, x)


def _sums(dout, ids, vocab):
    real = (ids >= 0) & (ids < vocab)
    return torch.zeros(vocab, dout.shape[1], dtype=torch.int64).index_add_(
        0, ids[real].long(), dout[real])


def _test(dev, dt, ids, vocab, cols, scale=0.5):
    g = torch.Generator().manual_seed(21)
    tokens = len(ids)
    assert 3 * (tokens + 1) * 4 < 1 << 24      # sums, in quarters
    dout, old = _whole(tokens, cols, g), _whole(vocab, cols, g)
    sums = _sums(dout, ids, vocab)
    d, i = dout.to(dt).to(dev), ids.to(dev)
    got = ops.embedding_backward(d, i, vocab, scale=scale).cpu()
    assert torch.equal(got, (sums * scale).to(dt))     # exact, then rounded once
    into = old.to(dt).to(dev)
    ops.embedding_backward(d, i, vocab, scale=scale, out=into, beta=1.0)
    assert torch.equal(into.cpu(), (sums * scale + old).to(dt))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("kind", ["mixed", "same", "spread"])
@pytest.mark.parametrize("tokens,vocab,cols", [
    (3, 2, 7), (64, 5, 40), (255, 70, 130), (256, 9, 33), (257, 9, 33), (1000, 5000, 64),
    (4097, 31, 1030), (16384, 3000, 72), (20000, 700, 2049), (32768, 1001, 40),
    (32769, 1001, 40), (65536, 40000, 36), (65537, 40000, 36), (9000, 100000, 9),
    (150000, 100000, 8), (300000, 1200000, 3), (530000, 700, 5), (1100000, 300, 3)])
def test_whole_numbers(dev, dt, kind, tokens, vocab, cols):
    print(dt, kind, tokens, vocab, cols, flush=True)
    _test(dev, dt, _ids(tokens, vocab, 6, kind), vocab, cols)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,vocab", [(200, 50), (3000, 800), (40000, 800), (200000, 30000)])
@pytest.mark.parametrize("run", [7, 8, 9, 31, 32, 33, 64, 127, 500])
def test_runs(dev, tokens, vocab, run):
    """Rows of `run` tokens each: runs of the sorted tokens that end before, at and behind a tile's end,
    some of them padding."""
    ids = (torch.arange(tokens) // run) % (vocab + 1)
    ids[::97] = -1
    ids = ids[torch.randperm(tokens, generator=torch.Generator().manual_seed(run))].int()
    _test(dev, torch.float32, ids, vocab, 20)


def test_one_token_is_seen():
    """What the comparison finds: any single token's loss changes every channel of its row."""
    g = torch.Generator().manual_seed(22)
    ids = _ids(5000, 40, 6)
    dout = _whole(5000, 4, g)
    sums = _sums(dout, ids, 40)
    for t in range(0, 5000, 83):
        less = ids.clone()
        less[t] = -1
        changed = (_sums(dout, less, 40) != sums).any(1)
        real = 0 <= int(ids[t]) < 40
        assert changed.sum() == (1 if real else 0)
