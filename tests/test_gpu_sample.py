"""Sampling against the 64-bit restatement (np_serve.sample): the same token, and its share of the kept weight, over
vocabularies from one token to 2^20, equal logits, empty rows, and every filter alone and together.

A decision may differ where a cumulative weight lies nearer to what it is compared with than the sums' own rounding:
2^-44 of the largest weight a token on this side, and less in numpy's. The tests' inputs are checked to be further
off than that (`near`), so tokens have to be equal; the share is rounded to f32 (2^-24) from sums within vocab * 2^-44
of a kept weight of at least 1, the largest."""
import ctypes

import numpy as np
import pytest

from np_serve import sample
from sepia_amd import hip

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return hip.Device()


def run(dev, x, vocab, u, temperature=None, top_p=None, min_p=None, top_k=None, prob=True):
    rows, stride = x.shape
    give = lambda a, t: None if a is None else dev.shared_from(np.broadcast_to(np.asarray(a, t), rows).copy())  # noqa: E731
    bufs = dict(u=give(u, np.float32), temperature=give(temperature, np.float32), top_p=give(top_p, np.float32),
                min_p=give(min_p, np.float32), top_k=give(top_k, np.int32))
    xb, tb, pb = dev.shared_from(x), dev.alloc(4 * rows), dev.alloc(4 * rows) if prob else None
    dev.run(dev.L.sepia_hip_sample, ctypes.byref(hip.SampleDesc(**bufs)), xb, rows, vocab, stride, tb, pb)
    got = dev.download(tb, rows, np.int32), dev.download(pb, rows) if prob else None
    for b in list(bufs.values()) + [xb, tb, pb]:
        if b:
            dev.free(b)
    return got


def check(dev, x, vocab, u, exact_ties=False, **params):
    rows = x.shape[0]
    token, prob = run(dev, x, vocab, u, **params)
    for r in range(rows):
        one = {k: (v if np.isscalar(v) else v[r]) for k, v in params.items()}
        want, share, near = sample(x[r, :vocab], u if np.isscalar(u) else u[r], **one)
        assert exact_ties or near > vocab * 2.0 ** -44, "the input decides within the sums' rounding"
        assert token[r] == want, (r, token[r], want, one)
        assert abs(prob[r] - share) <= share * (2.0 ** -23 + vocab * 2.0 ** -44), r


def logits(rng, rows, vocab, pad=0, spread=2.0):
    x = (rng.standard_normal((rows, vocab + pad)) * spread).astype(np.float32)
    for r in range(rows):
        x[r, rng.integers(0, vocab, min(50, vocab))] += rng.exponential(3.0, min(50, vocab)).astype(np.float32) + 2
    x[:, vocab:] = 1e9   # what lies in a row's padding is nobody's token
    return x


FILTERS = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=40), dict(top_p=0.9), dict(top_p=0.05), dict(min_p=0.05),
           dict(temperature=1.3, top_k=200, top_p=0.95, min_p=0.01), dict(temperature=0.0), dict(temperature=0.02, top_p=0.9),
           dict(temperature=30.0, top_p=0.8), dict(top_k=10 ** 9, top_p=1.0, min_p=0.0)]


@pytest.mark.parametrize("vocab,pad,rows", [(1, 0, 3), (2, 1, 5), (63, 0, 4), (64, 0, 4), (65, 3, 4), (1000, 0, 7), (4096, 0, 2),
                                            (8193, 5, 3), (50001, 0, 2), (100003, 61, 3), (1 << 20, 0, 1)], ids=str)
@pytest.mark.parametrize("params", FILTERS, ids=lambda p: ",".join("%s=%g" % i for i in p.items()) or "plain")
def test_filters(dev, vocab, pad, rows, params):
    rng = np.random.default_rng(vocab + len(params))
    check(dev, logits(rng, rows, vocab, pad), vocab, rng.random(rows).astype(np.float32), **params)


@pytest.mark.parametrize("rows,vocab", [(70, 3001), (300, 700), (2, 200003), (30, 30011), (600, 9001)])
def test_mixed_rows(dev, rows, vocab):
    """Each row with filters of its own."""
    rng = np.random.default_rng(rows)
    check(dev, logits(rng, rows, vocab, 4), vocab, rng.random(rows).astype(np.float32),
          temperature=rng.choice([0.0, 0.3, 1.0, 2.0], rows).astype(np.float32),
          top_p=rng.choice([0.3, 0.9, 1.0], rows).astype(np.float32), min_p=rng.choice([0.0, 0.02, 0.3], rows).astype(np.float32),
          top_k=rng.choice([0, 1, 5, 64, 1000], rows).astype(np.int32))


@pytest.mark.parametrize("vocab", [8, 1024, 65536, 100003, 1 << 20])
def test_equal_logits(dev, vocab):
    """All weights are 1: every sum is exact, and ties go to the lowest index."""
    x = np.full((6, vocab), 2.5, np.float32)
    x[5, ::2] = -0.0
    x[5, 1::2] = 0.0   # the two zeros are equal
    u = np.array([0.0, 0.25, 0.5, 1.0 - 2.0 ** -24, 0.75, 0.3], np.float32)
    for params in (dict(), dict(top_k=3), dict(top_p=0.5), dict(top_k=6, top_p=0.5, min_p=1.0), dict(temperature=0.0), dict(min_p=7.0)):
        check(dev, x, vocab, u, exact_ties=True, **params)


@pytest.mark.parametrize("vocab", [9000, 100003])
def test_far_below_the_largest(dev, vocab):
    """All tokens but one lie 14 to 60 octaves down, where bins are wider, then weigh nothing: borders on either side."""
    rng = np.random.default_rng(vocab)
    x = (-np.log(2.0) * np.where(rng.random((6, vocab)) < 500 / vocab, rng.uniform(14, 30, (6, vocab)),
                                 rng.uniform(30, 60, (6, vocab)))).astype(np.float32)
    x[:, vocab // 3] = 0.0
    u = np.array([0.2, 0.999, 0.99, 0.9999, 1.0 - 2.0 ** -14, 0.97], np.float32)
    for k in (0, 2, 300, vocab // 20, vocab // 2, vocab - 1):
        for params in (dict(), dict(top_p=1.0 - 2.0 ** -9), dict(top_p=0.995, min_p=2.0 ** -15)):
            check(dev, x, vocab, u, top_k=k, **params)


@pytest.mark.parametrize("spread", [0.3, 0.05, 0.02, 0.002])
@pytest.mark.parametrize("rows", [3, 40])
def test_flat_rows(dev, rows, spread):
    """Logits so close together that a bin holds hundreds, thousands or all of a row's tokens: more than a workgroup
    gathers, more than the row's list takes."""
    rng = np.random.default_rng(int(spread * 1000) + rows)
    vocab = 60000 if rows == 3 else 30000
    x = (rng.standard_normal((rows, vocab)) * spread).astype(np.float32)
    for params in (dict(), dict(top_p=0.97), dict(top_k=25000), dict(top_k=20000, top_p=0.4, min_p=0.9), dict(temperature=4.0, top_p=0.6)):
        check(dev, x, vocab, rng.random(rows).astype(np.float32), **params)


def test_few_distinct_logits(dev):
    """Long runs of equal logits below a few others: the border falls inside a run."""
    rng = np.random.default_rng(4)
    x = rng.choice(np.array([0.0, 1.0, 1.0 + 2.0 ** -23, -3.0], np.float32), (4, 30000))
    x[:, 17] = 6.0
    check(dev, x, 30000, rng.random(4).astype(np.float32), top_k=9000, top_p=0.7)
    check(dev, x, 30000, rng.random(4).astype(np.float32), top_p=0.99, temperature=0.5)


def test_empty_and_infinite_rows(dev):
    rng = np.random.default_rng(8)
    n = 5000
    x = logits(rng, 9, n)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, :] = -np.inf
    x[2, 77] = -3.0                                   # one token left
    x[3, rng.integers(0, n, 4000)] = -np.inf
    x[4, rng.integers(0, n, 4000)] = np.nan
    x[5, [9, 4000]] = np.inf                          # they have all the weight, half each
    x[6] = np.finfo(np.float32).min                   # the lowest value is a logit like another
    x[7] = np.finfo(np.float32).min
    x[7, 3] = 0.0
    x[8, 0] = np.finfo(np.float32).max
    u = np.array([0.3, 0.3, 0.9, 0.2, 0.6, 0.75, 0.5, 0.999, 0.9], np.float32)
    clean = np.where(np.isnan(x), -np.inf, x)
    for params in (dict(), dict(top_k=50, top_p=0.9, min_p=0.001), dict(temperature=0.0), dict(top_p=0.5, temperature=2.0)):
        token, prob = run(dev, x, n, u, **params)
        for r in range(9):
            want, share, _ = sample(clean[r], u[r], **params)
            assert token[r] == want and abs(prob[r] - share) <= share * (2.0 ** -23 + n * 2.0 ** -44), (r, params)
    assert list(token[:2]) == [-1, -1] and list(prob[:2]) == [0.0, 0.0]


def test_odd_parameters(dev):
    """u at and past its ends, NaN parameters, negative ones: off, greedy, or the nearest that is allowed."""
    x = logits(np.random.default_rng(2), 1, 3000)
    order = np.argsort(-x[0].astype(np.float64), kind="stable")
    assert run(dev, x, 3000, 0.0)[0][0] == order[0] and run(dev, x, 3000, -1.0)[0][0] == order[0]
    assert run(dev, x, 3000, np.nan)[0][0] == order[0]
    assert run(dev, x, 3000, 1.0, top_k=20)[0][0] == order[19] and run(dev, x, 3000, 5.0, top_k=20)[0][0] == order[19]
    assert run(dev, x, 3000, 0.9, temperature=np.nan)[0][0] == order[0] and run(dev, x, 3000, 0.9, temperature=-1.0)[0][0] == order[0]
    assert run(dev, x, 3000, 0.9, top_p=0.0)[0][0] == order[0] and run(dev, x, 3000, 0.9, top_p=-1.0)[0][0] == order[0]
    plain = run(dev, x, 3000, 0.9)[0][0]
    assert run(dev, x, 3000, 0.9, top_p=np.nan, min_p=np.nan, top_k=-7)[0][0] == plain
    assert run(dev, x, 3000, 0.9, prob=False)[0][0] == plain
    hot = run(dev, x, 3000, 0.5, temperature=np.inf)   # every weight 1
    assert hot[0][0] == order[1500] and abs(hot[1][0] - 1 / 3000) < 1e-9


def test_refusals(dev):
    L = dev.L
    x, t, p, f, small = dev.alloc(4 * 300), dev.alloc(4 * 3), dev.alloc(4 * 3), dev.alloc(4 * 3), dev.alloc(4)
    d = lambda **k: ctypes.byref(hip.SampleDesc(**dict(dict(u=f), **k)))  # noqa: E731
    assert L.sepia_hip_sample(d(), x, 3, 100, 100, t, p) == 0   # no batch is open
    dev.begin()
    assert L.sepia_hip_sample(d(), x, 3, 100, 100, t, p) == 1 and L.sepia_hip_sample(d(), x, 0, 100, 100, t, p) == 1
    assert L.sepia_hip_sample(d(temperature=f, top_p=f, min_p=f, top_k=f), x, 3, 98, 101, t, None) == 1
    for args in ((None, x, 3, 100, 100, t, p), (d(u=None), x, 3, 100, 100, t, p), (d(), None, 3, 100, 100, t, p),
                 (d(), x, 3, 100, 100, None, p), (d(), x, -1, 100, 100, t, p), (d(), x, 3, 0, 100, t, p), (d(), x, 3, 100, 99, t, p),
                 (d(), x, 3, 101, 101, t, p), (d(), x, 4, 10, 10, t, p), (d(), x, 3, (1 << 20) + 1, 1 << 21, t, p),
                 (d(), x, 2 ** 30, 100, 100, t, p), (d(), x, 3, 100, 2 ** 62, t, p), (d(), x, 3, 100, 100, small, p),
                 (d(), x, 3, 100, 100, t, small), (d(u=small), x, 3, 100, 100, t, p), (d(top_k=small), x, 3, 100, 100, t, p),
                 (d(), x, 3, 100, 100, t, t), (d(), x, 3, 100, 100, f, p), (d(top_p=p), x, 3, 100, 100, t, p), (d(), x, 1, 3, 3, x, p)):
        assert L.sepia_hip_sample(*args) == 0, args
    dev.end()
    for b in (x, t, p, f, small):
        dev.free(b)
