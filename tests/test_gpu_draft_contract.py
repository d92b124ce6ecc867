"""What a drafting engine has to know of the calls around drafted trees: where a request's list ends, what a draft that is
not accepted leaves behind in the pages of accepted tokens, and rows whose sequences' starts fall."""
import numpy as np
import pytest

import np_draft
from np_serve import Cache
from sepia_amd import hip
from test_gpu_draft import accept, adjust, keep
from test_gpu_kv8 import B, OnGpu, append, ints, normal
from test_gpu_kv8_masked import close, masked

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return hip.Device()


@pytest.mark.parametrize("vocab", [50, 20001])
def test_list_ends_before_row_0(dev, vocab):
    """Row 0's own token counts by its word: with a list that ends before it, each row of a chain has the bits that a
    call without a tree gives its whole list. A list that holds it too counts it twice."""
    rng = np.random.default_rng(vocab)
    old, drafted = [int(t) for t in rng.integers(0, 20, 30)], [7, 3, 7, 9]
    x = normal(rng, 4, vocab, scale=3.0)
    rates = dict(repetition=np.full(4, 1.3, np.float32), frequency=np.full(4, 0.3, np.float32), presence=np.full(4, 0.6, np.float32))
    words = np.array([(2 << i) - 1 for i in range(4)], np.uint64)
    got = adjust(dev, x, vocab, [0, 4], lists=[old], words=words, drafted=drafted, out_stride=vocab, **rates)
    whole = adjust(dev, x, vocab, lists=[old + drafted[:i + 1] for i in range(4)], out_stride=vocab, **rates)
    assert np.array_equal(got.view(np.uint32), whole.view(np.uint32))
    twice = adjust(dev, x, vocab, [0, 4], lists=[old + drafted[:1]], words=words, drafted=drafted, out_stride=vocab, **rates)
    counted = adjust(dev, x, vocab, lists=[old + drafted[:1] + drafted[:i + 1] for i in range(4)], out_stride=vocab, **rates)
    assert np.array_equal(twice.view(np.uint32), counted.view(np.uint32)) and np.all(twice[:, 7] < got[:, 7])


def read(dev, g, n_seqs, tokens):
    """Keys and values of each sequence's positions from 0 on."""
    starts = np.concatenate([[0], np.cumsum(tokens)])
    n, kv = int(starts[-1]), g.c.heads * g.c.dim
    bufs = [ints(dev, [0] * n_seqs), ints(dev, starts), dev.alloc(n * kv * 4), dev.alloc(n * kv * 4)]
    dev.run(dev.L.sepia_hip_kv8_read, B(g.desc), bufs[0], bufs[1], n, bufs[2], bufs[3])
    got = [dev.download(b, n * kv).reshape(n, g.c.heads, g.c.dim) for b in bufs[2:]]
    for b in bufs:
        dev.free(b)
    return [[x[starts[s]:starts[s + 1]] for x in got] for s in range(n_seqs)]


@pytest.mark.parametrize("value", [1000.0, np.nan])
@pytest.mark.parametrize("sampled", [[50, 0, 0, 0, 0], [11, 0, 0, 0, 0], [12, 0, 0, 0, 0]], ids=["none", "stays", "moves"])
def test_rejected_draft_stays_in_its_pages_scales(dev, value, sampled):
    """A draft of one large value, or of a NaN, that is not accepted: the tokens of its page (those that were there, and
    the accepted ones) keep that value's scale, also when rows move; other pages have nothing of it. A sequence whose
    tokens end with a page keeps all that it had as it was."""
    rng = np.random.default_rng(3)
    heads, dim, page, lens, news = 2, 32, 16, [20, 16], [5, 5]
    c = Cache(8, 2, 3, heads, dim, page, rng)
    for s in range(2):
        c.reserve(s, lens[s] + news[s])
    g = OnGpu(dev, c)
    k, v = normal(rng, 36, heads * dim), normal(rng, 36, heads * dim)
    append(dev, g, [0, 0], [0, 20, 36], k, v)
    c.append([0, 0], [0, 20, 36], k, v)
    before = read(dev, g, 2, lens)
    # rows 1 and 2 are row 0's children, row 3 row 1's, row 4 row 2's; row 3 has the value and is never accepted
    words = np.array([1, 3, 5, 11, 21] * 2, np.uint64)
    drafted, chosen = np.array([10, 11, 12, 13, 14] * 2), np.array(sampled * 2)
    k, v = normal(rng, 10, heads * dim), normal(rng, 10, heads * dim)
    for x in (k, v):
        x[[3, 8], 5] = value   # of the first head
    starts = [0, 5, 10]
    append(dev, g, lens, starts, k, v)
    c.append(lens, starts, k, v)
    (kept, counts, _), _ = accept(dev, words, starts, drafted, chosen, 2)
    assert list(counts) == ([1, 1] if sampled[0] == 50 else [2, 2]) and 3 not in kept
    codes, scales, known = np_draft.keep(c, lens, starts, kept)
    keep(dev, g, lens, starts, kept)
    got = g.scales()
    assert np.array_equal(np.isnan(got), np.isnan(scales)) and np.array_equal(got[~np.isnan(scales)], scales[~np.isnan(scales)])
    known &= ~np.isnan(scales)[..., None]
    assert np.array_equal(g.codes()[known], codes[known])
    after = read(dev, g, 2, [a + int(b) for a, b in zip(lens, counts)])
    step = np.float32(value) * np.float32(1 / 127)
    for s in range(2):
        hit = c.table[s, 1]   # the page of the drafts
        assert np.all(np.isnan(got[hit, :, 0])) if np.isnan(value) else np.all(got[hit, :, 0] == step)
        for was, now in zip(before[s], after[s]):
            assert np.array_equal(now[:16], was[:16])                       # the first page, and the second head's drafts
            assert np.all(np.abs(now[:, 1]) < 10)
            if np.isnan(value):
                assert np.isnan(now[16:, 0]).all()
            else:   # half a step of the page's scale, and the product's own rounding
                assert np.all(np.abs(now[16:lens[s], 0] - was[16:, 0]) <= step * np.float32(0.5001))
                assert not np.array_equal(now[16:lens[s], 0], was[16:, 0]) or lens[s] == 16
    # the next row sees the page as it is: NaN for the first head's queries
    c.codes[:], c.scales[:] = g.codes(), got
    lens = [a + int(b) for a, b in zip(lens, counts)]
    q = normal(rng, 2, 4, dim)
    want, tol = np_draft.attn(c, [a - 1 for a in lens], [0, 1, 2], q, scale=np.float32(1 / dim))
    assert np.isnan(want[:, :2]).all() == np.isnan(value) and np.isfinite(want[:, 2:]).all()
    close(masked(dev, g, [a - 1 for a in lens], [0, 1, 2], q, c=1 / dim), want, tol)
    g.free()


def test_logits_rows_where_starts_fall(dev):
    """Starts that fall: error 7, and each row is as it was or as a sequence that holds it has it."""
    rng = np.random.default_rng(5)
    vocab = 300
    x = normal(rng, 6, vocab)
    words, rates = np_draft.trees(rng, [0, 6], 6), np.full(6, 1.0, np.float32)
    for starts in ([0, 2, 1, 6], [3, 6, 0, 3], [0, 6, 5, 2], [2, 0, 6, 6]):
        got = adjust(dev, x, vocab, starts, lists=[[1], [2], [3]], words=words, drafted=[4] * 6, frequency=rates, ok=0)
        for r in range(6):
            right = [s for s in range(3) if starts[s] <= r < starts[s + 1] and not np.array_equal(got[r], x[r])]
            if not np.array_equal(got[r].view(np.uint32), x[r].view(np.uint32)):
                fits = []
                for s in right:
                    want, tol = np_draft.logits(x, starts[s:s + 2], vocab, lists=[[s + 1]], words=words, drafted=[4] * 6, frequency=rates)
                    fits.append(bool(np.all(np.abs(got[r] - want[r]) <= tol[r])))
                assert any(fits), (starts, r)
    assert dev.L.sepia_hip_take_device_error() == 0


def test_error_names_what_does_not_fit(dev, capfd):
    """A mask that is not there: the batch fails, and the log line does not speak of lengths and rows alone."""
    x = normal(np.random.default_rng(1), 2, 40)
    got = adjust(dev, x, 40, masks=np.zeros((1, 2), np.uint32), mask_row=[0, 1], ok=0)
    assert np.all(got[0] == -np.inf) and np.array_equal(got[1], x[1])
    assert "rows, a list, biases or a mask do not fit the call (device error 7)" in capfd.readouterr().err
    assert dev.L.sepia_hip_take_device_error() == 0
