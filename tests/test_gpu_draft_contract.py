"""What a drafting engine has to know of the calls around drafted trees: where a request's list ends."""
import numpy as np
import pytest

from sepia_amd import hip
from test_gpu_draft import adjust
from test_gpu_kv8 import normal

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
