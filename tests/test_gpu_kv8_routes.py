"""Attention that sees sinks or a tree, by each kernel that the host has a choice of: cases for kernels that a call's size
alone leads to (two short units a workgroup, a wave a unit), against the 64-bit restatement, with the kernel that ran
looked up; those captured and replayed over other lengths; and chains, whose words say what rows without words see."""
import numpy as np
import pytest

import np_draft
from sepia_amd import hip
from test_gpu_kv8 import B, OnGpu, attn, make, normal
from test_gpu_kv8_masked import close, masked, unseen_pages
from test_gpu_parity import Launches
from test_gpu_serve_run import Hip, on_gpu

pytestmark = pytest.mark.gpu
KERNELS = ["sepia_kv8_%s_%s_%s" % (sees, form, dim) for sees in ("sinks", "tree") for form in ("attn", "rows", "pair")
           for dim in ("128", "to128", "64", "to64")]
TOP = 2 ** 31 - 1


@pytest.fixture(scope="module")
def dev():
    return hip.Device()


NINE, SOME = [0, 5, 15, 16, 300, 63, 64, 33, 129], [20, 1, 7, 16, 17, 1, 3, 2, 5]
MANY = [k * 37 % 90 for k in range(17)]
TWENTY = [2, 1, 1, 3, 1, 1] + [1] * 11
# (kernel, query heads, kv heads, dim, page, lens, news, window, sinks, rel extent). A tile has 16 / (query heads / kv
# heads) tokens; 513 to 1023 units of up to 32 steps go two to a workgroup, more a wave each
CASES = [
    ("sinks_pair_128", 64, 64, 128, 16, [0, 5, 15, 16, 700, 63, 64, 333, 129], [1] * 9, 100, 4, 64),
    ("sinks_pair_128", 128, 16, 128, 64, [300, 0, 77], [30, 1, 39], 200, 70, 512),
    ("sinks_pair_to128", 99, 33, 80, 32, MANY, TWENTY, 20, 100, 30),    # an odd number of units
    ("sinks_pair_to128", 64, 64, 112, 16, NINE, SOME, 0, 3, 8),
    ("sinks_pair_64", 128, 8, 64, 16, [90, 0, 400], [25, 1, 44], 40, 33, 40),
    ("sinks_pair_64", 64, 64, 64, 32, [1900, 0, 1023, 1024, 64, 3, 127, 128, 9], [1] * 9, 1000, 500, 0),
    ("sinks_pair_to64", 64, 64, 48, 64, NINE, SOME, 33, 200, 50),
    ("sinks_pair_to64", 99, 33, 16, 16, MANY, TWENTY, 1, 1, 5),
    ("tree_pair_64", 64, 64, 64, 16, NINE, SOME, 60, 3, 64),
    ("tree_pair_64", 128, 32, 64, 32, [200, 0], [64, 6], 0, 0, 300),
    ("tree_pair_to64", 128, 8, 32, 64, [500, 0, 40], [40, 1, 29], 0, 0, 100),
    ("tree_pair_to64", 99, 33, 48, 16, MANY, TWENTY, 20, 2, 0),
    ("tree_rows_128", 64, 64, 128, 16, MANY, [1 + k % 4 for k in range(17)], 50, 5, 40),
    ("tree_rows_128", 128, 16, 128, 64, [130, 0, 64], [64, 2, 64], 0, 0, 64),
    ("tree_rows_128", 8, 4, 128, 64, [2100] + [3] * 259, [2] * 260, 0, 0, 5),   # long, of more than 256 sequences
    ("tree_rows_to128", 66, 66, 112, 32, MANY[:16], [1 + k % 5 for k in range(16)], 4, 70, 300),
    ("tree_rows_to128", 192, 64, 96, 16, MANY[:16], [2, 0, 3] * 5 + [6], 0, 0, 0),
    ("tree_rows_64", 64, 64, 64, 32, MANY, [64] + [1] * 16, 20, 33, 8),
    ("tree_rows_64", 128, 8, 64, 16, [70, 0, 5], [64, 63, 1], 0, 0, 33),
    ("sinks_rows_to64", 64, 64, 48, 16, MANY, [1 + k % 3 for k in range(17)], 20, 5, 30),
    # as many sinks as there may be: all is seen, and long units are cut
    ("sinks_attn_64", 64, 64, 64, 64, [2300, 0, 64, 9, 128, 3, 500, 31, 40], [1] * 9, 100, TOP, 64),
    ("sinks_attn_to128", 64, 64, 96, 16, [2300, 0, 64, 9, 128, 3, 500, 31, 40], [1] * 9, 100, 2 ** 40, 0),
    ("tree_attn_to64", 64, 64, 32, 16, [2300] + MANY[1:], [5] + [1] * 16, 100, TOP - 62, 20),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(a) if not isinstance(a, list) else "n%d" % len(a) for a in c))
def test_kernel(dev, case):
    kernel, H, heads, dim, page, lens, news, window, sinks, R = case
    rng = np.random.default_rng(H * 1000 + dim + sum(lens) + window)
    c, starts, n = make(rng, heads, dim, page, lens, news, rows_before=H % 2, rows_behind=H % 3)
    q = normal(rng, n, H, dim, scale=3.0)
    rel = normal(rng, n, H, R, scale=0.7) if R else None
    tau = rng.uniform(0.8, 1.4, n).astype(np.float32) if dim % 3 else None
    words = np_draft.trees(rng, starts, n, skew=[0.2, 1.3, 4.0][dim % 3]) if kernel.startswith("tree") else None
    if words is not None:   # a row that pads its tree
        words[starts[2] - 1] = 0
    want, tol = np_draft.attn(c, lens, starts, q, rel, tau, window, sinks, words, np.float32(1.0 / dim), fill=7.0)
    unseen_pages(c, lens, starts, window, sinks, rng)
    g = OnGpu(dev, c, off=16 * (H % 2))
    with Launches(dev) as ran:
        got = masked(dev, g, lens, starts, q, rel, tau, window, sinks, words, 1.0 / dim)
    assert [k for k in KERNELS if ran.count(k)] == ["sepia_kv8_" + kernel] and ran.count("sepia_kv8_" + kernel) == 1
    close(got, want, tol)
    g.free()


@pytest.mark.parametrize("n_seqs,form", [(9, "pair"), (17, "rows")])
def test_captured_follows_lengths(dev, n_seqs, form):
    """Both calls captured once and replayed over other lengths, rows, words and tables: right, and the bits of the same
    calls made eagerly."""
    L, h = dev.L, Hip(dev)
    rng = np.random.default_rng(n_seqs)
    H, dim, page, R, n, window, sinks, room = 64, 64, 32, 40, 60, 70, 9, 400
    pages = -(-(room + 64) // page)
    c, _, _ = make(rng, H, dim, page, [room] * n_seqs, [64] * n_seqs)
    c.table = np.ascontiguousarray(c.table[:, :pages])
    c.max_pages = pages
    bufs, d = on_gpu(h, c)
    q, rel = normal(rng, n, H, dim, scale=3.0), normal(rng, n, H, R)
    lb, sb, tb = [h.private(np.zeros(m, t)) for m, t in ((n_seqs, np.int32), (n_seqs + 1, np.int32), (n, np.uint64))]
    qb, rb = h.private(q), h.private(rel)
    ob = [h.private(np.zeros_like(q)) for _ in range(2)]
    ops = (lambda: L.sepia_hip_kv8_attn_sinks(B(d), lb, sb, n, qb, rb, None, ob[0], H, R, window, sinks, 1 / dim),
           lambda: L.sepia_hip_kv8_attn_tree(B(d), lb, sb, tb, n, qb, rb, None, ob[1], H, R, window, sinks, 1 / dim))
    with Launches(dev) as ran:
        for op in ops:
            dev.run(op)
    assert [k for k in KERNELS if ran.count(k)] == ["sepia_kv8_sinks_%s_64" % form, "sepia_kv8_tree_%s_64" % form]
    exe = h.capture(*ops)
    for step in range(4):
        lens = [int(v) for v in rng.integers(0, room, n_seqs)]
        news = rng.integers(0, 7, n_seqs)
        news[step % n_seqs] = 30
        while news.sum() > n:
            news[rng.integers(0, n_seqs)] = 0
        starts = [0] + [int(a) for a in np.cumsum(news)]
        words = np_draft.trees(rng, starts, n)
        c.table[:] = c.table[rng.permutation(n_seqs)]
        for b, a in ((lb, np.array(lens, np.int32)), (sb, np.array(starts, np.int32)), (tb, words), (bufs[2], c.table)):
            h.put(b, a)
        got = []
        for i in range(2):
            for b in ob:
                h.put(b, np.full_like(q, 5.0))
            if i == 0:
                h.replay(exe)
            else:
                dev.begin()
                assert [op() for op in ops] == [1, 1]
                dev.end()
            got.append([h.get(b, q.shape) for b in ob])
        for a, b, w in zip(got[0], got[1], (None, words)):
            assert np.array_equal(a.view(np.uint32), b.view(np.uint32)), step
            want, tol = np_draft.attn(c, lens, starts, q, rel, None, window, sinks, w, np.float32(1 / dim), fill=5.0)
            close(a, want, tol)
    h.R.hipGraphExecDestroy(exe)
    assert L.sepia_hip_take_device_error() == 0
    for b in bufs + [lb, sb, tb, qb, rb] + ob:
        dev.free(b)


@pytest.mark.parametrize("window", [0, 10, 25, 400])
def test_chain_has_the_bits_of_rows_without_words(dev, window):
    """Few units, none of them cut: the attention of a chain, of sinks and of neither walk the same columns in the same
    order (a chain's tiles may begin with more steps of which a row sees nothing, whose sums are 0)."""
    rng = np.random.default_rng(4)
    lens, news, H, heads, dim, R = [300, 17, 0], [64, 3, 20], 16, 4, 64, 50
    c, starts, n = make(rng, heads, dim, 32, lens, news)
    q, rel, tau = normal(rng, n, H, dim, scale=2.0), normal(rng, n, H, R), rng.uniform(0.8, 1.4, n).astype(np.float32)
    words = np.array([(1 << (i + 1)) - 1 for a in news for i in range(a)], np.uint64)
    g = OnGpu(dev, c)
    with Launches(dev) as ran:
        tree = masked(dev, g, lens, starts, q, rel, tau, window, 0, words, 1 / dim)
        rows = masked(dev, g, lens, starts, q, rel, tau, window, 0, None, 1 / dim)
        plain = attn(dev, g, lens, starts, q, rel, tau, window, 1 / dim)
    assert [ran.count("sepia_kv8_%sattn_64" % k) for k in ("tree_", "sinks_", "")] == [1, 1, 1]
    assert np.array_equal(tree.view(np.uint32), rows.view(np.uint32)) and np.array_equal(rows.view(np.uint32), plain.view(np.uint32))
    g.free()
