"""The serving operators at the edges of what a call may be handed."""
import ctypes
import subprocess
import sys

import numpy as np
import pytest

from sepia_amd import hip
from test_gpu_kv8 import B, OnGpu, append, attn, ints, make, normal
from test_gpu_sample import check, run
from test_gpu_serve_run import ROOT

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return hip.Device()


@pytest.mark.parametrize("heads,H", [(2, 4), (64, 64)], ids=["few", "many"])
def test_falling_starts(dev, heads, H):
    """Starts that fall, so that the search finds a sequence whose ids begin behind the one that is looked for: an error,
    and no page, row or output beside those of the sequences is touched. (As many units as take a wave each, too.)"""
    rng = np.random.default_rng(heads)
    dim, page, lens = 16, 16, [5, 5, 5]
    c, _, _ = make(rng, heads, dim, page, lens, [40, 40, 40], spare=6)
    n = 60
    q, k = normal(rng, n, H, dim), normal(rng, n, heads * dim)
    for starts in ([50, 60, 10, 20], [59, 60, 0, 1], [40, 41, 1, 2], [60, 0, 60, 0], [30, 60, 0, 30]):
        g = OnGpu(dev, c)
        before, scales = g.codes(), g.scales()
        out = np.full((n, H, dim), 7.0, np.float32)
        rows = np.full((n, heads * dim), 7.0, np.float32)
        bufs = [ints(dev, lens), ints(dev, starts), dev.shared_from(q), dev.shared_from(out), dev.shared_from(k),
                dev.shared_from(rows), dev.shared_from(rows)]
        for call in (lambda: dev.L.sepia_hip_kv8_attn(B(g.desc), bufs[0], bufs[1], n, bufs[2], None, None, bufs[3], H, 0, 0, 1 / dim),
                     lambda: dev.L.sepia_hip_kv8_read(B(g.desc), bufs[0], bufs[1], n, bufs[5], bufs[6]),
                     lambda: dev.L.sepia_hip_kv8_append(B(g.desc), bufs[0], bufs[1], n, bufs[4], bufs[4], None, 0.0)):
            dev.begin()
            assert call() == 1
            assert dev.L.sepia_gpu_end() == 0 and dev.L.sepia_hip_take_device_error() == 0
        fits = [(s, a, b) for s, (a, b) in enumerate(zip(starts, starts[1:])) if a <= b and lens[s] + b - a <= page * c.max_pages]
        inside = np.zeros(n, bool)
        for _, a, b in fits:
            inside[a:b] = True
        for b, a in ((bufs[3], out), (bufs[5], rows), (bufs[6], rows)):
            assert np.all(dev.download(b, a.size).reshape(a.shape)[~inside] == 7.0), starts
        mine = {c.table[s, p // page] for s, a, b in fits for p in range(lens[s], lens[s] + b - a)}
        rest = [p for p in range(c.n_pages) if p not in mine]
        assert np.array_equal(g.codes()[rest], before[rest]) and np.array_equal(g.scales()[rest], scales[rest]), starts
        for b in bufs:
            dev.free(b)
        g.free()


@pytest.mark.parametrize("vocab", [5000, 20000, 24575])
def test_few_below_a_long_run(dev, vocab):
    """A row of one workgroup, all but ten of whose logits are equal, more than a workgroup gathers, and whose k-th token
    is among the ten in a bin below: they are decided at once, without a search by pieces before."""
    rng = np.random.default_rng(vocab)
    x = np.full((64, vocab), 2.0, np.float32)
    for r in range(64):
        x[r, rng.choice(vocab, 10, replace=False)] = 1.0 - 0.0005 * np.arange(10, dtype=np.float32)
    # within the run, and at its end: one to ten tokens of weight 0.37 behind vocab - 10 of weight 1
    u = np.where(np.arange(64) % 2, 1.0 - 10.0 ** -rng.uniform(3.5, 5.5, 64), rng.random(64)).astype(np.float32)
    for below in (1, 5, 9):
        check(dev, x, vocab, u, top_k=vocab - 10 + below)
        check(dev, x, vocab, u, top_k=vocab - 10 + below, temperature=1.5, top_p=0.9999)


def test_few_gathered_of_chunks(dev):
    """Rows in chunks whose decisions are among a handful of gathered tokens, three decisions in a row."""
    rng = np.random.default_rng(5)
    vocab, rows = 30000, 24
    x = (rng.standard_normal((rows, vocab)) - 40).astype(np.float32)
    for r in range(rows):
        x[r, rng.choice(vocab, 12, replace=False)] = np.linspace(3, 0, 12).astype(np.float32)
    u = rng.random(rows).astype(np.float32)
    for params in (dict(), dict(top_k=7), dict(top_k=9, top_p=0.8), dict(top_k=10, top_p=0.95, min_p=0.2)):
        check(dev, x, vocab, u, **params)


@pytest.mark.parametrize("dim,page", [(64, 16), (16, 64), (128, 32)])
def test_append_behind_a_scale_of_zero(dev, dim, page):
    """Codes whose scale is 0 stand for 0, and still do when a page's scale grows: they are rounded anew to 0. A scale that
    stays 0 leaves them."""
    rng = np.random.default_rng(dim)
    heads, lens, news = 3, [page - 5, page + 7, 3], [2, page, 1]
    c, starts, n = make(rng, heads, dim, page, lens, news)
    firsts = [c.table[s, lens[s] // page] for s in range(3)]
    for p in firsts:
        c.scales[p, 0, :2] = 0.0   # K of heads 0 and 1, V of heads 1 and 2
        c.scales[p, 1, 1:] = 0.0
    k, v = normal(rng, n, heads * dim), normal(rng, n, heads * dim)
    k[:, dim:2 * dim] = 0.0        # head 1: nothing but zeros comes, the scale stays 0
    v[:, dim:2 * dim] = 0.0
    g = OnGpu(dev, c)
    append(dev, g, lens, starts, k, v)
    codes, scales = g.codes(), g.scales()
    c.append(lens, starts, k, v)   # its scales and new codes; of the old ones below
    assert np.array_equal(scales, c.scales)
    for s, p in enumerate(firsts):
        at = lens[s] % page
        for side, zero in ((0, 0), (1, 2)):
            assert scales[p, side, zero] > 0
            c.views(p)[side][:at, zero] = 0
        assert scales[p, 0, 1] == 0 and scales[p, 1, 1] == 0
    assert np.array_equal(codes, c.codes)
    # what the pages stand for: the old positions of those heads are 0
    rows = int(sum(lens))
    back = np.concatenate([[0], np.cumsum(lens)])
    bufs = [ints(dev, [0, 0, 0]), ints(dev, back), dev.alloc(rows * heads * dim * 4), dev.alloc(rows * heads * dim * 4)]
    dev.run(dev.L.sepia_hip_kv8_read, B(g.desc), bufs[0], bufs[1], rows, bufs[2], bufs[3])
    for side, zero in ((0, 0), (1, 2), (0, 1), (1, 1)):
        got = dev.download(bufs[2 + side], rows * heads * dim).reshape(rows, heads, dim)
        for s in range(3):
            old = got[back[s]:back[s + 1]]
            assert np.all(old[lens[s] // page * page:, zero] == 0.0)
    for b in bufs:
        dev.free(b)
    g.free()


GROWTH = r"""
import sys
sys.path[:0] = [sys.argv[1], sys.argv[1] + "/tests"]
import numpy as np
from np_serve import sample
from sepia_amd import hip
from test_gpu_serve_run import B, Hip, normal
dev = hip.Device()
L, h = dev.L, Hip(dev)
rng = np.random.default_rng(2)
rows, vocab = 3, 30000
x, u = normal(rng, rows, vocab, scale=3.0), rng.random(rows).astype(np.float32)
xb, ub, tb = h.private(x), h.private(u), dev.alloc(4 * rows, private=True)
desc = hip.SampleDesc(u=ub)
op = lambda: L.sepia_hip_sample(B(desc), xb, rows, vocab, vocab, tb, None)
tokens = [sample(x[r], u[r])[0] for r in range(rows)]
graphs, sizes = [], set()
for i in range(90):   # the engine's way: a call of the next size, once, then its capture
    assert L.sepia_hip_reserve_scratch((4 << 20) + (i << 18)) == 1, i
    sizes.add(L.sepia_hip_scratch_bytes())
    graphs.append(h.capture(op))
    if i % 9 == 0:
        for exe in graphs[::5] + graphs[-1:]:
            h.put(tb, np.full(rows, -7, np.int32))
            h.replay(exe)
            assert list(h.get(tb, rows, np.int32)) == tokens, i
assert L.sepia_hip_reserve_scratch(200 << 20) == 1
assert len(sizes) < 12 and max(sizes) < 2 * ((4 << 20) + (90 << 18)) + (1 << 20), sorted(sizes)
dev.begin()
assert op() == 1
dev.end()
assert list(h.get(tb, rows, np.int32)) == tokens
print("ok")
"""


def test_scratch_grows_among_many_captures():
    """In a process of its own: 90 calls, each of a little more scratch and captured once it ran. The regions that graphs
    hold are few, since each is at least twice the one before, and none of the calls is refused."""
    r = subprocess.run([sys.executable, "-c", GROWTH, ROOT], capture_output=True, text=True, cwd=ROOT, timeout=100)
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stdout + r.stderr


@pytest.mark.parametrize("rows,vocab", [(6, 3000), (3, 60000)], ids=["whole", "chunks"])
def test_infinite_temperature_and_logits(dev, rows, vocab):
    """A +inf logit leaves all others without weight at every temperature, an infinite one too."""
    rng = np.random.default_rng(vocab)
    for count in (1, 2, 40, 300):
        x = normal(rng, rows, vocab)
        at = [np.sort(rng.choice(vocab, count, replace=False)) for _ in range(rows)]
        for r in range(rows):
            x[r, at[r]] = np.inf
        u = rng.random(rows).astype(np.float32)
        for t in (np.inf, 3e38, 1.0, 1e-45):
            for more in (dict(), dict(top_k=vocab - 1), dict(top_p=0.75), dict(min_p=0.5)):
                token, prob = run(dev, x, vocab, u, temperature=t, **more)
                kept = max(1, int(np.ceil(0.75 * count))) if "top_p" in more else count
                for r in range(rows):
                    assert token[r] == at[r][min(int(np.float64(u[r]) * kept), kept - 1)], (count, t, more, r)
                    assert abs(prob[r] - 1 / kept) <= 2.0 ** -24 / kept * 2


def test_slots_without_rows(dev):
    """A cache of 4096 slots of which three have rows: right, and about as long as one of three slots (they are looked
    through; they were counted in the launch's grid, 2.6 ms in all)."""
    rng = np.random.default_rng(12)
    n_seqs, H, heads, dim, page = 4096, 16, 8, 64, 16
    at, lens, news = [0, 1700, 4095], np.zeros(n_seqs, int), np.zeros(n_seqs, int)
    lens[at], news[at] = [1500, 3, 900], [1, 2, 1]
    c, starts, n = make(rng, heads, dim, page, list(lens), list(news))
    q = normal(rng, n, H, dim)
    g = OnGpu(dev, c)
    got = attn(dev, g, lens, starts, q, None, None, 0, 1 / dim)
    want, tol = c.attn(lens, starts, q, None, None, 0, 1 / dim)
    assert np.all(np.abs(got - want) <= tol + np.abs(want) * 2.0 ** -23)
    count, ms, times = ctypes.c_int64(), ctypes.c_double(), []
    for _ in range(6):
        dev.L.sepia_hip_profile_reset()
        assert dev.L.sepia_hip_profile_start() == 1
        attn(dev, g, lens, starts, q, None, None, 0, 1 / dim)
        assert dev.L.sepia_hip_profile_stop() == 1
        assert dev.L.sepia_hip_profile_query(b"sepia_kv8_attn_64", ctypes.byref(count), ctypes.byref(ms)) == 1 and count.value == 1
        times.append(ms.value)
    assert min(times) < 0.6, times
    g.free()
