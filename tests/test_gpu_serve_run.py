"""The serving operators together, as an engine uses them: prompts and then single tokens of several sequences
through append, attention, a projection and sampling in one batch each, the pages taken from one pool; the same
captured and replayed while lengths, rows and the table change; and their scratch under capture."""
import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest

from np_serve import Cache, sample
from sepia_amd import hip
from test_gpu_kv8 import B, OnGpu, append, attn, ints, make, normal

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def dev():
    return hip.Device()


def test_decode_loop(dev):
    """Two layers, three sequences: their prompts in one ragged call, then six steps of a token each; the attention's
    rows of the last layer are summed to logits that are sampled. The cache and the tokens equal the restatement's."""
    L = dev.L
    rng = np.random.default_rng(77)
    H, heads, dim, page, R, window, vocab = 8, 2, 64, 16, 24, 40, 501
    lens, news = [0, 0, 0], [37, 5, 16]
    c = [Cache(40, 3, 6, heads, dim, page, rng) for _ in range(2)]
    g = None
    norm = 1 + normal(rng, dim, scale=0.1)
    for step in range(7):
        starts = [0] + list(np.cumsum(news))
        n = starts[-1]
        for x in c:
            for s in range(3):
                x.reserve(s, lens[s] + news[s])
        if g is None:
            g = [OnGpu(dev, x) for x in c]
        for x, y in zip(c, g):
            dev.upload(y.bufs[2], x.table)
        k, v = normal(rng, 2, n, heads * dim), normal(rng, 2, n, heads * dim)
        q, rel = normal(rng, 2, n, H, dim, scale=2.0), normal(rng, 2, n, H, R)
        u = rng.random(n).astype(np.float32)
        lb, sb, nb, ub = ints(dev, lens), ints(dev, starts), dev.shared_from(norm), dev.shared_from(u)
        kb, vb, qb, rb = [[dev.shared_from(a) for a in x] for x in (k, v, q, rel)]
        ob = [dev.alloc(q[0].nbytes) for _ in range(2)]
        tb, pb = dev.alloc(4 * n), dev.alloc(4 * n)
        desc = hip.SampleDesc(u=ub)
        dev.begin()
        for i in range(2):
            assert L.sepia_hip_kv8_append(B(g[i].desc), lb, sb, n, kb[i], vb[i], nb, 1e-5) == 1
            assert L.sepia_hip_kv8_attn(B(g[i].desc), lb, sb, n, qb[i], rb[i], None, ob[i], H, R, window, 1 / dim) == 1
        # the last layer's rows are the logits (H * dim of them, vocab used)
        assert L.sepia_hip_sample(B(desc), ob[1], n, vocab, H * dim, tb, pb) == 1
        dev.end()
        token = dev.download(tb, n, np.int32)
        for i in range(2):
            c[i].append(lens, starts, k[i], v[i], norm, 1e-5)
            assert np.array_equal(g[i].codes(), c[i].codes) and np.array_equal(g[i].scales(), c[i].scales), (step, i)
            want, tol = c[i].attn(lens, starts, q[i], rel[i], None, window, np.float32(1 / dim))
            got = dev.download(ob[i], q[i].size).reshape(q[i].shape)
            assert np.all(np.abs(got - want) <= tol + np.abs(want) * 2.0 ** -23), (step, i)
        for r in range(n):
            want, _, near = sample(got[r].reshape(-1)[:vocab], u[r])
            assert near > vocab * 2.0 ** -44 and token[r] == want, (step, r)
        for b in [lb, sb, nb, ub, tb, pb] + kb + vb + qb + rb + ob:
            dev.free(b)
        lens, news = [a + b for a, b in zip(lens, news)], [1, 1, 1] if step % 2 else [1, 0, 2]
    for x in g:
        x.free()


@pytest.mark.parametrize("n_seqs,rows", [(5000, 5000), (5000, 3), (4097, 70)])
def test_many_sequences(dev, n_seqs, rows):
    """More sequences than two looks of 64 find, most of them without rows where rows are few."""
    rng = np.random.default_rng(n_seqs + rows)
    at = np.sort(rng.choice(n_seqs, rows, replace=False))
    news = np.zeros(n_seqs, int)
    news[at] = 1
    lens = np.where(news > 0, rng.integers(0, 40, n_seqs), 0)
    c, starts, n = make(rng, 1, 16, 16, list(lens), list(news))
    g = OnGpu(dev, c)
    k, v, q = normal(rng, n, 16), normal(rng, n, 16), normal(rng, n, 2, 16)
    append(dev, g, lens, starts, k, v)
    c.append(lens, starts, k, v)
    assert np.array_equal(g.codes(), c.codes) and np.array_equal(g.scales(), c.scales)
    got = attn(dev, g, lens, starts, q, None, None, 0, 1 / 16)
    want, tol = c.attn(lens, starts, q, None, None, 0, 1 / 16)
    assert np.all(np.abs(got - want) <= tol + np.abs(want) * 2.0 ** -23)
    g.free()


class Hip:
    """Captures and replays on the library's stream."""

    def __init__(self, dev):
        self.R, self.stream, self.dev = ctypes.CDLL("libamdhip64.so"), ctypes.c_void_p(dev.stream()), dev

    def capture(self, *ops):
        graph, exe = ctypes.c_void_p(), ctypes.c_void_p()
        self.dev.begin()
        assert self.R.hipStreamBeginCapture(self.stream, 1) == 0
        ok = [op() for op in ops]
        assert self.R.hipStreamEndCapture(self.stream, ctypes.byref(graph)) == 0
        self.dev.end()
        assert ok == [1] * len(ops)
        assert self.R.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, ctypes.c_size_t(0)) == 0
        return exe

    def replay(self, exe):
        assert self.R.hipGraphLaunch(exe, self.stream) == 0
        assert self.R.hipStreamSynchronize(self.stream) == 0

    def put(self, buf, a, off=0):
        a = np.ascontiguousarray(a)
        p = ctypes.c_void_p(self.dev.L.sepia_gpu_gpu_addr(buf) + off)
        assert self.R.hipMemcpy(p, ctypes.c_void_p(a.ctypes.data), ctypes.c_size_t(a.nbytes), 1) == 0

    def get(self, buf, shape, dtype=np.float32):
        a = np.empty(shape, dtype)
        p = ctypes.c_void_p(self.dev.L.sepia_gpu_gpu_addr(buf))
        assert self.R.hipMemcpy(ctypes.c_void_p(a.ctypes.data), p, ctypes.c_size_t(a.nbytes), 2) == 0
        return a

    def private(self, a):
        a = np.ascontiguousarray(a)
        b = self.dev.alloc(a.nbytes, private=True)
        self.put(b, a)
        return b


def on_gpu(h, c):
    bufs = [h.private(a) for a in (c.codes, c.scales, c.table)]
    return bufs, hip.Kv8Cache(n_pages=c.n_pages, max_pages=c.max_pages, n_seqs=c.n_seqs, n_kv_heads=c.heads,
                              head_dim=c.dim, page=c.page, codes=bufs[0], scales=bufs[1], table=bufs[2])


@pytest.mark.parametrize("H,heads,page,room", [(16, 2, 16, 700), (64, 64, 32, 90)])
def test_captured_step_follows_lengths(dev, H, heads, page, room):
    """A step captured once (append, attention, sampling) is replayed over growing lengths, other rows and new pages,
    with the same calls made eagerly in between, and with a second captured graph that uses the same scratch. The
    shapes take the kernel whose units are cut and the one with a wave a unit."""
    L, h = dev.L, Hip(dev)
    rng = np.random.default_rng(H + page)
    dim, n, vocab = 128, 40, 9000
    c = Cache(2 * n * (-(-room // page)), n, -(-room // page), heads, dim, page, rng)
    lens = rng.integers(0, room // 2, n)
    lens[0] = 0
    news = np.ones(n, int)
    for s in range(n):
        c.reserve(s, lens[s] + 1)
        c.table[s][c.table[s] < 0] = 0   # a captured graph may be handed any valid number there
    bufs, d = on_gpu(h, c)
    starts = np.arange(n + 1)
    lb, sb = h.private(lens.astype(np.int32)), h.private(starts.astype(np.int32))
    k, v, q, x, u = normal(rng, n, heads * dim), normal(rng, n, heads * dim), normal(rng, n, H, dim), normal(rng, 2, vocab, scale=3), rng.random(2).astype(np.float32)
    kb, vb, qb, xb, ub = [h.private(a) for a in (k, v, q, x, u)]
    ob, tb, ob2 = dev.alloc(q.nbytes, private=True), dev.alloc(8, private=True), dev.alloc(q.nbytes, private=True)
    desc = hip.SampleDesc(u=ub)

    def step(out=ob):
        return (lambda: L.sepia_hip_kv8_append(B(d), lb, sb, n, kb, vb, None, 0.0),
                lambda: L.sepia_hip_kv8_attn(B(d), lb, sb, n, qb, None, None, out, H, 0, 0, 1 / dim),
                lambda: L.sepia_hip_sample(B(desc), xb, 2, vocab, vocab, tb, None))

    assert L.sepia_hip_reserve_scratch(64 << 20) == 1
    exe = h.capture(*step())
    other = h.capture(step(ob2)[1])
    for i in range(4):
        for s in range(n):   # the tables grow; what was 0 behind a sequence's end becomes its page
            need = -(-(lens[s] + 1) // page)
            for j in range(need):
                if c.table[s, j] == 0 and j >= -(-(max(lens[s], 1)) // page):
                    c.table[s, j] = c.free.pop()
        k, v, q, x, u = normal(rng, n, heads * dim), normal(rng, n, heads * dim), normal(rng, n, H, dim), normal(rng, 2, vocab, scale=3), rng.random(2).astype(np.float32)
        for b, a in ((bufs[2], c.table), (lb, lens.astype(np.int32)), (kb, k), (vb, v), (qb, q), (xb, x), (ub, u)):
            h.put(b, a)
        h.replay(exe)
        got, token = h.get(ob, q.shape), h.get(tb, 2, np.int32)
        c.append(lens, starts, k, v)
        assert np.array_equal(h.get(bufs[0], c.codes.shape, np.int8), c.codes), i
        assert np.array_equal(h.get(bufs[1], c.scales.shape), c.scales), i
        want, tol = c.attn(lens, starts, q, None, None, 0, 1 / dim)
        assert np.all(np.abs(got - want) <= tol + np.abs(want) * 2.0 ** -23), i
        for r in range(2):
            t, _, near = sample(x[r], u[r])
            assert near > vocab * 2.0 ** -44 and token[r] == t, i
        h.replay(other)
        assert np.array_equal(h.get(ob2, q.shape).view(np.uint32), got.view(np.uint32)), i
        dev.begin()   # eagerly, the same calls: the same bits (the rows are appended over themselves)
        assert [op() for op in step(ob2)] == [1, 1, 1]
        dev.end()
        assert np.array_equal(h.get(ob2, q.shape).view(np.uint32), got.view(np.uint32)), i
        assert np.array_equal(h.get(bufs[0], c.codes.shape, np.int8), c.codes), i
        lens = lens + 1
    assert L.sepia_hip_take_device_error() == 0
    for e in (exe, other):
        h.R.hipGraphExecDestroy(e)
    for b in bufs + [lb, sb, kb, vb, qb, xb, ub, ob, tb, ob2]:
        dev.free(b)


def test_graphs_outlive_their_scratch(dev):
    """Captured attention whose units are cut and sampling in chunks, replayed after later calls have grown the scratch
    twice: the graph's region is still there, and its arrival counters. Bit for bit what the calls give eagerly."""
    L, h = dev.L, Hip(dev)
    rng = np.random.default_rng(14)
    heads, dim, page, H, rows, vocab = 2, 64, 32, 16, 4, 40007
    lens = [4000, 17, 900]
    c, starts, n = make(rng, heads, dim, page, lens, [1, 1, 1])
    c.table[c.table < 0] = 0
    bufs, d = on_gpu(h, c)
    q, x, u = normal(rng, n, H, dim), normal(rng, rows, vocab, scale=3.0), rng.random(rows).astype(np.float32)
    lb, sb, qb, xb, ub = [h.private(a) for a in (np.array(lens, np.int32), np.array(starts, np.int32), q, x, u)]
    ob, tb, pb = [dev.alloc(m, private=True) for m in (q.nbytes, 4 * rows, 4 * rows)]
    desc = hip.SampleDesc(u=ub)
    ops = (lambda: L.sepia_hip_kv8_attn(B(d), lb, sb, n, qb, None, None, ob, H, 0, 0, 1 / dim),
           lambda: L.sepia_hip_sample(B(desc), xb, rows, vocab, vocab, tb, pb))

    def results():
        return [h.get(ob, q.shape).view(np.uint32), h.get(tb, rows, np.int32), h.get(pb, rows).view(np.uint32)]

    def eager():
        dev.begin()
        assert [op() for op in ops] == [1, 1]
        dev.end()

    eager()
    first = results()
    want, tol = c.attn(lens, starts, q, None, None, 0, 1 / dim)
    assert np.all(np.abs(h.get(ob, q.shape) - want) <= tol + np.abs(want) * 2.0 ** -23)
    assert list(first[1]) == [sample(x[r], u[r])[0] for r in range(rows)]
    graphs = [h.capture(*ops)]
    for _ in range(2):
        size = L.sepia_hip_scratch_bytes()
        assert L.sepia_hip_reserve_scratch(size + 1) == 1 and L.sepia_hip_scratch_bytes() > size
        graphs.append(h.capture(*ops))
        for exe in graphs + graphs:
            for b, m in ((ob, q.size), (tb, rows), (pb, rows)):
                h.put(b, np.zeros(m, np.float32))
            h.replay(exe)
            assert all(np.array_equal(a, b) for a, b in zip(results(), first))
            eager()
            assert all(np.array_equal(a, b) for a, b in zip(results(), first))
    assert L.sepia_hip_take_device_error() == 0
    for e in graphs:
        h.R.hipGraphExecDestroy(e)
    for b in bufs + [lb, sb, qb, xb, ub, ob, tb, pb]:
        dev.free(b)


def test_call_after_falling_starts(dev):
    """Starts that fall give sequences more row tiles than the call has: an error, and the next calls are right (the runs
    of a unit that is cut count themselves, and all of them or none have to be there)."""
    L = dev.L
    rng = np.random.default_rng(41)
    H, heads, dim, page, lens = 32, 2, 64, 16, [2500, 2500, 2500, 2500, 2500]
    c, starts, n = make(rng, heads, dim, page, lens, [7, 1, 0, 1, 1])
    g = OnGpu(dev, c)
    q = normal(rng, n, H, dim)
    want, tol = c.attn(lens, starts, q, None, None, 0, 1 / dim)
    lb, qb, ob = ints(dev, lens), dev.shared_from(q), dev.alloc(q.nbytes)
    for bad in ([0, 7, 0, 7, 0, 7], [0, n, 0, n, 0, n], [3, n, 1, n, 0, n]):
        sb = ints(dev, bad)
        dev.begin()
        assert L.sepia_hip_kv8_attn(B(g.desc), lb, sb, n, qb, None, None, ob, H, 0, 0, 1 / dim) == 1
        assert L.sepia_gpu_end() == 0
        dev.free(sb)
        got = attn(dev, g, lens, starts, q, None, None, 0, 1 / dim)
        assert np.all(np.abs(got - want) <= tol + np.abs(want) * 2.0 ** -23), bad
    for b in (lb, qb, ob):
        dev.free(b)
    g.free()


def test_grid_past_the_launch_limit(dev):
    """65536 sequences of 300 kv heads: more workgroups than a launch can have; refused, not cut short."""
    L = dev.L
    n_seqs, heads = 65536, 300
    bufs = [dev.alloc(m) for m in (2 * heads * 16 * 16, 2 * heads * 4, 4 * n_seqs, 4 * n_seqs, 4 * n_seqs + 4, 4 * heads * 16 * 4)]
    d = hip.Kv8Cache(n_pages=1, max_pages=1, n_seqs=n_seqs, n_kv_heads=heads, head_dim=16, page=16, codes=bufs[0],
                     scales=bufs[1], table=bufs[2])
    dev.begin()
    for n in (1, 4):
        assert L.sepia_hip_kv8_attn(B(d), bufs[3], bufs[4], n, bufs[5], None, None, bufs[5], heads, 0, 0, 1.0) == 0
    dev.end()
    for b in bufs:
        dev.free(b)


CHILD = r"""
import sys
sys.path[:0] = [sys.argv[1], sys.argv[1] + "/tests"]
import numpy as np
from np_serve import Cache, sample
from sepia_amd import hip
from test_gpu_serve_run import B, Hip, normal, on_gpu
dev = hip.Device()
L, h = dev.L, Hip(dev)
rng = np.random.default_rng(6)
assert L.sepia_hip_reserve_scratch(1) == 1
size = L.sepia_hip_scratch_bytes()
c = Cache(400, 1, 400, 8, 128, 16, rng)
c.reserve(0, 6000)
bufs, d = on_gpu(h, c)
q, x, u = normal(rng, 1, 64, 128), normal(rng, 200, 40000, scale=3.0), rng.random(200).astype(np.float32)
lb, sb, qb, xb, ub = [h.private(a) for a in (np.array([5999], np.int32), np.array([0, 1], np.int32), q, x, u)]
ob, tb = dev.alloc(q.nbytes, private=True), dev.alloc(800, private=True)
desc = hip.SampleDesc(u=ub)
ops = (lambda: L.sepia_hip_kv8_attn(B(d), lb, sb, 1, qb, None, None, ob, 64, 0, 0, 1 / 128),
       lambda: L.sepia_hip_sample(B(desc), xb, 200, 40000, 40000, tb, None))
exe = h.capture(*ops)
assert L.sepia_hip_scratch_bytes() == size
want, tol = c.attn([5999], [0, 1], q, None, None, 0, 1 / 128)
tokens = [sample(x[r], u[r])[0] for r in range(200)]
for i in range(3):
    h.replay(exe)
    assert np.all(np.abs(h.get(ob, q.shape) - want) <= tol + np.abs(want) * 2.0 ** -23)
    assert list(h.get(tb, 200, np.int32)) == tokens
    h.put(ob, np.zeros_like(q))
dev.begin()
assert [op() for op in ops] == [1, 1]
dev.end()
assert L.sepia_hip_scratch_bytes() > size      # uncaptured they take what they want
assert np.all(np.abs(h.get(ob, q.shape) - want) <= tol + np.abs(want) * 2.0 ** -23)
assert list(h.get(tb, 200, np.int32)) == tokens
print("ok")
"""


def test_captured_with_little_scratch():
    """In a process of its own, whose scratch has its smallest size, 4 MiB: a captured call takes fewer runs (attention)
    or a workgroup a row (sampling) and the scratch does not grow."""
    r = subprocess.run([sys.executable, "-c", CHILD, ROOT], capture_output=True, text=True, cwd=ROOT, timeout=100)
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stdout + r.stderr


def test_bad_page_many_rows(dev):
    """The kernel with a wave a unit reports a page outside the pool too; the other sequences' rows are right."""
    rng = np.random.default_rng(12)
    c, starts, n = make(rng, 64, 16, 16, [20, 5, 40], [200, 3, 100])
    q = normal(rng, n, 64, 16)
    want, tol = c.attn([20, 5, 40], starts, q, None, None, 0, 1 / 16)
    held, c.table[1, 0] = c.table[1, 0], c.n_pages + 7
    g = OnGpu(dev, c)
    c.table[1, 0] = held
    lb, sb, qb, ob = ints(dev, [20, 5, 40]), ints(dev, starts), dev.shared_from(q), dev.alloc(q.nbytes)
    dev.begin()
    assert dev.L.sepia_hip_kv8_attn(B(g.desc), lb, sb, n, qb, None, None, ob, 64, 0, 0, 1 / 16) == 1
    assert dev.L.sepia_gpu_end() == 0 and dev.L.sepia_hip_take_device_error() == 0
    got = dev.download(ob, q.size).reshape(q.shape)
    for s in (0, 2):
        rows = slice(starts[s], starts[s + 1])
        assert np.all(np.abs(got[rows] - want[rows]) <= tol[rows] + np.abs(want[rows]) * 2.0 ** -23)
    for b in (lb, sb, qb, ob):
        dev.free(b)
    g.free()
