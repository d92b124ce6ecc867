"""Device memory of another allocator under the serving calls (sepia_hip_wrap_device): the same bits as in the library's
own buffers, nothing behind the ranges touched, and no other call takes it."""
import ctypes

import numpy as np
import pytest

from sepia_amd import hip
from test_gpu_kv8 import B, make, normal
from test_gpu_serve_run import Hip

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return hip.Device()


class Pool:
    """One hipMalloc, cut up at multiples of 16 bytes with a guard between."""

    def __init__(self, h, nbytes):
        self.h, self.base, self.size, self.at = h, ctypes.c_void_p(), nbytes, 0
        assert h.R.hipMalloc(ctypes.byref(self.base), ctypes.c_size_t(nbytes)) == 0
        self.put(0, np.full(nbytes, 0xA5, np.uint8))
        self.used = np.zeros(nbytes, bool)

    def put(self, off, a):
        a = np.ascontiguousarray(a)
        assert self.h.R.hipMemcpy(ctypes.c_void_p(self.base.value + off), ctypes.c_void_p(a.ctypes.data), ctypes.c_size_t(a.nbytes), 1) == 0

    def get(self, off, shape, dtype):
        a = np.empty(shape, dtype)
        assert self.h.R.hipMemcpy(ctypes.c_void_p(a.ctypes.data), ctypes.c_void_p(self.base.value + off), ctypes.c_size_t(a.nbytes), 2) == 0
        return a

    def take(self, a):
        off, self.at = self.at, (self.at + a.nbytes + 16 + 15) // 16 * 16
        assert self.at <= self.size
        self.put(off, a)
        self.used[off:off + a.nbytes] = True
        return off, self.h.dev.wrap(self.base.value + off, a.nbytes)

    def free(self):
        assert self.h.R.hipFree(self.base) == 0


def test_same_bits(dev):
    L, h = dev.L, Hip(dev)
    rng = np.random.default_rng(8)
    H, heads, dim, page, R, vocab, rows = 8, 2, 80, 16, 20, 30001, 3
    lens, news = [100, 0, 33], [1, 40, 2]
    c, starts, n = make(rng, heads, dim, page, lens, news)
    kv = heads * dim
    first = [int(a // page * page) for a in lens]
    back = np.concatenate([[0], np.cumsum([a + b - f for a, b, f in zip(lens, news, first)])]).astype(np.int32)
    m = int(back[-1])
    arrays = dict(codes=c.codes, scales=c.scales, table=c.table, lens=np.array(lens, np.int32), starts=np.array(starts, np.int32),
                  k=normal(rng, n, kv, scale=3.0), v=normal(rng, n, kv, scale=3.0), norm=1 + normal(rng, dim, scale=0.1),
                  first=np.array(first, np.int32), back=back, kb=np.zeros((m, kv), np.float32), vb=np.zeros((m, kv), np.float32),
                  q=normal(rng, n, H, dim), rel=normal(rng, n, H, R), tau=rng.uniform(0.8, 1.2, n).astype(np.float32),
                  out=np.zeros((n, H, dim), np.float32), x=normal(rng, rows, vocab, scale=3.0), u=rng.random(rows).astype(np.float32),
                  p=np.full(rows, 0.9, np.float32), token=np.zeros(rows, np.int32), prob=np.zeros(rows, np.float32))
    pool = Pool(h, sum(a.nbytes + 48 for a in arrays.values()))
    offs, theirs = {}, {}
    for name, a in arrays.items():
        offs[name], theirs[name] = pool.take(a)
    ours = {name: h.private(a) for name, a in arrays.items()}

    def step(b):
        d = hip.Kv8Cache(n_pages=c.n_pages, max_pages=c.max_pages, n_seqs=3, n_kv_heads=heads, head_dim=dim, page=page,
                         codes=b["codes"], scales=b["scales"], table=b["table"])
        s = hip.SampleDesc(u=b["u"], top_p=b["p"])
        dev.begin()
        assert L.sepia_hip_kv8_append(B(d), b["lens"], b["starts"], n, b["k"], b["v"], b["norm"], 1e-6) == 1
        assert L.sepia_hip_kv8_read(B(d), b["first"], b["back"], m, b["kb"], b["vb"]) == 1
        assert L.sepia_hip_kv8_attn(B(d), b["lens"], b["starts"], n, b["q"], b["rel"], b["tau"], b["out"], H, R, 50, 1 / dim) == 1
        assert L.sepia_hip_sample(B(s), b["x"], rows, vocab, vocab, b["token"], b["prob"]) == 1
        dev.end()

    step(ours)
    step(theirs)
    changed = ("codes", "scales", "kb", "vb", "out", "token", "prob")
    for name, a in arrays.items():
        got = pool.get(offs[name], a.shape, a.dtype)
        want = h.get(ours[name], a.shape, a.dtype) if name in changed else a
        assert np.array_equal(got.view(np.uint8), want.view(np.uint8)), name
    assert np.all(pool.get(0, pool.size, np.uint8)[~pool.used] == 0xA5)
    for b in ours.values():
        dev.free(b)
    for b in theirs.values():
        assert L.sepia_gpu_host_ptr(b) is None
        dev.free(b)
    assert np.all(pool.get(0, pool.size, np.uint8)[~pool.used] == 0xA5)   # the memory is still the caller's
    pool.free()


def test_refusals(dev):
    L, h = dev.L, Hip(dev)
    pool = Pool(h, 1 << 12)
    wrap = lambda p, n: L.sepia_hip_wrap_device(ctypes.c_void_p(p), n)  # noqa: E731
    at = pool.base.value
    host = np.zeros(64, np.float32)
    for p, n in ((None, 16), (at, 0), (at + 4, 16), (at, (1 << 12) + 1), (at + 2048, 2049), (at, 2 ** 63), (at + 16, 2 ** 64 - 16),
                 ((host.ctypes.data + 15) // 16 * 16, 16), (16, 16)):
        assert wrap(p, n) is None, (p, n)
    b, whole = wrap(at + 16, 64), wrap(at, 1 << 12)
    assert b and whole and L.sepia_gpu_gpu_addr(b) == at + 16 and L.sepia_gpu_host_ptr(b) is None
    own = dev.alloc(256)
    dev.begin()
    for args in ((b, own, own), (own, b, own), (own, own, b)):
        assert L.sepia_gpu_add(*args, 16) == 0
    assert L.sepia_gpu_copy(b, 0, own, 0, 4) == 0 and L.sepia_gpu_matvec_q(8, b, 0, own, own, 1, 32) == 0
    assert L.sepia_hip_sample(B(hip.SampleDesc(u=b)), own, 1, 16, 16, whole, None) == 1
    assert L.sepia_hip_sample(B(hip.SampleDesc(u=b)), own, 17, 1, 1, whole, None) == 0   # u past its 64 bytes
    dev.end()
    assert L.sepia_gpu_selftest_touch(b, 4) == 0
    for x in (b, whole, own):
        dev.free(x)
    pool.free()
