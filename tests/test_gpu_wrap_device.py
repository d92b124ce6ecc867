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
    head = wrap(at, 16)
    assert L.sepia_hip_sample(B(hip.SampleDesc(u=b)), own, 1, 16, 16, head, None) == 1
    assert L.sepia_hip_sample(B(hip.SampleDesc(u=b)), own, 17, 1, 1, whole, None) == 0   # u past its 64 bytes
    dev.end()
    assert L.sepia_gpu_selftest_touch(b, 4) == 0
    for x in (b, whole, own, head):
        dev.free(x)
    pool.free()


def test_overlapping_handles(dev):
    """Two handles over the same memory are refused where one buffer is: what a call writes lies apart from what else it
    takes, by a byte's overlap; side by side, in one allocation or in one buffer, is taken."""
    L, h = dev.L, Hip(dev)
    pool = Pool(h, 1 << 20)
    pool.put(0, np.zeros(1 << 20, np.uint8))
    base, handles = pool.base.value, []

    def at(off, n):
        handles.append(dev.wrap(base + off, n))
        return handles[-1]

    heads, dim, page, n_pages, n, H, R, rows, vocab = 2, 16, 16, 4, 3, 4, 5, 4, 8
    size = dict(codes=n_pages * 2 * heads * page * dim, scales=n_pages * 2 * heads * 4, table=16, lens=4, starts=8, k=n * heads * dim * 4,
                v=n * heads * dim * 4, norm=dim * 4, q=n * H * dim * 4, out=n * H * dim * 4, rel=n * H * R * 4, tau=n * 4,
                logits=rows * vocab * 4, u=rows * 4, p=rows * 4, tokens=rows * 4, prob=rows * 4)
    off, place = {}, 0
    for name, b in size.items():
        off[name], place = place, place + (b + 15) // 16 * 16
    pool.put(off["starts"], np.array([0, n], np.int32))

    def calls(which, **moved):
        o = dict(off, **moved)
        b = {name: at(o[name], size[name]) for name in size}
        d = hip.Kv8Cache(n_pages=n_pages, max_pages=4, n_seqs=1, n_kv_heads=heads, head_dim=dim, page=page, codes=b["codes"],
                         scales=b["scales"], table=b["table"])
        s = hip.SampleDesc(u=b["u"], top_p=b["p"])
        return dict(append=lambda: L.sepia_hip_kv8_append(B(d), b["lens"], b["starts"], n, b["k"], b["v"], b["norm"], 1e-5),
                    read=lambda: L.sepia_hip_kv8_read(B(d), b["lens"], b["starts"], n, b["k"], b["v"]),
                    attn=lambda: L.sepia_hip_kv8_attn(B(d), b["lens"], b["starts"], n, b["q"], b["rel"], b["tau"], b["out"], H, R, 0, 1.0),
                    sample=lambda: L.sepia_hip_sample(B(s), b["logits"], rows, vocab, vocab, b["tokens"], b["prob"]))[which]()

    dev.begin()
    assert [calls(w) for w in ("append", "read", "attn", "sample")] == [1, 1, 1, 1]   # side by side
    assert calls("attn", q=off["out"]) == 1
    writes = dict(append=("codes", "scales"), read=("k", "v"), attn=("out",), sample=("tokens", "prob"))
    takes = dict(append=("codes", "scales", "table", "lens", "starts", "k", "v", "norm"), read=("codes", "scales", "table", "lens", "starts", "k", "v"),
                 attn=("codes", "scales", "table", "lens", "starts", "q", "rel", "tau"), sample=("logits", "u", "p", "tokens", "prob"))
    for which in writes:
        for w in writes[which]:
            for t in takes[which]:
                if t == w:
                    continue
                last = off[w] + (size[w] - 1) // 16 * 16   # the 16 bytes with w's last
                assert calls(which, **{t: last}) == 0, (which, w, t)
                if (which, t) != ("attn", "q"):
                    assert calls(which, **{t: off[w]}) == 0, (which, w, t)
    assert calls("attn", q=off["out"] + 16) == 0
    assert calls("append", k=off["v"]) == 1   # both are read
    dev.end()
    # in one buffer of the library's, at offsets
    own = dev.alloc(1 << 16)
    lens, starts, k = dev.shared_from(np.zeros(1, np.int32)), dev.shared_from(np.array([0, n], np.int32)), dev.alloc(size["k"])
    dev.begin()
    for scales_off, want in ((size["codes"], 1), (size["codes"] - 4, 0), (0, 0)):
        d = hip.Kv8Cache(n_pages=n_pages, max_pages=4, n_seqs=1, n_kv_heads=heads, head_dim=dim, page=page, codes=own, scales=own,
                         table=own, scales_off=scales_off, table_off=size["codes"] + size["scales"])
        assert L.sepia_hip_kv8_append(B(d), lens, starts, n, k, k, None, 0.0) == want
    dev.end()
    for x in handles + [own, lens, starts, k]:
        dev.free(x)
    pool.free()
