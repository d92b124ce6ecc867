"""The paged 8-bit key/value cache against the 64-bit restatement (np_serve.py): appended codes and scales bit for
bit, rows read back, and attention over the cache, at the sizes, masks and values where they can go wrong."""
import ctypes

import numpy as np
import pytest

from np_serve import Cache
from sepia_amd import hip

pytestmark = pytest.mark.gpu
B = ctypes.byref


@pytest.fixture(scope="module")
def dev():
    return hip.Device()


class OnGpu:
    """A Cache's arrays in the library's shared buffers."""

    def __init__(self, dev, c, off=0):
        self.dev, self.c, self.off = dev, c, off
        pad = np.zeros(off, np.uint8)
        self.bufs = [dev.shared_from(np.concatenate([pad, np.ascontiguousarray(a).view(np.uint8).reshape(-1)]))
                     for a in (c.codes, c.scales, c.table)]
        self.desc = hip.Kv8Cache(n_pages=c.n_pages, max_pages=c.max_pages, n_seqs=c.n_seqs, n_kv_heads=c.heads,
                                 head_dim=c.dim, page=c.page, codes=self.bufs[0], scales=self.bufs[1],
                                 table=self.bufs[2], codes_off=off, scales_off=off, table_off=off)

    def codes(self):
        return self.dev.download(self.bufs[0], self.c.codes.size, np.int8, self.off).reshape(self.c.codes.shape)

    def scales(self):
        return self.dev.download(self.bufs[1], self.c.scales.size, np.float32, self.off).reshape(self.c.scales.shape)

    def free(self):
        for b in self.bufs:
            self.dev.free(b)


def ints(dev, a):
    return dev.shared_from(np.asarray(a, np.int32))


def append(dev, g, lens, starts, k, v, norm=None, eps=0.0):
    bufs = [ints(dev, lens), ints(dev, starts), dev.shared_from(k), dev.shared_from(v)]
    nb = None if norm is None else dev.shared_from(norm)
    dev.run(dev.L.sepia_hip_kv8_append, B(g.desc), bufs[0], bufs[1], len(k), bufs[2], bufs[3], nb, eps)
    for b in bufs + ([nb] if nb else []):
        dev.free(b)


def attn(dev, g, lens, starts, q, rel=None, tau=None, window=0, c=1.0, fill=7.0):
    out = np.full(q.shape, fill, np.float32)
    bufs = [ints(dev, lens), ints(dev, starts), dev.shared_from(q), dev.shared_from(out)]
    more = [None if a is None else dev.shared_from(a) for a in (rel, tau)]
    dev.run(dev.L.sepia_hip_kv8_attn, B(g.desc), bufs[0], bufs[1], len(q), bufs[2], more[0], more[1], bufs[3],
            q.shape[1], 0 if rel is None else rel.shape[2], window, c)
    got = dev.download(bufs[3], q.size).reshape(q.shape)
    for b in bufs + [m for m in more if m]:
        dev.free(b)
    return got


def make(rng, heads, dim, page, lens, news, spare=3, rows_before=0, rows_behind=0):
    """A cache whose pages hold random codes for `lens` tokens a sequence and have room for `news` more."""
    n = len(lens)
    most = max(1, max(-(-(a + b) // page) for a, b in zip(lens, news)))
    need = sum(-(-(a + b) // page) for a, b in zip(lens, news))
    c = Cache(need + spare, n, most + 1, heads, dim, page, rng)
    for s in range(n):
        c.reserve(s, lens[s] + news[s])
    starts = rows_before + np.concatenate([[0], np.cumsum(news)])
    return c, [int(a) for a in starts], int(starts[-1]) + rows_behind


def normal(rng, *shape, scale=1.0):
    return (rng.standard_normal(shape) * scale).astype(np.float32)


# (kv heads, dim, page, lens, news): one token into an empty page, at its last slot, past it; prompts from nothing
# and from inside a page; pages touched whole, in part, one after the other; sequences without rows; narrow dims
APPENDS = [
    (1, 16, 16, [0], [1]), (8, 128, 16, [20000], [1]), (2, 64, 32, [31], [1]), (2, 64, 32, [32], [1]), (3, 80, 16, [5], [11]),
    (3, 80, 16, [5], [12]), (1, 128, 64, [63], [66]), (4, 48, 64, [0, 0, 7], [0, 130, 0]), (2, 128, 16, [0, 16, 3], [16, 16, 45]),
    (16, 128, 32, [100, 0, 31, 64, 1], [1, 1, 1, 1, 1]), (1, 112, 64, [15, 47, 48], [1, 1, 20]), (5, 32, 16, [0] * 70, [2] * 70),
    (2, 96, 32, [9], [700]), (1, 16, 64, list(range(0, 130)), [k % 3 for k in range(130)]),
]


@pytest.mark.parametrize("norm", [False, True], ids=["plain", "norm"])
@pytest.mark.parametrize("case", APPENDS, ids=lambda c: "-".join(str(a) if not isinstance(a, list) else "n%d" % len(a) for a in c))
def test_append(dev, case, norm):
    heads, dim, page, lens, news = case
    rng = np.random.default_rng(dim * 100 + len(lens))
    c, starts, n = make(rng, heads, dim, page, lens, news, rows_before=len(lens) % 3, rows_behind=dim % 5)
    g = OnGpu(dev, c, off=16 * (dim % 3))
    kv = heads * dim
    # magnitudes over some powers of two, so that scales grow in some pages and stay in others
    k, v = [normal(rng, n, kv) * np.exp2(rng.integers(-4, 3, (n, 1))).astype(np.float32) for _ in range(2)]
    w = 1 + normal(rng, dim, scale=0.2) if norm else None
    append(dev, g, lens, starts, k, v, w, 1e-6)
    c.append(lens, starts, k, v, w, 1e-6)
    assert np.array_equal(g.scales().view(np.uint32), c.scales.view(np.uint32))
    assert np.array_equal(g.codes(), c.codes)
    # the pages read back, every position
    back = np.concatenate([[0], np.cumsum([a + b for a, b in zip(lens, news)])])
    rows = int(back[-1])
    bufs = [ints(dev, [0] * len(lens)), ints(dev, back), dev.alloc(rows * kv * 4 + 4), dev.alloc(rows * kv * 4 + 4)]
    dev.run(dev.L.sepia_hip_kv8_read, B(g.desc), bufs[0], bufs[1], rows, bufs[2], bufs[3])
    for side, b in enumerate(bufs[2:]):
        got = dev.download(b, rows * kv).reshape(rows, heads, dim)
        for s, (a, e) in enumerate(zip(back, back[1:])):
            if e > a:
                want = c.rows(s, 0, int(e - a))[side].astype(np.float32)
                assert np.array_equal(got[a:e], want), (side, s)
    for b in bufs:
        dev.free(b)
    g.free()


def test_append_token_by_token(dev):
    """A page filled one token at a time: scales only grow, old codes are rounded anew each time they do, and a page
    that is used again starts afresh whatever it held."""
    rng = np.random.default_rng(5)
    c, _, _ = make(rng, 2, 64, 16, [0, 0], [40, 33])
    g = OnGpu(dev, c)
    lens = [0, 0]
    for i in range(33):
        k, v = normal(rng, 2, 128, scale=1.0 + 0.1 * i), normal(rng, 2, 128, scale=2.0 ** (i % 7 - 3))
        append(dev, g, lens, [0, 1, 2], k, v, np.ones(64, np.float32), 1e-5)
        c.append(lens, [0, 1, 2], k, v, np.ones(64, np.float32), 1e-5)
        lens = [a + 1 for a in lens]
        assert np.array_equal(g.codes(), c.codes) and np.array_equal(g.scales(), c.scales), i
    g.free()


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_append_nonfinite_and_zero(dev, bad):
    """A value that is not finite makes its page's scale of its head NaN (K or V alone), also for tokens appended
    later; rows of zeros and of denormals give finite codes."""
    rng = np.random.default_rng(9)
    c, starts, n = make(rng, 3, 32, 16, [2, 0, 16], [20, 18, 3])
    g = OnGpu(dev, c)
    k, v = normal(rng, n, 96), normal(rng, n, 96)
    k[1, 40], v[25, 3], k[38:41], v[38:41] = bad, bad, 0.0, np.float32(1e-42)
    append(dev, g, [2, 0, 16], starts, k, v)
    c.append([2, 0, 16], starts, k, v)
    s = g.scales()
    assert np.array_equal(np.isnan(s), np.isnan(c.scales)) and np.isnan(s).sum() == 2
    assert np.array_equal(s[~np.isnan(s)], c.scales[~np.isnan(s)])
    fine = ~np.isnan(s)
    assert np.array_equal(g.codes()[fine], c.codes[fine])
    append(dev, g, [22, 18, 19], [0, 1, 2, 3], np.ones((3, 96), np.float32), np.ones((3, 96), np.float32))
    # the poisoned K page of sequence 0 is full; V's of sequence 1 takes the new token and stays NaN
    assert np.isnan(g.scales()).sum() == 2
    g.free()


# (query heads, kv heads, dim, page, lens, news, window, rel extent)
ATTNS = [
    (1, 1, 16, 16, [0], [1], 0, 0), (8, 1, 128, 16, [1], [1], 0, 4), (64, 8, 128, 16, [700], [1], 0, 1024),
    (64, 16, 128, 16, [600], [1], 512, 512), (16, 1, 128, 64, [63], [2], 0, 16), (7, 1, 64, 32, [64], [1], 64, 1),
    (28, 4, 80, 32, [65, 0, 127, 128], [1, 1, 1, 1], 0, 50), (6, 2, 48, 16, [15, 16, 17, 31], [1, 0, 3, 2], 20, 300),
    (5, 5, 112, 64, [200], [9], 0, 64), (32, 8, 64, 32, [190, 3, 77], [5, 5, 5], 0, 100), (9, 3, 32, 16, [0, 0], [70, 1], 0, 33),
    (4, 2, 128, 16, [33], [100], 50, 40), (8, 8, 128, 64, [130], [140], 0, 128), (16, 2, 128, 16, [0], [200], 1, 8),
    (64, 8, 128, 16, [300, 0], [33, 64], 0, 512), (3, 3, 96, 32, [0] * 80, [k % 4 for k in range(80)], 0, 5),
    (16, 1, 16, 16, [1000], [1], 100, 7), (8, 2, 128, 32, [3000], [1], 0, 100),
    # many rows: a wave a unit
    (128, 64, 128, 16, [200, 0, 3], [130, 0, 9], 0, 64), (96, 32, 128, 64, [64], [180], 90, 0),
    (48, 16, 64, 32, [70, 0], [200, 150], 100, 40), (112, 56, 80, 16, [17, 0], [100, 60], 0, 300),
    # long: few units of many runs, whose partials are folded in groups first
    (16, 2, 128, 16, [5000], [1], 0, 1024), (14, 2, 80, 32, [9001, 100], [2, 0], 0, 50), (4, 4, 64, 64, [4500, 4400], [3, 1], 0, 0),
    (8, 1, 16, 16, [6000], [9], 0, 7), (2, 1, 32, 32, [30000], [1], 0, 0), (8, 1, 16, 64, [70000], [1], 0, 33),
]


@pytest.mark.parametrize("case", ATTNS, ids=lambda c: "-".join(str(a) if not isinstance(a, list) else "n%d" % len(a) for a in c))
def test_attn(dev, case):
    H, heads, dim, page, lens, news, window, R = case
    rng = np.random.default_rng(H * 1000 + dim + sum(lens))
    c, starts, n = make(rng, heads, dim, page, lens, news, rows_before=H % 2, rows_behind=H % 3)
    g = OnGpu(dev, c, off=16 * (H % 2))
    q = normal(rng, n, H, dim, scale=3.0)
    rel = normal(rng, n, H, R, scale=0.7) if R else None
    tau = rng.uniform(0.8, 1.4, n).astype(np.float32) if H % 3 else None
    got = attn(dev, g, lens, starts, q, rel, tau, window, 1.0 / dim)
    want, tol = c.attn(lens, starts, q, rel, tau, window, np.float32(1.0 / dim), fill=7.0)
    err = np.abs(got - want)
    # a result is rounded to f32 once more
    assert np.all(err <= tol + np.abs(want) * 2.0 ** -23), float((err - tol).max())
    g.free()


def test_attn_masked_values(dev):
    """NaN and infinities where nobody looks (pages before the window, slots behind the last token, rel_logits past
    the row's band) change nothing; the type's lowest value as a mask hides a column, and as the only score of a row
    gives the mean; -inf hides too, and a row of nothing but -inf is NaN."""
    rng = np.random.default_rng(3)
    H, heads, dim, page, lens, news, window, R = 6, 2, 64, 16, [150, 40], [2, 18], 40, 30
    c, starts, n = make(rng, heads, dim, page, lens, news)
    q, rel = normal(rng, n, H, dim, scale=2.0), normal(rng, n, H, R)
    want, tol = c.attn(lens, starts, q, rel, None, window, np.float32(1 / 64))
    for s, seen in ((0, 150 - 39), (1, 40 - 39)):
        for i in range(seen // page):
            c.scales[c.table[s, i]] = [[np.nan] * heads, [np.inf] * heads]
    rel2 = rel.copy()
    rel2[0, :, 12:] = np.finfo(np.float32).min            # hides the far columns of its band
    rel2[1, 0] = -np.inf                                   # the band hidden: only columns past it are left
    wantb, tolb = c.attn(lens, starts, q, rel2, None, window, np.float32(1 / 64))
    for r, w, t in ((rel, want, tol), (rel2, wantb, tolb)):
        g = OnGpu(dev, c)
        got = attn(dev, g, lens, starts, q, r, None, window, 1 / 64)
        assert np.isfinite(w).all() and np.all(np.abs(got - w) <= t + np.abs(w) * 2.0 ** -23)
        g.free()
    # every column within the band: the lowest value everywhere gives the mean of v, -inf everywhere NaN
    rel3 = np.full((n, H, 256), np.finfo(np.float32).min, np.float32)
    rel3[0] = -np.inf
    g = OnGpu(dev, c)
    got = attn(dev, g, lens, starts, q, rel3, None, window, 1 / 64)
    wantc, tolc = c.attn(lens, starts, q * 0, None, None, window, 1.0)
    assert np.isnan(got[0]).all()
    assert np.all(np.abs(got[1:] - wantc[1:]) <= tolc[1:] + np.abs(wantc[1:]) * 2.0 ** -23)
    g.free()


@pytest.mark.parametrize("H,heads,R", [(32, 32, 1), (64, 32, 3), (32, 32, 37), (96, 32, 64), (30, 30, 131), (128, 32, 300)])
def test_attn_many_rows_rel(dev, H, heads, R):
    """A wave a unit: rel_logits of other rows lie beside a row's own, in rows of every alignment; those nobody sees (past
    the row's position) are NaN, infinite or the lowest value, up to the buffer's first and last element."""
    rng = np.random.default_rng(H + R)
    lens, news, dim = [0, 90, 7], [150, 1, 400], 16 if R % 2 else 64
    c, starts, n = make(rng, heads, dim, 16, lens, news)
    q, rel = normal(rng, n, H, dim, scale=3.0), normal(rng, n, H, R, scale=0.7)
    tau = rng.uniform(0.8, 1.4, n).astype(np.float32)
    pos = np.concatenate([a + np.arange(b) for a, b in zip(lens, news)])
    unseen = np.broadcast_to(np.arange(R) > pos[:, None, None], rel.shape)
    want, tol = c.attn(lens, starts, q, np.where(unseen, 0, rel), tau, 0, np.float32(1 / dim))
    rel[unseen] = rng.choice(np.array([np.nan, np.inf, -np.inf, np.finfo(np.float32).min], np.float32), int(unseen.sum()))
    g = OnGpu(dev, c)
    got = attn(dev, g, lens, starts, q, rel, tau, 0, 1 / dim)
    assert np.all(np.abs(got - want) <= tol + np.abs(want) * 2.0 ** -23), float((np.abs(got - want) - tol).max())
    g.free()


@pytest.mark.parametrize("T", [1, 40])
def test_attn_nonfinite(dev, T):
    """A NaN scale of K or V reaches exactly the rows and heads that see its page; a NaN or infinite q its own head."""
    rng = np.random.default_rng(T)
    H, heads, dim, page, lens, news, window = 4, 2, 128, 16, [200], [T], 48
    c, starts, n = make(rng, heads, dim, page, lens, news)
    q = normal(rng, n, H, dim)
    first = (200 + T - 1 - 47) // page
    c.scales[c.table[0, first + 1], 0, 0] = np.nan
    c.scales[c.table[0, first + 2], 1, 1] = np.nan
    q[n - 1, 1, 3] = np.inf
    q[0, 3, 5] = np.nan
    g = OnGpu(dev, c)
    got = attn(dev, g, lens, starts, q, None, None, window, 1 / 128)
    want, tol = c.attn(lens, starts, q, None, None, window, 1 / 128)
    nan = np.isnan(want)
    assert nan.any() and (T == 1 or not nan.all()) and np.array_equal(nan, np.isnan(got))
    assert np.all(np.abs(got - want)[~nan] <= (tol + np.abs(want) * 2.0 ** -23)[~nan])
    g.free()


def test_large_magnitudes(dev):
    """Scales at both ends of the float range: scores of +-1e4, V of 1e30 and of 1e-30 in neighbouring pages."""
    rng = np.random.default_rng(17)
    H, heads, dim, page, lens, news = 4, 1, 64, 16, [100], [3]
    c, starts, n = make(rng, heads, dim, page, lens, news)
    c.scales[c.table[0, :7], 1] = np.array([1e28, 1e-30, 1.0, 1e28, 1e-38, 0.0, 1e10], np.float32)[:, None]
    q = normal(rng, n, H, dim, scale=0.05)
    got = attn(dev, (g := OnGpu(dev, c)), lens, starts, q, None, None, 0, 1 / 64)
    want, tol = c.attn(lens, starts, q, None, None, 0, 1 / 64)
    assert np.all(np.abs(got - want) <= tol + np.abs(want) * 2.0 ** -23)
    big = q * 4e5
    got = attn(dev, g, lens, starts, big, None, None, 0, 1 / 64)
    want, tol = c.attn(lens, starts, big, None, None, 0, 1 / 64)
    assert np.isfinite(got).all() and np.all(np.abs(got - want) <= tol + np.abs(want) * 2.0 ** -23)
    g.free()


def test_in_place_and_shared_pages(dev):
    """out may be q, and sequences may share the pages of a prefix."""
    rng = np.random.default_rng(23)
    c, starts, n = make(rng, 2, 64, 16, [64, 64, 64], [1, 2, 3])
    for s in (1, 2):
        c.table[s, :4] = c.table[0, :4]
    q = normal(rng, n, 8, 64)
    g = OnGpu(dev, c)
    bufs = [ints(dev, [64] * 3), ints(dev, starts), dev.shared_from(q)]
    dev.run(dev.L.sepia_hip_kv8_attn, B(g.desc), bufs[0], bufs[1], n, bufs[2], None, None, bufs[2], 8, 0, 0, 1 / 64)
    want, tol = c.attn([64] * 3, starts, q, None, None, 0, 1 / 64)
    got = dev.download(bufs[2], q.size).reshape(q.shape)
    assert np.all(np.abs(got - want) <= tol + np.abs(want) * 2.0 ** -23)
    for b in bufs:
        dev.free(b)
    g.free()


def test_offsets_past_32_bits(dev):
    """A pool of 5 GB: pages at its end, written, read back and attended to."""
    heads, dim, page, n_pages = 8, 128, 64, 40000
    rng = np.random.default_rng(31)
    c = Cache(4, 1, 4, heads, dim, page)
    c.reserve(0, 100)
    high = np.array([[n_pages - 1, n_pages - 7, -1, -1]], np.int32)
    small = {a: b for a, b in zip(high[0, :2], c.table[0, :2])}
    codes, scales = dev.alloc(n_pages * 2 * heads * page * dim, private=True), dev.alloc(n_pages * 2 * heads * 4, private=True)
    d = hip.Kv8Cache(n_pages=n_pages, max_pages=4, n_seqs=1, n_kv_heads=heads, head_dim=dim, page=page, codes=codes,
                     scales=scales, table=ints(dev, high))
    k, v = normal(rng, 100, heads * dim), normal(rng, 100, heads * dim)
    bufs = [ints(dev, [0]), ints(dev, [0, 100]), dev.shared_from(k), dev.shared_from(v), dev.alloc(k.nbytes), dev.alloc(v.nbytes)]
    dev.run(dev.L.sepia_hip_kv8_append, B(d), *bufs[:2], 100, bufs[2], bufs[3], None, 0.0)
    dev.run(dev.L.sepia_hip_kv8_read, B(d), *bufs[:2], 100, bufs[4], bufs[5])
    c.append([0], [0, 100], k, v)
    assert len(small) == 2
    for side in range(2):
        assert np.array_equal(dev.download(bufs[4 + side], k.size).reshape(100, heads, dim), c.rows(0, 0, 100)[side].astype(np.float32))
    q = normal(rng, 1, 16, dim)
    at = [ints(dev, [99]), ints(dev, [0, 1]), dev.shared_from(q), dev.alloc(q.nbytes)]
    dev.run(dev.L.sepia_hip_kv8_attn, B(d), at[0], at[1], 1, at[2], None, None, at[3], 16, 0, 0, 1 / 128)
    want, tol = c.attn([99], [0, 1], q, None, None, 0, 1 / 128)
    assert np.all(np.abs(dev.download(at[3], q.size).reshape(q.shape) - want) <= tol + np.abs(want) * 2.0 ** -23)
    for b in bufs + at + [codes, scales, d.table]:
        dev.free(b)


def test_device_errors(dev):
    """A page outside the pool and rows that do not fit fail the batch; the sequences that are whole are done, and
    nothing else is touched."""
    rng = np.random.default_rng(41)
    L = dev.L
    c, starts, n = make(rng, 2, 32, 16, [20, 5, 40], [2, 3, 1])
    q = normal(rng, n, 4, 32)
    want, tol = c.attn([20, 5, 40], starts, q, None, None, 0, 1 / 32)
    for word, lens, st, page in ((6, [20, 5, 40], starts, (1, 0, c.n_pages)), (6, [20, 5, 40], starts, (1, 0, -5)),
                                 (7, [20, -1, 40], starts, None), (7, [20, 2 ** 31 - 2, 40], starts, None),
                                 (7, [20, 5, 40], [0, 5, 2, 6], None), (7, [20, 5, 40], [0, 2, 5, 7], None),
                                 (7, [20, 64, 40], starts, None)):
        held = c.table.copy()
        if page:
            c.table[page[0], page[1]] = page[2]
        g = OnGpu(dev, c)
        c.table[:] = held
        k = normal(rng, n, 64)
        bufs = [ints(dev, lens), ints(dev, st), dev.shared_from(q), dev.alloc(q.nbytes), dev.shared_from(k), dev.alloc(k.nbytes),
                dev.alloc(k.nbytes)]
        before = g.codes()
        for call in (lambda: L.sepia_hip_kv8_attn(B(g.desc), bufs[0], bufs[1], n, bufs[2], None, None, bufs[3], 4, 0, 0, 1 / 32),
                     lambda: L.sepia_hip_kv8_read(B(g.desc), bufs[0], bufs[1], n, bufs[5], bufs[6]),
                     lambda: L.sepia_hip_kv8_append(B(g.desc), bufs[0], bufs[1], n, bufs[4], bufs[4], None, 0.0)):
            dev.begin()
            assert call() == 1
            assert L.sepia_gpu_end() == 0, (word, lens, st, page)
            assert L.sepia_hip_take_device_error() == 0   # end reported it
        if st == starts:
            got = dev.download(bufs[3], q.size).reshape(q.shape)
            for s in (0, 2):
                rows = slice(starts[s], starts[s + 1])
                assert np.all(np.abs(got[rows] - want[rows]) <= tol[rows] + np.abs(want[rows]) * 2.0 ** -23)
        free = {c.table[s, p // 16] for s, p0, p1 in ((0, 20, 22), (1, 0, 64), (2, 40, 41)) for p in range(p0, min(p1, 16 * c.max_pages))}
        kept = [p for p in range(c.n_pages) if p not in free]
        assert np.array_equal(g.codes()[kept], before[kept])
        for b in bufs:
            dev.free(b)
        g.free()
    dev.run(L.sepia_gpu_add, *(lambda b: (b, b, b))(dev.alloc(16)), 4)   # the batch after works


def test_refusals(dev):
    L = dev.L
    c, starts, n = make(np.random.default_rng(1), 2, 32, 16, [4], [2])
    g = OnGpu(dev, c)
    q, k, small = dev.alloc(n * 4 * 32 * 4), dev.alloc(n * 64 * 4), dev.alloc(16)
    k2, q2, rel = dev.alloc(n * 64 * 4), dev.alloc(n * 4 * 32 * 4), dev.alloc(n * 4 * 8 * 4)
    lens, st = ints(dev, [4]), ints(dev, starts)

    def calls(d, lens=lens, st=st, n=n, k=k, v=k2, q=q, out=q2, rel=None, tau=None, H=4, R=0, window=0, norm=None, eps=0.0,
              which="ara"):
        fns = {"a": lambda: L.sepia_hip_kv8_append(B(d) if d else None, lens, st, n, k, v, norm, eps),
               "r": lambda: L.sepia_hip_kv8_read(B(d) if d else None, lens, st, n, k, v),
               "t": lambda: L.sepia_hip_kv8_attn(B(d) if d else None, lens, st, n, q, rel, tau, out, H, R, window, 1.0)}
        return [fns[w]() for w in which]

    def desc(**over):
        d = hip.Kv8Cache.from_buffer_copy(g.desc)
        for key, val in over.items():
            setattr(d, key, val)
        return d

    assert calls(g.desc, which="art") == [0, 0, 0]   # no batch is open
    dev.begin()
    assert calls(g.desc, which="art") == [1, 1, 1] and calls(g.desc, n=0, which="art") == [1, 1, 1]
    for d in (None, desc(n_pages=0), desc(n_pages=c.n_pages + 1), desc(n_pages=2 ** 62), desc(max_pages=0), desc(max_pages=2 ** 40),
              desc(n_seqs=0), desc(n_seqs=2), desc(n_seqs=1 << 20), desc(n_kv_heads=0), desc(n_kv_heads=4), desc(n_kv_heads=-2),
              desc(head_dim=24), desc(head_dim=0), desc(head_dim=144), desc(head_dim=64), desc(page=8), desc(page=17), desc(page=128),
              desc(page=32), desc(codes=None), desc(scales=None), desc(table=None), desc(codes_off=8), desc(codes_off=16),
              desc(scales_off=2), desc(scales_off=4), desc(table_off=1), desc(table_off=4), desc(scales_off=2 ** 63)):
        assert calls(d, which="art") == [0, 0, 0]
    for over in (dict(lens=None), dict(st=None), dict(n=-1), dict(n=2 ** 40), dict(n=n + 1), dict(st=lens), dict(lens=small, st=small, n=n + 1)):
        assert calls(g.desc, which="art", **over) == [0, 0, 0], over
    for over in (dict(k=None), dict(v=None), dict(k=small), dict(v=small), dict(k=g.bufs[0]), dict(v=lens)):
        assert calls(g.desc, which="ar", **over) == [0, 0], over
    assert calls(g.desc, v=k, which="r") == [0] and calls(g.desc, norm=small, which="a") == [0]
    assert calls(g.desc, norm=k, eps=-1.0, which="a") == [0] and calls(g.desc, norm=k, eps=float("nan"), which="a") == [0]
    for over in (dict(q=None), dict(out=None), dict(q=small), dict(out=small), dict(out=g.bufs[0]), dict(out=lens), dict(out=g.bufs[2]),
                 dict(H=0), dict(H=3), dict(H=34), dict(H=6), dict(R=8), dict(rel=rel), dict(rel=rel, R=-1), dict(rel=rel, R=9),
                 dict(rel=rel, R=2 ** 31), dict(window=-1), dict(tau=small, n=5), dict(rel=q2, R=8), dict(tau=q2)):
        assert calls(g.desc, which="t", **over) == [0], over
    dev.end()
    for b in (q, k, small, k2, q2, rel, lens, st):
        dev.free(b)
    g.free()
