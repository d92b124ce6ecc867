"""The serving operators (include/sepia_hip_ext.h: kv8_append, kv8_read, kv8_attn, sample) restated in numpy, in 64
bits and value by value, from their definitions; and the cache's layout, so that tests fill and read pages."""
import numpy as np


class Cache:
    """A cache's codes [page][2][head][page * dim], scales and table, and what the operators do to them."""

    def __init__(self, n_pages, n_seqs, max_pages, heads, dim, page, rng=None):
        self.n_pages, self.n_seqs, self.max_pages = n_pages, n_seqs, max_pages
        self.heads, self.dim, self.page = heads, dim, page
        self.codes = np.zeros((n_pages, 2, heads, page * dim), np.int8)
        self.scales = np.zeros((n_pages, 2, heads), np.float32)
        if rng is not None:   # what earlier users of the pages left there
            self.codes[:] = rng.integers(-127, 128, self.codes.shape)
            self.scales[:] = rng.uniform(1e-3, 3e-2, self.scales.shape)
        order = rng.permutation(n_pages) if rng is not None else np.arange(n_pages)
        self.table = np.full((n_seqs, max_pages), -1, np.int32)   # never read behind a sequence's last token
        self.free = list(order)

    def reserve(self, s, tokens):
        """Pages for the first `tokens` tokens of sequence s."""
        for i in range(-(-tokens // self.page)):
            if self.table[s, i] < 0:
                self.table[s, i] = self.free.pop()

    def views(self, page):
        """K and V codes of a page as [token][head][dim]."""
        c = self.codes[page]
        return (c[0].reshape(self.heads, self.page, self.dim).transpose(1, 0, 2),
                c[1].reshape(self.heads, self.dim, self.page).transpose(2, 0, 1))

    def append(self, lens, starts, k, v, norm=None, eps=0.0):
        k64 = k.reshape(len(k), self.heads, self.dim).astype(np.float64)
        if norm is not None:
            k64 = k64 / np.sqrt((k64 ** 2).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * norm.astype(np.float64)
        v64 = v.reshape(len(v), self.heads, self.dim).astype(np.float64)
        for s in range(self.n_seqs):
            n = starts[s + 1] - starts[s]
            for p0 in range(lens[s] // self.page * self.page, lens[s] + n, self.page):
                lo, hi = max(lens[s], p0), min(lens[s] + n, p0 + self.page)
                if lo >= hi:
                    continue
                page = self.table[s, p0 // self.page]
                rows = slice(starts[s] + lo - lens[s], starts[s] + hi - lens[s])
                for side, x in enumerate((k64[rows], v64[rows])):
                    codes = self.views(page)[side]
                    for h in range(self.heads):
                        with np.errstate(all="ignore"):
                            y = x[:, h]
                            most = np.abs(y).max().astype(np.float32)
                            old = self.scales[page, side, h] if lo > p0 else np.float32(0)
                            new = np.float32(np.maximum(old, most * np.float32(1 / 127)))
                            if not np.isfinite(new):
                                self.scales[page, side, h] = np.nan
                                continue
                            if new > old > 0:
                                was = codes[:lo - p0, h].astype(np.float64)
                                codes[:lo - p0, h] = np.rint(was * np.float64(old) / np.float64(new))
                            c = np.rint(y / np.float64(new)) if new > 0 else np.zeros_like(y)
                            codes[lo - p0:hi - p0, h] = np.clip(c, -127, 127)
                            self.scales[page, side, h] = new

    def rows(self, s, lo, hi):
        """Cached K and V at positions [lo, hi) of sequence s, [position][head][dim], in 64 bits."""
        out = [np.zeros((hi - lo, self.heads, self.dim)) for _ in range(2)]
        for p in range(lo, hi):
            page = self.table[s, p // self.page]
            for side in range(2):
                with np.errstate(invalid="ignore"):   # a page may be NaN, and a code 0 of an infinite scale is
                    out[side][p - lo] = (self.views(page)[side][p % self.page].astype(np.float64) *
                                         self.scales[page, side][:, None].astype(np.float64))
        return out

    def attn(self, lens, starts, q, rel=None, tau=None, window=0, c=1.0, fill=np.nan):
        """(out, tolerance), both [rows][heads][dim]; rows outside all sequences hold `fill`.

        The tolerance, in units of u = 2^-24 (half a step of f32 relative to the value): a dot product of D terms
        of summed magnitude A (after the scale c) is off by at most D A u as an f32 chain (less as an exact sum of
        q's 24-bit roundings); adding the bias and the scales' products are 4 roundings of at most the largest
        score S; the difference to the maximum (at most 2 S) rounds once more, and the exponential is within 2 u and
        its argument's product with log2 e within 2 S u. So a weight is off by d = (D A + 8 S + 4) u relative, the
        quotient of the two sums by 2 d, and the sums themselves by (tiles of 64 + 80) u of the weighted magnitudes
        (64 terms, or a 23-bit rounding of each weight relative to the tile's largest, then a chain over the tiles
        and the splits). Everything relative to the largest |v| in sight."""
        n_rows, H = q.shape[0], q.shape[1]
        out, tol = np.full(q.shape, fill, np.float64), np.zeros(q.shape)
        for s in range(self.n_seqs):
            n = starts[s + 1] - starts[s]
            if not n:
                continue
            k, v = self.rows(s, 0, lens[s] + n)
            for i in range(n):
                t, pos = starts[s] + i, lens[s] + i
                lo = max(0, pos - window + 1) if window else 0
                dist = pos - np.arange(lo, pos + 1)
                for h in range(H):
                    hk = h // (H // self.heads)
                    kk, vv, qq = k[lo:pos + 1, hk], v[lo:pos + 1, hk], q[t, h].astype(np.float64)
                    with np.errstate(all="ignore"):
                        z = kk @ qq * c
                        if rel is not None:
                            R = rel.shape[2]
                            b = rel[t, h, np.minimum(dist, R - 1)].astype(np.float64) * (1.0 if tau is None else tau[t])
                            z = z + np.where(dist < R, b, 0.0)
                        e = np.exp(z - z.max())
                        out[t, h] = e @ vv / e.sum()
                        fin = np.isfinite(z) & (np.abs(z) < 1e30)
                        A = (np.abs(kk) @ np.abs(qq)).max() * c
                        S = np.abs(z[fin]).max() if fin.any() else 0.0
                        d = (self.dim * A + 8 * S + 4) * 2.0 ** -24
                        tol[t, h] = (2 * d + (len(dist) / 64 + 81) * 2.0 ** -24) * np.abs(vv).max()
        return out, tol


def sample(x, u, temperature=1.0, top_p=1.0, min_p=0.0, top_k=0):
    """(token, its share, how near the decision was: the smallest distance of a cumulative weight that decided
    something to what it was compared with, the largest weight being 1)."""
    x = x.astype(np.float64)
    on = x > -np.inf
    if not on.any():
        return -1, 0.0, 1.0
    idx = np.flatnonzero(on)
    order = idx[np.argsort(-x[idx], kind="stable")]
    if not temperature > 0:
        return order[0], 1.0, 1.0
    if top_k > 0:
        order = order[:top_k]
    m = x[order[0]]
    with np.errstate(all="ignore"):
        w = np.where(x[order] == m, 1.0, np.exp((x[order] - m) / np.float64(np.float32(temperature))))
    cum, near = np.cumsum(w), 1.0
    n = len(order)
    if top_p < 1:
        want = np.float64(np.float32(max(top_p, 0.0))) * cum[-1]
        n = int(np.argmax(cum >= want)) + 1 if want > 0 else 1
        near = min(near, np.abs(cum - want).min())
    if min_p > 0:
        floor = np.float64(np.float32(min(min_p, 1.0)))
        n = min(n, int((w >= floor).sum()))
        near = min(near, np.abs(w[w != 1.0] - floor).min() if (w != 1.0).any() else 1.0)
    total = cum[n - 1]
    cut = np.float64(np.float32(min(max(u, 0.0), 1.0))) * total
    j = min(int(np.searchsorted(cum[:n], cut, side="right")), n - 1)
    near = min(near, np.abs(cum[:n] - cut).min())
    return order[j], w[j] / total, near
