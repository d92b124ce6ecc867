// sample.h -- the next token of each row of logits: temperature, top-k,
// top-p, min-p, and a draw by a given uniform number.
//
// With x the row's logits, m their maximum and T the temperature, a token's
// weight is w = e^((x - m) / T); -inf and NaN have none, nor has a token below
// one of +inf. The tokens are
// ordered by falling logit, equal ones by index. Kept are the first k of them
// (top-k), of these the shortest beginning whose weight reaches p of theirs
// (top-p), and of these the ones with w >= min-p: a beginning of the order
// each time. The draw is the first token whose cumulative weight exceeds u
// times the kept weight. T <= 0: the first token of the order.
//
// Weights are summed as integers in units of 2^-43 of the largest, so that
// every sum is exact and does not depend on its order: a row of up to 2^20
// tokens sums to at most 2^63, and a weight is within 2^-44 of its value
// (over n tokens the sums err by about sqrt(n) 2^-45, 3e-11 at most).
//
// Nothing is sorted but the few tokens next to a decision. One pass over the
// row counts and sums the tokens by their weight's logarithm (1024 bins, 32 to
// the octave, 16 from 2^-16 on, so that the last one, from 2^-48, weighs
// nothing and never decides). The bins' prefix sums then bound where the k-th token, the
// top-p border and the draw fall: each decision's bound gives the next one's,
// a bin or a few in all. A second pass gathers the tokens of those bins, and
// the three are decided in turn: a decision's bin is cut into 1024 pieces by
// place in the order, its piece again while it has more than a few tokens (equal
// logits: by index), and those few are compared with each other. Where the
// gathered tokens are too many (flat rows, long runs of equal logits) the same
// is done with passes over the row. (One row of 256 that gathered 5376 of 199999
// tokens, with room for 4096, made the call 340 us in the place of 196.) (Sorting the gathered tokens by a network
// took 10 us for 250 of them and 25 us for 1100.)
//
// A row is cut into chunks where the rows are fewer than the chip's places,
// and the passes become launches: each chunk's first token of the order (the
// row's maximum), each chunk's bins, and the gathering: every workgroup of it
// sums the row's bins and finds the bins to gather for itself, and the last of
// a row to arrive with its chunk's tokens decides. (Bins added up by atomics
// took 73 us at 48 rows of 10 chunks: 64-bit device-scope atomics are carried
// out at the memory's side.)
#pragma once
#include "common.h"
#include "serve.h"
#include "serve_layout.h"
#include <stddef.h>

#define SAMPLE_ONE 8796093022208.0    // 2^43: the largest weight
#define SAMPLE_WAVES (SAMPLE_NT / 64)
#define SAMPLE_CAP 4096               // gathered tokens in shared memory
#define SAMPLE_FEW 16                 // tokens that are compared with each other (60 of them took 4 us)

// Keys fall as logits rise: 0 is the largest. -0 and +0 are equal.
__device__ __forceinline__ uint32_t sample_key(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
    return (int32_t)b < 0 ? b : ~b & 0x7FFFFFFFu;
}
__device__ __forceinline__ float sample_logit(uint32_t key) {
    return __builtin_bit_cast(float, (int32_t)key < 0 ? key : ~key & 0x7FFFFFFFu);
}
// Place in the order: key, then index. Tokens without weight: the last.
__device__ __forceinline__ float sample_token(unsigned long long place) { return sample_logit((uint32_t)(place >> 20)); }
#define SAMPLE_NONE 0xFFFFFFFFFFFFFFFFull
__device__ __forceinline__ unsigned long long sample_place(float x, int i) {
    return x > -INFINITY ? ((unsigned long long)sample_key(x) << 20) | (uint32_t)i : SAMPLE_NONE;
}

// 2^(j / 256), filled by the workgroup: a product of the powers that j's bits
// stand for, within 8 roundings of 2^-53.
struct SamplePow {
    double t[256];
    __device__ __forceinline__ void fill() {
        const double p[8] = {0x1.00b1afa5abcbfp+0, 0x1.0163da9fb3335p+0, 0x1.02c9a3e778061p+0, 0x1.059b0d3158574p+0,
                             0x1.0b5586cf9890fp+0, 0x1.172b83c7d517bp+0, 0x1.306fe0a31b715p+0, 0x1.6a09e667f3bcdp+0};
        const int j = (int)threadIdx.x;
        if (j >= 256) return;
        double e = 1.0;
#pragma unroll
        for (int i = 0; i < 8; i++) e *= j >> i & 1 ? p[i] : 1.0;
        t[j] = e;
    }
};
// The weight's logarithm in units of 1/256 octave, (x - m) 256 log2(e) / T,
// at least -15360 (2^-60). The minimum also makes 0 of infinity - infinity.
__device__ __forceinline__ double sample_log(float x, float m, double scale) {
    return __builtin_fmax(__builtin_fmin(((double)x - (double)m) * scale, 0.0), -15360.0);
}
// Its nearest integer (1.5 * 2^52 leaves it in the sum's low word), and the
// bin of eight of those, or from 512 on of sixteen. (With eights throughout the
// last bin began at 2^-32: a k-th token in there, as a low temperature has it,
// was sought among most of a row: sepia_sample_pick took 70 us for 16 rows of
// 128000 with a top-k, 15 us with the wider ones.)
#define SAMPLE_BIG 6755399441055744.0
__device__ __forceinline__ int sample_low(double t) { return (int)(uint32_t)__builtin_bit_cast(uint64_t, t); }
__device__ __forceinline__ int sample_bin(double z) {
    const int t = -sample_low(z + SAMPLE_BIG);
    return min(min(t >> 3, (t >> 4) + 256), SAMPLE_BINS - 1);
}
// The least of bin b's.
__device__ __forceinline__ int sample_edge(int b) { return b < 512 ? 8 * b : 16 * (b - 256); }
// 2^(z / 256 + shift): the nearest integer by the table, the rest, at most 1/2,
// by the fourth power of the series of 2^(r / 256) (4e-17 off).
__device__ __forceinline__ double sample_pow(double z, const SamplePow &P, int shift) {
    const double c = 0.69314718055994530942 / 256.0, t = z + SAMPLE_BIG, r = z - (t - SAMPLE_BIG);
    const int n = sample_low(t);
    double e = __builtin_fma(r, c * c * c * c / 24.0, c * c * c / 6.0);
    e = __builtin_fma(e, r, c * c / 2.0);
    e = __builtin_fma(e, r, c);
    e = __builtin_fma(e, r, 1.0);
    return __builtin_ldexp(e * P.t[n & 255], (n >> 8) + shift);
}
// The weight in units of 2^-43 (2^52 leaves it in the sum's low 52 bits).
__device__ __forceinline__ unsigned long long sample_mass(double z, const SamplePow &P) {
    return __builtin_bit_cast(unsigned long long, sample_pow(z, P, 43) + 4503599627370496.0) & 0xFFFFFFFFFFFFFull;
}

struct SampleLds {
    // by bin, then by a bin's pieces; of the bins before
    unsigned long long mass[SAMPLE_BINS + 1], upto[SAMPLE_BINS + 1];
    uint32_t count[SAMPLE_BINS + 1], cupto[SAMPLE_BINS + 1];
    unsigned long long list[SAMPLE_CAP], few[SAMPLE_FEW];
    unsigned long long over_min, wave[SAMPLE_WAVES], set[SAMPLE_BINS / 64];
    uint32_t n;
    SamplePow pow;
};

// f(value, index) for the row's tokens i0 .. i1 - 1, SAMPLE_LOADS loads of a
// thread in flight at a time (one at a time, a pass over 100003 logits by one
// workgroup took 40 us, a loaded memory round trip an iteration).
#define SAMPLE_LOADS 8
template <class F>
__device__ __forceinline__ void sample_walk(const float *__restrict__ x, int i0, int i1, F f) {
    for (int i = i0 + (int)threadIdx.x; i < i1; i += SAMPLE_LOADS * SAMPLE_NT) {
        float v[SAMPLE_LOADS];
#pragma unroll
        for (int j = 0; j < SAMPLE_LOADS; j++) v[j] = x[min(i + j * SAMPLE_NT, i1 - 1)];
#pragma unroll
        for (int j = 0; j < SAMPLE_LOADS; j++)
            if (i + j * SAMPLE_NT < i1 && v[j] > -INFINITY) f(v[j], i + j * SAMPLE_NT);
    }
}

__device__ __forceinline__ unsigned long long sample_lane(unsigned long long v, int l) {
    return (unsigned long long)(uint32_t)__builtin_amdgcn_readlane((int)v, l) |
           (unsigned long long)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32;
}
// f over the lanes up to each lane's own, by lane moves (by LDS permutes, and
// with the bins' tail summed by three such scans, 48 rows took 57.8 us in the
// place of 54.8): rows of 16, then a
// row's last lane to the next row, then two rows' to the next two. `none`: f's
// neutral value.
template <class F>
__device__ __forceinline__ unsigned long long sample_lanes(unsigned long long v, unsigned long long none, F f) {
#define SAMPLE_DPP(ctrl, rows)                                                                                         \
    {                                                                                                                  \
        const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)v, ctrl, rows, 0xF, false);          \
        const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp((int)(none >> 32), (int)(v >> 32), ctrl, rows, 0xF, false); \
        v = f(v, (unsigned long long)hi << 32 | lo);                                                                   \
    }
    SAMPLE_DPP(0x111, 0xF)
    SAMPLE_DPP(0x112, 0xF)
    SAMPLE_DPP(0x114, 0xF)
    SAMPLE_DPP(0x118, 0xF)
    SAMPLE_DPP(0x142, 0xA)
    SAMPLE_DPP(0x143, 0xC)
#undef SAMPLE_DPP
    return v;
}
__device__ __forceinline__ unsigned long long sample_sums(unsigned long long v) {
    return sample_lanes(v, 0, [](unsigned long long a, unsigned long long b) { return a + b; });
}
// Exclusive prefix sums over the workgroup's threads; the total too.
__device__ __forceinline__ unsigned long long sample_scan(unsigned long long v, unsigned long long *wave,
                                                          unsigned long long &total) {
    const int lane = (int)threadIdx.x & 63, w = (int)threadIdx.x >> 6;
    const unsigned long long s = sample_sums(v);
    __syncthreads();
    if (lane == 63) wave[w] = s;
    __syncthreads();
    unsigned long long before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < SAMPLE_WAVES; i++) {
        const unsigned long long t = wave[i];
        if (i < w) before += t;
        total += t;
    }
    return before + s - v;
}
__device__ __forceinline__ unsigned long long sample_min(unsigned long long v, unsigned long long *wave) {
    v = sample_lanes(v, ~0ull, [](unsigned long long a, unsigned long long b) { return b < a ? b : a; });
    __syncthreads();
    if ((threadIdx.x & 63) == 63) wave[threadIdx.x >> 6] = v;
    __syncthreads();
    v = wave[0];
#pragma unroll
    for (int i = 0; i < SAMPLE_WAVES; i++) v = wave[i] < v ? wave[i] : v;
    return v;
}

__device__ __forceinline__ void sample_clear(SampleLds &L) {
    for (int i = (int)threadIdx.x; i < SAMPLE_BINS; i += SAMPLE_NT) L.mass[i] = 0, L.count[i] = 0;
    __syncthreads();
}
// Prefix sums of L.mass and, where counted, L.count, to `upto` and `cupto`
// (which may be the same arrays).
__device__ __forceinline__ void sample_prefix(SampleLds &L, unsigned long long *upto, uint32_t *cupto, bool counted) {
    const int b = 2 * (int)threadIdx.x;
    unsigned long long total;
    __syncthreads();
    const unsigned long long m0 = L.mass[b], c0 = L.count[b];
    const unsigned long long m = sample_scan(m0 + L.mass[b + 1], L.wave, total);
    upto[b] = m;
    upto[b + 1] = m + m0;
    if (b == 0) upto[SAMPLE_BINS] = total;
    if (!counted) {
        __syncthreads();
        return;
    }
    const unsigned long long c = sample_scan(c0 + L.count[b + 1], L.wave, total);
    cupto[b] = (uint32_t)c;
    cupto[b + 1] = (uint32_t)(c + c0);
    if (b == 0) cupto[SAMPLE_BINS] = (uint32_t)total;
    __syncthreads();
}
// The bin with upto[b] <= over < upto[b + 1] (cupto with by_count), by every
// wave for itself: 64 bins apart, then 16 of them.
__device__ __forceinline__ int sample_seek(const unsigned long long *upto, const uint32_t *cupto, bool by_count,
                                           unsigned long long over) {
    const int lane = (int)threadIdx.x & 63;
    const uint64_t far = __ballot((by_count ? cupto[16 * lane] : upto[16 * lane]) <= over);
    const int b = 16 * (63 - __builtin_clzll(far)) + (lane & 15);
    const uint64_t near = __ballot((by_count ? cupto[b] : upto[b]) <= over) & 0xFFFF;
    return 16 * (63 - __builtin_clzll(far)) + 31 - __builtin_clz((uint32_t)near);
}

// What a row asks for, as its workgroups need it.
struct SampleAsk {
    const float *x;
    float m, t, p, f, u;           // largest logit, temperature, top-p, min-p (0: off), u
    int vocab, k;
    double scale;
    unsigned long long over_min;   // the weight of its tokens of w >= min-p (no min-p: the largest number)
    bool by_k, by_p;
};
__device__ __forceinline__ unsigned long long sample_share(float f, unsigned long long total) {
    return (unsigned long long)((double)f * (double)total);
}
// The least cumulative weight that is at least p of the total.
__device__ __forceinline__ unsigned long long sample_want(float p, unsigned long long total) {
    const double w = __builtin_ceil((double)fmaxf(p, 0.0f) * (double)total);
    return w >= 1.0 ? (unsigned long long)w : 1;
}
__device__ __forceinline__ unsigned long long sample_over(float u, unsigned long long kept) {
    const unsigned long long over = u > 0.0f ? sample_share(fminf(u, 1.0f), kept) : 0;
    return over >= kept ? kept ? kept - 1 : 0 : over;
}
// A logit that no token of bin b lies below, and one that none lies above.
__device__ __forceinline__ float sample_least(const SampleAsk &q, int b) {
    if (q.m == INFINITY) return q.m;   // all other tokens are in the last bin
    const double x = (double)q.m - (double)(sample_edge(b + 1) + 1) / q.scale;
    return (float)(x - (fabs(x) + fabs((double)q.m)) * 0x1p-20);   // rounded down, surely
}
__device__ __forceinline__ float sample_most(const SampleAsk &q, int b) {
    if (b == 0 || q.m == INFINITY) return q.m;
    const double x = (double)q.m - (double)(sample_edge(b) - 1) / q.scale;
    return fminf(q.m, (float)(x + (fabs(x) + fabs((double)q.m)) * 0x1p-20));
}
// From the row's bins in L.mass (and L.count, if its k may cut): their prefix
// sums, and in L.set the bins that decide. Returns the least logit of those.
__device__ __forceinline__ float sample_bounds(SampleAsk &q, SampleLds &L) {
    const int tid = (int)threadIdx.x;
    sample_prefix(L, L.upto, L.cupto, q.k > 0);
    const unsigned long long all = L.upto[SAMPLE_BINS];
    q.by_k = q.k > 0 && (uint32_t)q.k < L.cupto[SAMPLE_BINS];   // counts are there for a k alone
    q.by_p = q.p < 1.0f;
    // each decision's bin, or the range of bins that the one before leaves it
    unsigned long long lo = all, hi = all;   // the weight kept so far is in [lo, hi]
    int bk = -1, p0 = 0, p1 = -1;
    if (q.by_k) {
        bk = sample_seek(L.upto, L.cupto, true, (unsigned long long)q.k - 1);
        q.by_k = L.upto[bk] < all;   // else nothing that weighs is cut
        if (!q.by_k) bk = -1;
        else lo = L.upto[bk], hi = L.upto[bk + 1];
    }
    if (q.by_p) {
        const unsigned long long w0 = sample_want(q.p, lo), w1 = sample_want(q.p, hi);
        p0 = sample_seek(L.upto, L.cupto, false, w0 - 1);
        p1 = w0 == w1 ? p0 : sample_seek(L.upto, L.cupto, false, w1 - 1);
        lo = w0;
        hi = L.upto[p1 + 1];
    }
    lo = lo < q.over_min ? lo : q.over_min;
    hi = hi < q.over_min ? hi : q.over_min;
    const int d0 = sample_seek(L.upto, L.cupto, false, sample_over(q.u, lo));
    const int d1 = lo == hi ? d0 : sample_seek(L.upto, L.cupto, false, sample_over(q.u, hi));
    for (int b = tid; b < SAMPLE_BINS; b += SAMPLE_NT) {
        const unsigned long long word = __ballot(b == bk || (b >= p0 && b <= p1) || (b >= d0 && b <= d1));
        if ((tid & 63) == 0) L.set[b >> 6] = word;
    }
    if (tid == 0) L.n = 0;
    __syncthreads();
    return sample_least(q, max(max(bk, p1), d1));
}
// One to the row's list in scratch; r->n counts them, also past its end.
__device__ __forceinline__ void sample_put(SampleRow *r, uint32_t at, unsigned long long place) {
    if (at < SAMPLE_MANY) __hip_atomic_store(&r->list[at], place, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// The chosen bins' tokens among the row's i0 .. i1 - 1 into L.list; L.n counts
// them, also where they are more than the list holds. Those go to the row's
// list, if there is one.
__device__ __forceinline__ void sample_gather(const SampleAsk &q, float least, int i0, int i1, SampleLds &L, SampleRow *r) {
    sample_walk(q.x, i0, i1, [&](float v, int i) {
        if (!(v >= least)) return;
        const int b = sample_bin(sample_log(v, q.m, q.scale));
        if (!(L.set[b >> 6] >> (b & 63) & 1)) return;
        const uint32_t at = atomicAdd(&L.n, 1u);
        if (at < SAMPLE_CAP) L.list[at] = sample_place(v, i);
        else if (r) sample_put(r, __hip_atomic_fetch_add(&r->n, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT), sample_place(v, i));
    });
    __syncthreads();
}
// The first token of bin b whose cumulative weight from the bin's start
// (by_count: place from 1) exceeds `over`, and the weight up to and with it,
// among the n gathered tokens, in shared memory where they fit, else in the
// row's list (far), or among the whole row's (neither).
struct SampleAt {
    unsigned long long place, cum;
};
__device__ __forceinline__ SampleAt sample_settle(const SampleAsk &q, int b, bool by_count, unsigned long long over,
                                                  uint32_t n, const SampleRow *far, SampleLds &L) {
    const int lane = (int)threadIdx.x & 63;
    const bool listed = n <= SAMPLE_CAP;
    const auto walk = [&](auto f) {
        if (listed) {
            for (uint32_t i = threadIdx.x; i < n; i += SAMPLE_NT) {
                const unsigned long long p = L.list[i];
                const double z = sample_log(sample_token(p), q.m, q.scale);
                if (sample_bin(z) == b) f(p, z);
            }
        } else if (far) {
            for (uint32_t i = threadIdx.x; i < n; i += SAMPLE_LOADS * SAMPLE_NT) {
                unsigned long long p[SAMPLE_LOADS];
#pragma unroll
                for (uint32_t j = 0; j < SAMPLE_LOADS; j++)
                    p[j] = __hip_atomic_load(&far->list[min(i + j * SAMPLE_NT, n - 1)], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
                for (uint32_t j = 0; j < SAMPLE_LOADS; j++) {
                    const double z = sample_log(sample_token(p[j]), q.m, q.scale);
                    if (i + j * SAMPLE_NT < n && sample_bin(z) == b) f(p[j], z);
                }
            }
        } else {
            sample_walk(q.x, 0, q.vocab, [&](float v, int i) {
                const double z = sample_log(v, q.m, q.scale);
                if (sample_bin(z) == b) f(sample_place(v, i), z);
            });
        }
    };
    unsigned long long first = 0, before = 0;   // the places from `first` on, 2^bits of them
    int bits = 0;
    uint32_t left = listed || far ? n : q.by_k ? L.cupto[b + 1] - L.cupto[b] : ~0u;   // at most (bins are counted for a k)
    if (!(listed && n <= SAMPLE_FEW)) {
        first = (unsigned long long)sample_key(sample_most(q, b)) << 20;
        const unsigned long long last = ((unsigned long long)sample_key(fmaxf(sample_least(q, b), -3.402823466e38f)) << 20) | 0xFFFFF;
        bits = 64 - __builtin_clzll((last - first) | 1);
    }
    while (left > SAMPLE_FEW) {
        const int drop = max(bits - 10, 0);
        sample_clear(L);
        walk([&](unsigned long long p, double z) {
            const unsigned long long piece = (p - first) >> drop;
            if (piece >= SAMPLE_BINS) return;
            atomicAdd(&L.count[piece], 1u);
            atomicAdd(&L.mass[piece], sample_mass(z, L.pow));
        });
        sample_prefix(L, L.mass, L.count, true);
        const int piece = sample_seek(L.mass, L.count, by_count, over);
        over -= by_count ? L.count[piece] : L.mass[piece];
        before += L.mass[piece];
        left = L.count[piece + 1] - L.count[piece];
        first += (unsigned long long)piece << drop;
        bits = drop;
        __syncthreads();
    }
    // a few tokens: every wave compares them with each other
    int m = (int)n;
    unsigned long long p = SAMPLE_NONE, w = 0;
    if (listed && n <= SAMPLE_FEW) {
        if (lane < m) p = L.list[lane];
    } else {
        if (threadIdx.x == 0) L.n = 0;
        __syncthreads();
        walk([&](unsigned long long p, double) {
            if ((p - first) >> bits == 0) L.few[atomicAdd(&L.n, 1u)] = p;
        });
        __syncthreads();
        m = (int)L.n;
        if (lane < m) p = L.few[lane];
        __syncthreads();
    }
    bool here = p != SAMPLE_NONE;
    if (here) {
        const double z = sample_log(sample_token(p), q.m, q.scale);
        here = sample_bin(z) == b;
        if (here) w = sample_mass(z, L.pow);
        else p = SAMPLE_NONE;
    }
    unsigned long long cum = w, place = 1;
    for (int j = 0; j < m; j++) {
        const unsigned long long pj = sample_lane(p, j), wj = sample_lane(w, j);
        cum += pj < p ? wj : 0;
        place += pj < p;
    }
    const uint64_t hit = __ballot(here && (by_count ? place == over + 1 : cum - w <= over && over < cum));
    const int l = hit ? __builtin_ctzll(hit) : 0;
    return SampleAt{sample_lane(p, l), before + sample_lane(cum, l)};
}
// The decisions, from the gathered tokens where they fit L.list: the k-th
// token, the top-p border, the draw.
__device__ __forceinline__ void sample_finish(const SampleArgs &a, int row, const SampleAsk &q, uint32_t n, const SampleRow *far,
                                              SampleLds &L) {
    unsigned long long kept = L.upto[SAMPLE_BINS], place = 0;
    for (int step = q.by_k ? 0 : q.by_p ? 1 : 2; step <= 2; step = step == 0 && q.by_p ? 1 : step == 2 ? 3 : 2) {
        if (step == 2 && kept > q.over_min) kept = q.over_min;
        const unsigned long long over = step == 0 ? (unsigned long long)q.k - 1
                                        : step == 1 ? sample_want(q.p, kept) - 1 : sample_over(q.u, kept);
        const int b = sample_seek(L.upto, L.cupto, step == 0, over);
        const SampleAt r = sample_settle(q, b, step == 0, over - (step == 0 ? L.cupto[b] : L.upto[b]), n, far, L);
        if (step == 2) place = r.place;
        else kept = L.upto[b] + r.cum;
    }
    if (threadIdx.x == 0) {
        a.token[row] = (int32_t)(place & 0xFFFFF);
        if (a.prob)
            a.prob[row] = (float)(sample_pow(sample_log(sample_token(place), q.m, q.scale), L.pow, 43) / (double)kept);
    }
}

// A row's first token of the order among i0 .. i1 - 1.
__device__ __forceinline__ unsigned long long sample_best(const float *x, int i0, int i1, unsigned long long *wave) {
    unsigned long long best = SAMPLE_NONE;
    sample_walk(x, i0, i1, [&](float v, int i) {
        const unsigned long long p = sample_place(v, i);
        best = p < best ? p : best;
    });
    return sample_min(best, wave);
}
// A row's first token from its chunks'.
__device__ __forceinline__ unsigned long long sample_first(const SampleArgs &a, int row, unsigned long long *wave) {
    unsigned long long best = SAMPLE_NONE;
    if ((int)threadIdx.x < a.chunks) best = a.bins[(int64_t)row * a.chunks + (int)threadIdx.x].best;
    return sample_min(best, wave);
}
// A row's parameters: loads without branches, in flight together at a kernel's
// entry (what is not there is read from u, and the value that is off taken).
__device__ __forceinline__ SampleAsk sample_ask(const SampleArgs &a, int row) {
    SampleAsk q;
    const float t = (a.temperature ? a.temperature : a.u)[row], p = (a.top_p ? a.top_p : a.u)[row];
    const float f = (a.min_p ? a.min_p : a.u)[row];
    const int k = (a.top_k ? a.top_k : (const int32_t *)a.u)[row];
    q.u = a.u[row];
    q.x = a.logits + (int64_t)row * a.stride;
    q.vocab = a.vocab;
    q.t = a.temperature ? t : 1.0f;
    q.p = a.top_p ? p : 1.0f;
    q.f = a.min_p && f > 0.0f ? fminf(f, 1.0f) : 0.0f;
    q.k = a.top_k ? k : 0;
    q.over_min = ~0ull;
    return q;
}
// From the row's first token its largest logit and scale; whether that token is
// all there is to decide (the workgroup of `write` says so).
__device__ __forceinline__ bool sample_done(const SampleArgs &a, int row, SampleAsk &q, unsigned long long best, bool write) {
    q.m = sample_logit((uint32_t)(best >> 20));
    q.scale = 256.0 * 1.4426950408889634074 / (q.m < INFINITY ? (double)q.t : 1.0);   // below +inf nothing weighs, at any T
    if (best != SAMPLE_NONE && q.t > 0.0f && q.k != 1) return false;
    if (write && threadIdx.x == 0) {
        a.token[row] = best == SAMPLE_NONE ? -1 : (int32_t)(best & 0xFFFFF);
        if (a.prob) a.prob[row] = best == SAMPLE_NONE ? 0.0f : 1.0f;
    }
    return true;
}
// The bins of the row's tokens i0 .. i1 - 1 in L.mass and, where its k may
// cut, L.count; q.over_min.
__device__ __forceinline__ void sample_bins(SampleAsk &q, int i0, int i1, SampleLds &L) {
    const int tid = (int)threadIdx.x;
    const unsigned long long floor_mass = q.f > 0.0f ? (unsigned long long)__builtin_ceil((double)q.f * SAMPLE_ONE) : 0;
    L.pow.fill();
    if (tid == 0) L.over_min = 0;
    sample_clear(L);
    unsigned long long tail = 0, over_min = 0;
    uint32_t ntail = 0;
    const bool counted = q.k > 0;
    const auto add = [&](float v, bool floor) {
        const double z = sample_log(v, q.m, q.scale);
        const int b = sample_bin(z);
        const unsigned long long w = sample_mass(z, L.pow);
        if (floor && w >= floor_mass) over_min += w;
        if (b == SAMPLE_BINS - 1) {   // many of a row's tokens: not one by one to the same bin
            tail += w;
            ntail++;
        } else {
            atomicAdd(&L.mass[b], w);
            if (counted) atomicAdd(&L.count[b], 1u);
        }
    };
    if (floor_mass) sample_walk(q.x, i0, i1, [&](float v, int) { add(v, true); });
    else sample_walk(q.x, i0, i1, [&](float v, int) { add(v, false); });
    // the waves' sums, by each wave's last lane
    tail = sample_sums(tail);
    if (floor_mass) over_min = sample_sums(over_min);
    if (counted) ntail = (uint32_t)sample_sums(ntail);
    if ((tid & 63) == 63) {
        atomicAdd(&L.mass[SAMPLE_BINS - 1], tail);
        if (floor_mass) atomicAdd(&L.over_min, over_min);
        if (counted) atomicAdd(&L.count[SAMPLE_BINS - 1], ntail);
    }
    __syncthreads();
    if (floor_mass) q.over_min = L.over_min;
}

// Grid (chunks, rows): the chunk's first token of the order; the row's counters
// cleared. One row of 100003 4.6 us; 256 of 199999 38 us (5.4 TB/s).
extern "C" __global__ __launch_bounds__(SAMPLE_NT) void sepia_sample_max(SampleArgs a) {
    __shared__ unsigned long long wave[SAMPLE_WAVES];
    serve_args<64>();
    const int c = (int)blockIdx.x, row = (int)blockIdx.y;
    const unsigned long long best =
        sample_best(a.logits + (int64_t)row * a.stride, c * a.chunk, min(a.vocab, (c + 1) * a.chunk), wave);
    if (threadIdx.x) return;
    a.bins[(int64_t)row * a.chunks + c].best = best;
    if (c == 0) a.rows[row].n = a.rows[row].arrived = 0;
}

// Grid (chunks, rows): the chunk's bins. 6.8 and 71 us for those, the latter
// bound by the weights' doubles and the sums in shared memory.
extern "C" __global__ __launch_bounds__(SAMPLE_NT) void sepia_sample_bins(SampleArgs a) {
    __shared__ SampleLds L;
    serve_args<64>();
    const int c = (int)blockIdx.x, row = (int)blockIdx.y, tid = (int)threadIdx.x;
    SampleAsk q = sample_ask(a, row);
    if (sample_done(a, row, q, sample_first(a, row, L.wave), c == 0)) return;
    sample_bins(q, c * a.chunk, min(a.vocab, (c + 1) * a.chunk), L);
    SampleChunk *o = a.bins + (int64_t)row * a.chunks + c;
    for (int b = tid; b < SAMPLE_BINS; b += SAMPLE_NT) {
        o->mass[b] = L.mass[b];
        if (q.k > 0) o->count[b] = L.count[b];
    }
    if (tid == 0) o->over_min = q.over_min;
}

// A thread's two bins of the row's chunks added up, eight chunks' loads in
// flight (four: 3.0 us of 13 chunks, as each round of them is one of memory).
template <class T>
__device__ __forceinline__ void sample_add(const SampleChunk *o, int chunks, size_t field, T *to) {
    typedef T Pair __attribute__((ext_vector_type(2)));
    Pair sum = {0, 0};
    for (int i = 0; i < chunks; i += 8) {
        Pair v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = ((const Pair *)((const char *)(o + min(i + j, chunks - 1)) + field))[threadIdx.x];
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (i + j < chunks) sum += v[j];
    }
    to[2 * threadIdx.x] = sum[0];
    to[2 * threadIdx.x + 1] = sum[1];
}

// Grid (chunks, rows): the decision, over the chunks' bins. 10 and 75 us: the
// row read again, then scans, barriers and the last workgroup's decisions.
extern "C" __global__ __launch_bounds__(SAMPLE_NT) void sepia_sample_pick(SampleArgs a) {
    __shared__ SampleLds L;
    serve_args<64>();
    const int c = (int)blockIdx.x, row = (int)blockIdx.y, tid = (int)threadIdx.x;
    SampleAsk q = sample_ask(a, row);
    if (sample_done(a, row, q, sample_first(a, row, L.wave), false)) return;
    const SampleChunk *o = a.bins + (int64_t)row * a.chunks;
    sample_add<unsigned long long>(o, a.chunks, offsetof(SampleChunk, mass), L.mass);
    if (q.k > 0) sample_add<uint32_t>(o, a.chunks, offsetof(SampleChunk, count), L.count);
    if (q.f > 0.0f) {   // a lane a chunk, every wave for itself
        const unsigned long long sum = sample_sums((tid & 63) < a.chunks ? o[tid & 63].over_min : 0);
        q.over_min = sample_lane(sum, 63);
    }
    L.pow.fill();
    const float least = sample_bounds(q, L);
    SampleRow *r = a.rows + row;
    sample_gather(q, least, c * a.chunk, min(a.vocab, (c + 1) * a.chunk), L, r);
    // The gathered tokens cross workgroups as relaxed agent-scope atomics: the
    // wait and the barrier order them before the arrival, the last arriver's
    // loads come after its own (a fence would write back the whole L2).
    const uint32_t n = min(L.n, (uint32_t)SAMPLE_CAP);
    __shared__ uint32_t at;
    if (tid == 0) at = __hip_atomic_fetch_add(&r->n, n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    for (int i = tid; i < (int)n; i += SAMPLE_NT) sample_put(r, at + i, L.list[i]);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (tid == 0) at = __hip_atomic_fetch_add(&r->arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (at + 1 != (uint32_t)a.chunks) return;
    const uint32_t total = __hip_atomic_load(&r->n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (total <= SAMPLE_CAP)
        for (int i = tid; i < (int)total; i += SAMPLE_NT)
            L.list[i] = __hip_atomic_load(&r->list[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();   // a few tokens are compared at once, by every wave
    sample_finish(a, row, q, total, total <= SAMPLE_MANY ? r : nullptr, L);
}

// Grid (1, rows): a row by one workgroup (28 us a call of 11625 logits, its
// batch included).
extern "C" __global__ __launch_bounds__(SAMPLE_NT) void sepia_sample(SampleArgs a) {
    __shared__ SampleLds L;
    serve_args<64>();
    const int row = (int)blockIdx.y;
    SampleAsk q = sample_ask(a, row);
    if (sample_done(a, row, q, sample_best(q.x, 0, a.vocab, L.wave), true)) return;
    sample_bins(q, 0, a.vocab, L);
    const float least = sample_bounds(q, L);
    sample_gather(q, least, 0, a.vocab, L, nullptr);
    const uint32_t n = L.n;
    __syncthreads();   // every wave has it: a decision among few tokens of many uses L.n at once
    sample_finish(a, row, q, n, nullptr, L);
}
