// kv8_attn.h -- attention over the paged 8-bit cache (kv8.h) on the int8
// matrix cores.
//
// Row t of sequence s at position pos sees the columns [max(0, pos - window +
// 1), pos]: score (q . k) c + [pos - col < R] rel[t][h][pos - col] tau[t],
// softmax, weighted v. The codes are operands as they lie in the cache; what
// meets them is split into three signed base-256 digits, 24 bits in all, whose
// products with codes are exact integers:
//   q    relative to the row's largest |q|;
//   p v  each weight times its page's V scale, relative to the largest power
//        of two below the row's largest such product among the step's 64
//        columns (products below 2^-100 are multiples of 2^-122).
// A wave owns 16 rows, each a (token, query head) pair of one kv head, and
// walks the columns in steps of 64:
//   S^T = K q^T   v_mfma_i32_16x16x64_i8, four tiles of 16 columns; row 4 g + i
//         of tile t is column 16 g + 4 t + i of the step, so that lane (n, g)
//         = (lane & 15, lane >> 4) gets columns 16 g .. + 15 of row n: the
//         scales of one page, one run of rel_logits, and the row's softmax
//         in two exchanges between lane groups;
//   O^T = V^T P^T with k = column in the same order, so that the weights'
//         digits are an operand where they are made (no LDS, no exchange) and
//         a dim's 16 columns of a page, side by side in V's layout, the other.
// O stays in registers, f32, per row n: dims 16 ct + 4 g + i.
//
// The type of the call says what a row sees (SEES); every function here is one
// piece of code for all three:
//   Kv8Attn   the window above;
//   Kv8Sinks  the columns below min(sinks, pos + 1) too;
//   Kv8Tree   rows are nodes of a tree of drafted tokens, up to 64 a sequence,
//             whose keys are the columns len, len + 1, .. in the rows' order.
//             Bit j of row i's word, j <= i, says that row j lies on its path.
//             With `before` the bits below i, the row's position is len +
//             popcount(before), it sees cached columns as above and the
//             drafted ones of its path, and column len + j of them lies
//             popcount(before >> j) positions before it: parents come first,
//             so no other row's word is needed.
// A row tile walks the steps that hold the columns below the sinks and the
// steps of its window; the pages between are not read.
#pragma once
#include "kv8.h"

#define KV8_C 8355711.0f     // 0x7F7F7F: the largest magnitude of three digits
#define KV8_CP 4177855.0f    // half of it: a weight's place relative to a power of two
#define KV8_L2E 1.44269504f
#define KV8_LAZY 5.0f        // how far a maximum may rise before the sums are scaled anew

enum { KV8_WINDOW, KV8_SINKS, KV8_TREE };
struct Kv8Attn : Kv8AttnCall {
    static constexpr int SEES = KV8_WINDOW;
};
template <int S>
struct Kv8Masked : Kv8AttnCall {
    static constexpr int SEES = S;
    const uint64_t *tree;
    int32_t sinks;
};
typedef Kv8Masked<KV8_SINKS> Kv8Sinks;
typedef Kv8Masked<KV8_TREE> Kv8Tree;
static_assert(sizeof(Kv8Attn) == sizeof(Kv8AttnCall) && sizeof(Kv8Sinks) == sizeof(Kv8MaskCall), "the host's layout");

typedef int32_t kv8_i4 __attribute__((ext_vector_type(4)));
typedef float kv8_f4 __attribute__((ext_vector_type(4)));
typedef kv8_f4 kv8_f4u __attribute__((aligned(4)));

// Over the four lane groups (lanes n, n + 16, n + 32, n + 48): the halves of
// the rows of 16 lanes change places, then the halves of the wave.
template <class F>
__device__ __forceinline__ float kv8_over_g(float v, F f) {
    const auto a = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    v = f(__builtin_bit_cast(float, (uint32_t)a[0]), __builtin_bit_cast(float, (uint32_t)a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    return f(__builtin_bit_cast(float, (uint32_t)b[0]), __builtin_bit_cast(float, (uint32_t)b[1]));
}
__device__ __forceinline__ float kv8_max_g(float v) {
    return kv8_over_g(v, [](float x, float y) { return fmaxf(x, y); });
}
__device__ __forceinline__ float kv8_sum_g(float v) {
    return kv8_over_g(v, [](float x, float y) { return x + y; });
}

// How a call's work is cut: sequence s has rt row tiles of TT tokens and at
// most `steps` steps of 64 columns in each; a unit (row tile, kv head) is cut
// into `splits` runs of about `chunk` steps, so that the runs of all units are
// about `budget`. Every workgroup works this out for itself from the lengths.
struct Kv8Plan {
    int s, k, hk, x, splits, slot, len, r0, r1;   // slot: of split 0 of the unit (splits > 1); + Hkv a split
};
template <class B>
__device__ __forceinline__ void kv8_cost(const Kv8Args &a, const B &b, int s, int &rt, int &steps, int &len, int &r0,
                                         int &r1) {
    rt = steps = 0;
    if (s >= a.n_seqs || !kv8_seq(a, s, len, r0, r1) || r1 == r0) return;
    if (B::SEES == KV8_TREE && r1 - r0 > KV8_NODES) return;
    rt = (r1 - r0 + b.TT - 1) / b.TT;
    steps = kv8_steps(len + (r1 - r0));
    if constexpr (B::SEES == KV8_WINDOW) {
        if (b.window > 0) steps = min(steps, (int)(((int64_t)b.window + b.TT + 61) / 64) + 1);
    } else if (b.window > 0) {
        const int64_t wide = (int64_t)b.window + (B::SEES == KV8_TREE ? KV8_NODES : b.TT) + 61;
        steps = (int)min((int64_t)steps, wide / 64 + 1 + ((int64_t)b.sinks + 63) / 64);
    }
}
// Inclusive sums over the wave's lanes.
template <class T>
__device__ __forceinline__ T kv8_scan(T v) {
#define KV8_DPP(ctrl, rows, ctl)                                                                                        \
    v += __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), ctrl, rows, 0xF, ctl))
    KV8_DPP(0x111, 0xF, true);    // row_shr 1, 2, 4, 8
    KV8_DPP(0x112, 0xF, true);
    KV8_DPP(0x114, 0xF, true);
    KV8_DPP(0x118, 0xF, true);
    KV8_DPP(0x142, 0xA, false);   // the last lane of a row to the next, of two rows to the next two
    KV8_DPP(0x143, 0xC, false);
#undef KV8_DPP
    return v;
}
template <class T>
__device__ __forceinline__ T kv8_last(T v) {
    return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
// The id-th run in the order sequence, row tile, split, kv head; 0 past the last.
template <class B>
__device__ __forceinline__ int kv8_plan(const Kv8Args &a, const B &b, int id, Kv8Plan &p) {
    const int lane = (int)(threadIdx.x & 63);
    float total = 0.0f, tiles = 0.0f;
    int rt, steps, len, r0, r1;
    for (int s0 = 0; s0 < a.n_seqs; s0 += 64) {
        kv8_cost(a, b, s0 + lane, rt, steps, len, r0, r1);
        total += kv8_last(kv8_scan((float)rt * (float)steps));
        tiles += kv8_last(kv8_scan((float)rt));
    }
    // More tiles than the grid was made for: starts fall somewhere (an error,
    // kv8_check). No run then, since a unit with some of its runs would leave its
    // counter behind.
    if (tiles > (float)(a.n / b.TT + min(a.n, a.n_seqs))) return 0;
    const int chunk = b.budget > 0 ? max(KV8_NW, (int)ceilf(fminf(total * (float)a.Hkv / (float)b.budget, 1e9f))) : 0x7FFFFFFF;
    // A unit of two steps a wave stays whole: the fold takes longer than the
    // second step (32 sequences of up to 500 columns, 8 kv heads: 12.2 us against
    // 9.8).
    const int whole = 2 * KV8_NW;
    p.hk = id % a.Hkv;
    const int at = id / a.Hkv;
    int base = 0, slots = 0;
    for (int s0 = 0; s0 < a.n_seqs; s0 += 64) {
        if (a.n_seqs > 64) kv8_cost(a, b, s0 + lane, rt, steps, len, r0, r1);   // else they are still here
        const int splits = steps <= whole ? 1 : (int)(((int64_t)steps + chunk - 1) / chunk);
        const int mine = rt * splits;
        const int cut = splits > 1 ? rt * splits : 0;
        const int sum = kv8_scan(mine), csum = kv8_scan(cut);
        const uint64_t hit = __ballot(at >= base + sum - mine && at < base + sum);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            p.s = s0 + l;
            p.splits = __builtin_amdgcn_readlane(splits, l);
            const int i = at - base - __builtin_amdgcn_readlane(sum - mine, l);
            p.k = i / p.splits;
            p.x = i - p.k * p.splits;
            p.slot = (slots + __builtin_amdgcn_readlane(csum - cut, l) + p.k * p.splits) * a.Hkv + p.hk;
            p.len = __builtin_amdgcn_readlane(len, l);
            p.r0 = __builtin_amdgcn_readlane(r0, l);
            p.r1 = __builtin_amdgcn_readlane(r1, l);
            return 1;
        }
        base += kv8_last(sum);
        slots += kv8_last(csum);
    }
    return 0;
}

// A row tile's tokens and its steps of 64 columns.
struct Kv8Tile {
    int t0, nt, pos0, lo, last, step0, steps;   // lo, last: the first and last column any row sees
    int span, runs;                             // steps of a run, runs that have any
    // The columns below lo that the rows see, the last of their pages, their steps
    // in front of step0, and the steps between.
    int first, first_page, front, gap;
};
template <class B>
__device__ __forceinline__ Kv8Tile kv8_tile(const Kv8Args &a, const B &b, const Kv8Plan &p, int splits) {
    Kv8Tile t;
    t.t0 = p.r0 + p.k * b.TT;
    t.nt = min(b.TT, p.r1 - t.t0);
    t.pos0 = p.len + p.k * b.TT;
    t.last = t.pos0 + t.nt - 1;
    // of a tree's rows the first stand at len, whatever their places
    t.lo = b.window > 0 ? max(0, (B::SEES == KV8_TREE ? p.len : t.pos0) - b.window + 1) : 0;
    t.step0 = t.lo >> 6;
    t.steps = (t.last >> 6) - t.step0 + 1;
    if constexpr (B::SEES != KV8_WINDOW) {
        t.first = min(b.sinks, t.lo);
        t.first_page = (t.first - 1) >> a.lg;
        t.front = min(((t.first - 1) >> 6) + 1, t.step0);
        t.gap = t.step0 - t.front;
        t.steps += t.front;
    }
    t.span = (t.steps + splits - 1) / splits;
    t.runs = (t.steps + t.span - 1) / t.span;
    return t;
}

// The i-th of a tile's steps.
template <class B>
__device__ __forceinline__ int kv8_step(const Kv8Tile &t, int i) {
    return B::SEES == KV8_WINDOW ? t.step0 + i : i < t.front ? i : i + t.gap;
}

// Row `i` of a tree: its path's rows before it, the rows that it sees, its
// position and the first column in its window. Of a path longer than the window
// it sees the nearest rows, and those at positions below the sinks.
struct Kv8Node {
    uint64_t before, path;
    int32_t pos, lo;
};
template <class B>
__device__ __forceinline__ Kv8Node kv8_node(const B &b, const Kv8Plan &p, int i) {
    const uint64_t word = b.tree[p.r0 + i], own = 1ull << i;
    Kv8Node d;
    d.before = word & (own - 1);
    const int depth = __builtin_popcountll(d.before);
    d.pos = p.len + depth;
    d.lo = b.window > 0 ? max(0, d.pos - b.window + 1) : 0;
    uint64_t near = d.before, rest = d.before;
    if (b.window > 0 && depth >= b.window) {
        for (int k = depth - b.window + 1; k > 0; k--) near &= near - 1;
        for (int k = min(depth, b.sinks - p.len); k > 0; k--) rest &= rest - 1;
        near |= d.before ^ rest;
    }
    d.path = near | (word & own);
    return d;
}
// Whether row `row` of the tile sees no column at all.
template <class B>
__device__ __forceinline__ bool kv8_blank(const Kv8Args &a, const B &b, const Kv8Plan &p, int row) {
    if constexpr (B::SEES != KV8_TREE) return false;
    else {
        const Kv8Node d = kv8_node(b, p, p.k * b.TT + row / (b.H / a.Hkv));
        return d.path == 0 && p.len <= d.lo && min(b.sinks, p.len) <= 0;
    }
}

// Three digit planes of four 24-bit places in the three low bytes of u0..u3
// (the lower two digits offset by 128): planes 0 (low) to 2.
__device__ __forceinline__ void kv8_planes(const uint32_t *u, int32_t &p0, int32_t &p1, int32_t &p2) {
    const uint32_t a = __builtin_amdgcn_perm(u[1], u[0], 0x05010400), b = __builtin_amdgcn_perm(u[3], u[2], 0x05010400);
    const uint32_t c = __builtin_amdgcn_perm(u[1], u[0], 0x0C0C0602), d = __builtin_amdgcn_perm(u[3], u[2], 0x06020C0C);
    p0 = (int32_t)(__builtin_amdgcn_perm(b, a, 0x05040100) ^ 0x80808080u);
    p1 = (int32_t)(__builtin_amdgcn_perm(b, a, 0x07060302) ^ 0x80808080u);
    p2 = (int32_t)(c | d);
}
// hi 65536 + mid 256 + lo of exact sums (|sum| <= 2^21): mid 256 + lo is exact.
// (lo rounded to a multiple of 256 and added into mid's sum by the matrix op
// would save 48 of a step's 520 instructions; it was no faster, and four times
// as far off over 12000 columns.)
__device__ __forceinline__ float kv8_join(int32_t hi, int32_t mid, int32_t lo) {
    return __builtin_fmaf((float)hi, 65536.0f, (float)(int32_t)(((uint32_t)mid << 8) + (uint32_t)lo));
}

// A wave's place for a step's rel_logits; rows 272 bytes apart, so that 16 rows'
// 16-byte pieces lie in different banks.
struct Kv8Rel {
    alignas(16) float at[16][68];
};
// A value that is the same in all lanes, in scalar registers.
__device__ __forceinline__ int64_t kv8_same(int64_t v) {
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)v) |
                     (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32);
}

// One wave's 16 rows of D dims (FULL), or of up to D (a.Dh). NK: K operands a
// row (64 dims each), NC: tiles of 16 dims. LINES: rel_logits by whole rows.
template <class B, int D, bool FULL, bool LINES>
struct Kv8Wave {
    static constexpr int NK = D / 64, NC = D / 16;
    static __device__ __forceinline__ int dh(const Kv8Args &a) { return FULL ? D : a.Dh; }
    kv8_i4 qd[3][NK];       // q's digits: lane (n, g) dims 64 ks + 16 g .. + 15 of row n
    kv8_f4 O[NC];
    // Row n's reference, its maximum or at most KV8_LAZY below; this lane's part
    // of its sum; q's scale times c.
    float m, l, qs, tau;
    int32_t lo, pos;        // row n's columns (inactive: none)
    int64_t th;             // row n's (token, head)
    bool on;                // whether there is a row n
    const float *rel;       // row n's rel_logits
    int32_t rpos, R;        // pos, for an inactive row some active one's; the band
    // LINES: the element of the first row and column 0, the first and the last
    // step whose elements all rows' lie inside the buffer, and this lane's four
    // pieces, bytes behind the first row
    int64_t rel0;
    int32_t rel_s0, rel_s1;
    uint32_t piece[4];
    int32_t lo_max, pos_min;   // over the active rows; of a tree, pos_min is the last cached column
    // Besides the window: the columns below sinks; cached columns end before
    // `end` (inactive: 0), drafted ones begin at `len`, row n's are those of path.
    int32_t sinks, end, len;
    uint64_t before, path;

    __device__ __forceinline__ void init(const Kv8Args &a, const B &b, const Kv8Plan &p, const Kv8Tile &t) {
        const int n = (int)(threadIdx.x & 15), G = b.H / a.Hkv, ti = n / G, hk = p.hk;
        on = ti < t.nt;
        th = (int64_t)(t.t0 + (on ? ti : 0)) * b.H + hk * G + (on ? n - ti * G : 0);
        pos = on ? t.pos0 + ti : -1;
        lo = on ? (b.window > 0 ? max(0, pos - b.window + 1) : 0) : 0x7FFFFFFF;
        tau = b.tau ? b.tau[t.t0 + (on ? ti : 0)] : 1.0f;
        rel = b.rel ? b.rel + th * b.R : nullptr;
        rpos = on ? pos : t.pos0;
        R = b.R;
        if (LINES && b.rel) {
            // elements of the buffer before and behind the tile's first and last
            // row's column 0; a step needs 63 + 64 step of them before
            const int rows = t.nt * G, gi = (rows - 1) % G;
            const int64_t before = ((int64_t)t.t0 * b.H + hk * G) * b.R + t.pos0;
            const int64_t span = ((int64_t)(t.nt - 1) * b.H + gi) * b.R + t.nt - 1;
            const int64_t behind = (int64_t)a.n * b.H * b.R - 1 - before - span;
            rel0 = kv8_same(before);
            rel_s0 = behind >= 0 ? 0 : (int32_t)min((int64_t)0x7FFFFFFF, (63 - behind) >> 6);
            rel_s1 = before < 63 || span > 0x1FFFFFFF ? -1 : (int32_t)min((int64_t)0x7FFFFFFF, (before - 63) >> 6);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int row = 4 * i + ((int)(threadIdx.x & 63) >> 4), r = row < rows ? row : 0, ri = r / G;
                piece[i] = 4u * ((uint32_t)(ri * b.H + r - ri * G) * (uint32_t)b.R + (uint32_t)ri + 4u * (threadIdx.x & 15));
            }
        }
        lo_max = b.window > 0 ? max(0, t.last - b.window + 1) : 0;
        pos_min = t.pos0;
        if constexpr (B::SEES != KV8_WINDOW) {
            sinks = b.sinks;
            end = pos + 1;
        }
        if constexpr (B::SEES == KV8_TREE) {
            const Kv8Node d = kv8_node(b, p, on ? p.k * b.TT + ti : 0);
            len = p.len;
            pos = on ? d.pos : -1;
            lo = on ? d.lo : 0x7FFFFFFF;
            end = on ? len : 0;
            path = on ? d.path : 0;
            before = d.before;
            rpos = d.pos;
            // no row's window begins behind the one of a path of all rows
            lo_max = b.window > 0 ? max(0, len + (p.r1 - p.r0) - b.window) : 0;
            pos_min = len - 1;
        }
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int i = 0; i < NC; i++) O[i] = kv8_f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    // q of row n at dims 64 (i / 4) + 16 g + 4 (i % 4) .. (0 past the rows and Dh).
    __device__ __forceinline__ void load_q(const Kv8Args &a, const B &b, kv8_f4 (&v)[4 * NK]) const {
        const int g = (int)(threadIdx.x & 63) >> 4;
        const float *q = b.q + th * dh(a);
#pragma unroll
        for (int i = 0; i < 4 * NK; i++) {
            const int d = 64 * (i / 4) + 16 * g + 4 * (i % 4);
            v[i] = *(const kv8_f4 *)(q + (FULL || d < a.Dh ? d : 0));
        }
    }
    // Its digits and its scale.
    __device__ __forceinline__ void digits(const Kv8Args &a, const B &b, kv8_f4 (&v)[4 * NK]) {
        const int g = (int)(threadIdx.x & 63) >> 4;
        float most = 0.0f;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < 4 * NK; i++) {
            const bool in = on && (FULL || 64 * (i / 4) + 16 * g < a.Dh);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                v[i][e] = in ? v[i][e] : 0.0f;
                most = fmaxf(most, fabsf(v[i][e]));
                bad |= !(fabsf(v[i][e]) < INFINITY);
            }
        }
        most = kv8_max_g(bad ? INFINITY : most);
        const float inv = most > 0.0f && most < INFINITY ? KV8_C / most : 0.0f;
        qs = most < INFINITY ? most * (b.c / KV8_C) : NAN;
#pragma unroll
        for (int i = 0; i < 4 * NK; i++) {
            uint32_t u[4];
            int32_t p0, p1, p2;
#pragma unroll
            for (int e = 0; e < 4; e++)
                u[e] = (uint32_t)(int32_t)__builtin_rintf(fmaxf(-KV8_C, fminf(KV8_C, v[i][e] * inv))) + 0x8080u;
            kv8_planes(u, p0, p1, p2);
            qd[0][i / 4][i % 4] = p0;
            qd[1][i / 4][i % 4] = p1;
            qd[2][i / 4][i % 4] = p2;
        }
    }

    // The table's entries for a step: of this lane's K row and of its columns
    // 16 g .. . Columns outside [lo, last] of the tile take the nearest page
    // inside. page() checks one when it is used, so that it is not waited for
    // where it is loaded.
    static __device__ __forceinline__ void entries(const Kv8Args &a, const Kv8Plan &p, const Kv8Tile &t, int step, int32_t &ek,
                                                   int32_t &ev) {
        const int lane = (int)(threadIdx.x & 63), first = t.lo >> a.lg, end = t.last >> a.lg;
        const int ik = (64 * step + 16 * ((lane & 15) >> 2)) >> a.lg, iv = (64 * step + 16 * (lane >> 4)) >> a.lg;
        const int32_t *row = a.table + (int64_t)p.s * a.max_pages;
        if constexpr (B::SEES == KV8_WINDOW) {
            ek = row[max(first, min(end, ik))];
            ev = row[max(first, min(end, iv))];
        } else {   // and the columns before the window that are seen
            ek = row[ik <= t.first_page ? ik : max(first, min(end, ik))];
            ev = row[iv <= t.first_page ? iv : max(first, min(end, iv))];
        }
    }
    // Which of a step's columns c0 .. c0 + 15 row n sees, a bit a column.
    __device__ __forceinline__ uint32_t seen(int c0) const {
        const auto below = [&](int x) { return (1u << max(0, min(16, x - c0))) - 1; };
        uint32_t f = below(end) & (~below(lo) | below(sinks));
        if constexpr (B::SEES == KV8_TREE) {
            const int j = c0 - len;   // the first column's row
            f |= (uint32_t)(j >= 0 ? j < KV8_NODES ? path >> j : 0 : j > -16 ? path << -j : 0) & 0xFFFFu;
        }
        return f;
    }
    // How many positions before row n column c0 + j stands, of those that it sees.
    __device__ __forceinline__ int back(int c0, int j) const {
        const int c = c0 + j - len;
        if (B::SEES == KV8_TREE && c >= 0) return __builtin_popcountll(before >> min(c, KV8_NODES - 1));
        return rpos - c0 - j;
    }
    static __device__ __forceinline__ uint32_t page(const Kv8Args &a, int32_t entry) {
        const bool bad = (uint32_t)entry >= (uint64_t)a.n_pages;
        if (__ballot(bad)) sepia_report_error(nullptr, KV8_ERR_PAGE, (int)(threadIdx.x & 63));
        return bad ? 0u : (uint32_t)entry;
    }
    // K operand [t][ks]: column 16 (n >> 2) + 4 t + (n & 3), dims 64 ks + 16 g.
    static __device__ __forceinline__ void load_k(const Kv8Args &a, uint32_t page, int hk, int step, kv8_i4 (&K)[4][NK]) {
        const int lane = (int)(threadIdx.x & 63), n = lane & 15, g = lane >> 4;
        const int slot = (64 * step + 16 * (n >> 2) + (n & 3)) & (a.P() - 1);
        const int8_t *k = a.k_codes(page, hk) + slot * dh(a) + (FULL || 16 * g < dh(a) ? 16 * g : 0);
#pragma unroll
        for (int t = 0; t < 4; t++) {
            K[t][0] = *(const kv8_i4 *)(k + 4 * t * dh(a));
            if constexpr (NK == 2) K[t][1] = *(const kv8_i4 *)(k + 4 * t * dh(a) + (FULL || 64 + 16 * g < dh(a) ? 64 : 0));
        }
    }
    // V operand [ct]: dim 16 ct + n, columns 16 g .. + 15.
    static __device__ __forceinline__ void load_v(const Kv8Args &a, uint32_t page, int hk, int step, kv8_i4 (&V)[NC]) {
        const int lane = (int)(threadIdx.x & 63), n = lane & 15, g = lane >> 4;
        const int8_t *v = a.v_codes(page, hk) + ((int64_t)n << a.lg) + ((64 * step + 16 * g) & (a.P() - 1));
#pragma unroll
        for (int ct = 0; ct < NC; ct++) V[ct] = *(const kv8_i4 *)(v + ((int64_t)(FULL || 16 * ct < dh(a) ? 16 * ct : 0) << a.lg));
    }
    // rel_logits of row n and column 16 g + j of a step, where the row sees the
    // column and its band reaches it, in r[15 - j]. 0: no such column in the
    // step, 1: all are, 2: some are not. (A branch and a load a column, waited
    // for one after the other, were most of a step: 5.5 us.)
    // LINES: a lane's own 16 elements are a quarter of the lines that each load
    // touches, and every line is asked for four times. So the step's 64 elements
    // of each row are loaded side by side, r[4 i + e] being element 4 (lane % 16)
    // + e of row 4 i + lane / 16 (5: all in the bands, 6: not all), and
    // spread_rel() brings them to the lanes that want them: a chunk of 500 rows
    // 115 -> 104 us, of which 22 and 11 for rel_logits. Not where those would lie
    // outside the buffer, nor in the kernels of few rows (16.7 -> 20.4 us at dim
    // 64, whose third wave a SIMD it costs; as long as before at 128).
    __device__ __forceinline__ int load_rel(const B &b, int step, float (&r)[16]) const {
        if (!b.rel || pos_min - (64 * step + 63) >= b.R) return 0;
        const int d0 = rpos - (64 * step + 16 * ((int)(threadIdx.x & 63) >> 4));
        if (LINES && step >= rel_s0 && step <= rel_s1) {
            const char *from = (const char *)(b.rel + (rel0 - 64 * (int64_t)__builtin_amdgcn_readfirstlane(step) - 63));
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const kv8_f4 x = *(const kv8_f4u *)(from + piece[i]);
#pragma unroll
                for (int e = 0; e < 4; e++) r[4 * i + e] = x[e];
            }
            return __ballot(d0 < 15 || d0 >= b.R) == 0 ? 5 : 6;
        }
        const bool drafted = B::SEES == KV8_TREE && 64 * step + 63 >= len;
        if (!drafted && __ballot(d0 < 15 || d0 >= b.R) == 0) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const kv8_f4 x = *(const kv8_f4u *)(rel + (d0 - 15 + 4 * i));
#pragma unroll
                for (int e = 0; e < 4; e++) r[4 * i + e] = x[e];
            }
            return 1;
        }
#pragma unroll
        for (int j = 0; j < 16; j++) r[15 - j] = rel[max(0, min(b.R - 1, drafted ? back(rpos - d0, j) : d0 - j))];
        return 2;
    }
    // r[15 - j] from the pieces, through the wave's own rows of shared memory.
    __device__ __forceinline__ void spread_rel(Kv8Rel &rows) {
        const int lane = (int)(threadIdx.x & 63);
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < 4; i++)
            *(kv8_f4 *)&rows.at[4 * i + (lane >> 4)][4 * (lane & 15)] = kv8_f4{r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]};
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const kv8_f4 x = *(const kv8_f4 *)&rows.at[lane & 15][48 - 16 * (lane >> 4) + 4 * i];
#pragma unroll
            for (int e = 0; e < 4; e++) r[4 * i + e] = x[e];
        }
    }
    // Scores' digit sums of a step.
    __device__ __forceinline__ void dots(const kv8_i4 (&K)[4][NK], float (&s)[16]) const {
#pragma unroll
        for (int t = 0; t < 4; t++) {
            kv8_i4 d[3];
#pragma unroll
            for (int p = 0; p < 3; p++) {
                d[p] = __builtin_amdgcn_mfma_i32_16x16x64_i8(K[t][0], qd[p][0], kv8_i4{0, 0, 0, 0}, 0, 0, 0);
                if constexpr (NK == 2) d[p] = __builtin_amdgcn_mfma_i32_16x16x64_i8(K[t][1], qd[p][1], d[p], 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) s[4 * t + i] = kv8_join(d[2][i], d[1][i], d[0][i]);
        }
    }
    // Scores from their digit sums.
    __device__ __forceinline__ void scores(int step, float (&s)[16], Kv8Rel *rows) {
        const int d0 = rpos - (64 * step + 16 * ((int)(threadIdx.x & 63) >> 4));
        const float sc = qs * ks;
#pragma unroll
        for (int j = 0; j < 16; j++) s[j] *= sc;
        if (LINES && (near & 4)) spread_rel(*rows);
        if (near & 2) {
#pragma unroll
            for (int j = 0; j < 16; j++) r[15 - j] = (B::SEES == KV8_TREE ? back(rpos - d0, j) : d0 - j) < R ? r[15 - j] : 0.0f;
        }
        if (near) {
#pragma unroll
            for (int j = 0; j < 16; j++) s[j] = __builtin_fmaf(r[15 - j], tau, s[j]);
        }
    }
    // The step's softmax and weighted v; vs: the scale of the page of columns
    // 16 g .. .
    __device__ __forceinline__ void step(const Kv8Args &a, int step, float (&s)[16], float vs, const kv8_i4 (&V)[NC]) {
        const int g = (int)(threadIdx.x & 63) >> 4, c0 = 64 * step + 16 * g;
        bool any = true;
        if (64 * step < lo_max || 64 * step + 63 > pos_min) {
            if constexpr (B::SEES == KV8_WINDOW) {
                any = c0 <= pos && c0 + 15 >= lo;
#pragma unroll
                for (int j = 0; j < 16; j++) s[j] = c0 + j >= lo && c0 + j <= pos ? s[j] : -INFINITY;
            } else {
                const uint32_t f = seen(c0);
                any = f != 0;
#pragma unroll
                for (int j = 0; j < 16; j++) s[j] = f >> j & 1 ? s[j] : -INFINITY;
            }
        }
        float mx = s[0];
#pragma unroll
        for (int j = 1; j < 16; j++) mx = fmaxf(mx, s[j]);
        const float mn = fmaxf(m, kv8_max_g(mx));
        if (__ballot(mn > m + KV8_LAZY)) {
            const float al = __builtin_amdgcn_exp2f((m - (mn == -INFINITY ? 0.0f : mn)) * KV8_L2E);   // 1 where the maximum stays
            l *= al;
#pragma unroll
            for (int ct = 0; ct < NC; ct++) O[ct] *= al;
            m = mn;
        }
        const float ref = m == -INFINITY ? 0.0f : m;
        vs = any ? vs : 0.0f;
        // the row's largest product, as the power of two below it
        const float wm = kv8_max_g(__builtin_amdgcn_exp2f((mx - ref) * KV8_L2E) * vs);
        const uint32_t e = max(__builtin_bit_cast(uint32_t, wm) & 0x7F800000u, 27u << 23);
        const float place = fminf(vs * (KV8_CP * __builtin_bit_cast(float, (254u << 23) - e)), 3e38f);
        const float back = __builtin_bit_cast(float, e) * (1.0f / KV8_CP);
        kv8_i4 pd[3];
        float sum = vs * 0.0f;   // a NaN or infinite scale of V makes the row NaN
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint32_t u[4];
            int32_t p0, p1, p2;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float p = __builtin_amdgcn_exp2f((s[4 * i + j] - ref) * KV8_L2E);
                sum += p;
                // 2^23 + 0x8080 + the place: its low bytes are the digits
                u[j] = __builtin_bit_cast(uint32_t, __builtin_fmaf(p, place, 8421504.0f));
            }
            kv8_planes(u, p0, p1, p2);
            pd[0][i] = p0;
            pd[1][i] = p1;
            pd[2][i] = p2;
        }
        l += sum;
#pragma unroll
        for (int ct = 0; ct < NC; ct++) {
            kv8_i4 d[3];
#pragma unroll
            for (int p = 0; p < 3; p++) d[p] = __builtin_amdgcn_mfma_i32_16x16x64_i8(V[ct], pd[p], kv8_i4{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; i++) O[ct][i] = __builtin_fmaf(kv8_join(d[2][i], d[1][i], d[0][i]), back, O[ct][i]);
        }
    }
    // Steps s0, s0 + stride, .. below s1 (of the tile's steps). Loads return in
    // the order they are issued in, and HBM's latency under load is a whole
    // step: a step's K, scales and rel_logits are asked for a step ahead, by
    // table entries that are asked for another step ahead, and its V at its
    // beginning, in the order in which they are waited for.
    kv8_i4 K[4][NK];
    float r[16], ks, vs;     // of the step to come
    int near;
    int32_t ev, nk, nv;      // table entries: V's of that step, both of the next
    __device__ __forceinline__ void ask(const Kv8Args &a, const B &b, const Kv8Plan &p, int step, uint32_t pk, uint32_t pv) {
        load_k(a, pk, p.hk, step, K);
        ks = *a.scale(pv, 0, p.hk);
        vs = *a.scale(pv, 1, p.hk);
        near = load_rel(b, step, r);
    }
    __device__ __forceinline__ void start(const Kv8Args &a, const Kv8Plan &p, const Kv8Tile &t, int s0, int s1, int stride, int32_t &ek) {
        if (s0 >= s1) return;
        entries(a, p, t, kv8_step<B>(t, s0), ek, ev);
        entries(a, p, t, kv8_step<B>(t, min(s0 + stride, s1 - 1)), nk, nv);
    }
    __device__ __forceinline__ void walk(const Kv8Args &a, const B &b, const Kv8Plan &p, const Kv8Tile &t, int s0, int s1,
                                         int stride, int32_t ek, Kv8Rel *rows) {
        if (s0 >= s1) return;
        kv8_f4 q[4 * NK];
        load_q(a, b, q);
        ask(a, b, p, kv8_step<B>(t, s0), page(a, ek), page(a, ev));
        digits(a, b, q);
        for (int i = s0; i < s1; i += stride) {
            const int at = kv8_step<B>(t, i);
            int32_t mk, mv;
            entries(a, p, t, kv8_step<B>(t, min(i + 2 * stride, s1 - 1)), mk, mv);
            kv8_i4 V[NC];
            load_v(a, page(a, ev), p.hk, at, V);
            float s[16];
            dots(K, s);
            scores(at, s, rows);
            const float vs_i = vs;
            if (i + stride < s1) ask(a, b, p, kv8_step<B>(t, i + stride), page(a, nk), page(a, nv));
            step(a, at, s, vs_i, V);
            ev = nv;
            nk = mk;
            nv = mv;
        }
    }
};

// Partials cross workgroups as relaxed agent-scope atomics (kv8_attn_run).
__device__ __forceinline__ void kv8_put(float *p, kv8_f4 v) {
    unsigned long long w[2];
    __builtin_memcpy(w, &v, 16);
    __hip_atomic_store((unsigned long long *)p, w[0], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store((unsigned long long *)p + 1, w[1], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ kv8_f4 kv8_get(const float *p) {
    kv8_f4 v;
    unsigned long long w[2];
    w[0] = __hip_atomic_load((const unsigned long long *)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    w[1] = __hip_atomic_load((const unsigned long long *)p + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __builtin_memcpy(&v, w, 16);
    return v;
}
__device__ __forceinline__ float *kv8_out(const Kv8Args &a, const Kv8AttnCall &b, const Kv8Plan &p, const Kv8Tile &t, int n) {
    const int G = b.H / a.Hkv, ti = n / G;
    return b.out + ((int64_t)(t.t0 + ti) * b.H + p.hk * G + (n - ti * G)) * a.Dh;
}
#define KV8_AHEAD 8   // partials whose loads are in flight at a time
#define KV8_RUNS 16   // of a unit that are folded at once; more are folded in groups first

// Row `row`'s dims d .. d + 3 of n partials, `step` places apart from place `at`
// on: the sums so far, relative to their maximum.
struct Kv8Sum {
    float top, sum;
    kv8_f4 o;
};
__device__ __forceinline__ Kv8Sum kv8_fold(const Kv8Args &a, const Kv8AttnCall &b, int64_t at, int n, int step, int row, int d) {
    Kv8Sum r = {-INFINITY, 0.0f, {0.0f, 0.0f, 0.0f, 0.0f}};
    for (int x0 = 0; x0 < n; x0 += KV8_AHEAD) {
        kv8_f4 v[KV8_AHEAD];
        float vm[KV8_AHEAD], vl[KV8_AHEAD], mx = r.top;
#pragma unroll
        for (int j = 0; j < KV8_AHEAD; j++) {
            const int64_t i = at + (int64_t)min(x0 + j, n - 1) * step;
            v[j] = kv8_get(b.part + (i * 16 + row) * a.Dh + d);
            vm[j] = __hip_atomic_load(&b.ml[i * 32 + row], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            vl[j] = __hip_atomic_load(&b.ml[i * 32 + 16 + row], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
#pragma unroll
        for (int j = 0; j < KV8_AHEAD; j++) mx = fmaxf(mx, vm[j]);
        const float from = mx == -INFINITY ? 0.0f : mx, al = __builtin_amdgcn_exp2f((r.top - from) * KV8_L2E);
        r.sum *= al;
        r.o *= al;
        r.top = mx;
#pragma unroll
        for (int j = 0; j < KV8_AHEAD; j++) {
            const float e = x0 + j < n ? __builtin_amdgcn_exp2f((vm[j] - from) * KV8_L2E) : 0.0f;
            if (x0 + j < n) {
                r.sum += vl[j] * e;
                r.o += v[j] * e;
            }
        }
    }
    return r;
}
// Whether this workgroup is the last of n to arrive; the counter is zero again
// then. What crosses workgroups are relaxed agent-scope atomics: the wait and
// the barrier order the stores before the arrival, and the last arriver's loads
// come after its own (a release fence would write back the whole L2).
__device__ __forceinline__ bool kv8_arrive(uint32_t *counter, int n) {
    __shared__ uint32_t before;
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0) before = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (before + 1 != (uint32_t)n) return false;
    if (threadIdx.x == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return true;
}

// Grid: the plan's runs, KV8_NW waves each (U = 2: two units that are not cut a
// workgroup, half as many waves each). Bound by memory for long contexts
// (48 sequences of 278000 columns in all, 8 kv heads of 128: 118.5 us, 4.9 TB/s),
// else by the chain from the plan to the fold: one sequence of 20000 columns
// 17.5 us, 32 in a window of 512 18.5 us (16 kv heads). A tree of 25 rows behind
// 20001 columns (64 heads on 8) 70 us, of 13 row tiles a kv head; 24 trees of 502
// rows behind 58900 columns 183 us. Two units a workgroup: 9 trees of 377 rows in a
// window of 300 17.9 us (dim 64, 32 heads on 8), 40 sequences in a window of 512
// behind 4 sinks 25.4 us (64 heads on 16). The trees behind long contexts are bound by
// VALU and matrix instructions that a wave issues in turn (54 and 18% of SIMD cycles),
// at two waves a SIMD; the pairs by latency: VALU 27-42%, 40% of wave cycles waiting,
// 1.0-1.3 waves a SIMD on average. Registers: 224 and more above dim 64, where two waves
// a SIMD fit; up to 64 the ones of sinks in pairs 165 and 167, where a third fits (168),
// cut into runs 169 and 170, trees' 170 to 174.
template <int D, bool FULL, int U, class B>
__device__ __forceinline__ void kv8_attn_run(const Kv8Args &a, const B &b) {
    constexpr int NW = KV8_NW / U;   // waves of a unit
    typedef Kv8Wave<B, D, FULL, false> Wave;
    __shared__ kv8_f4 so[KV8_NW][Wave::NC][64];
    __shared__ float sm[KV8_NW][16], sl[KV8_NW][16];
    serve_args<128>();
    kv8_check(a, B::SEES == KV8_TREE ? KV8_NODES : 0x7FFFFFFF);
    Kv8Plan p;
    int w0 = 0;   // the unit's first wave
    bool have = true;
    if constexpr (U == 1) {
        if (!kv8_plan(a, b, (int)blockIdx.x, p)) return;
    } else {   // waves without a unit keep the others company
        const int unit = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) / NW;
        w0 = unit * NW;
        have = kv8_plan(a, b, (int)blockIdx.x * U + unit, p);
        if (!have) p.s = p.k = p.hk = p.x = p.slot = p.len = p.r0 = p.r1 = 0, p.splits = 1;
    }
    const Kv8Tile t = kv8_tile(a, b, p, p.splits);
    const int s0 = p.x * t.span, s1 = min(t.steps, s0 + t.span);
    if (U == 1 && s0 >= s1) return;
    const int w = ((int)threadIdx.x >> 6) - w0, lane = (int)threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    Wave W;
    int32_t ek;
    if (U == 1 || have) {
        W.start(a, p, t, s0 + w, s1, NW, ek);
        W.init(a, b, p, t);
        W.walk(a, b, p, t, s0 + w, s1, NW, ek, nullptr);
        const float l = kv8_sum_g(W.l);
        if (g == 0) {
            sm[w0 + w][n] = W.m;
            sl[w0 + w][n] = l;
        }
#pragma unroll
        for (int ct = 0; ct < Wave::NC; ct++) so[w0 + w][ct][lane] = W.O[ct];
    }
    __syncthreads();
    if (U > 1 && !have) return;
    // fold the waves: wave w takes dims 16 ct .. of ct = w, w + NW
    float M = -INFINITY, f[NW], L = 0.0f;
#pragma unroll
    for (int i = 0; i < NW; i++) M = fmaxf(M, sm[w0 + i][n]);
    const float ref = M == -INFINITY ? 0.0f : M;
#pragma unroll
    for (int i = 0; i < NW; i++) {
        f[i] = __builtin_amdgcn_exp2f((sm[w0 + i][n] - ref) * KV8_L2E);
        L += sl[w0 + i][n] * f[i];
    }
    const int64_t slot = p.slot + (int64_t)p.x * a.Hkv;
    const int rows = t.nt * (b.H / a.Hkv);
    if (n < rows) {
        const float by = B::SEES == KV8_TREE && L == 0.0f && kv8_blank(a, b, p, n) ? 1.0f : L;   // a row that sees nothing: 0
        float *out = kv8_out(a, b, p, t, n);
        for (int ct = w; 16 * ct < a.Dh; ct += NW) {
            kv8_f4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < NW; i++) o += so[w0 + i][ct][lane] * f[i];
            if (t.runs > 1) kv8_put(b.part + (slot * 16 + n) * a.Dh + 16 * ct + 4 * g, o);
            else *(kv8_f4 *)(out + 16 * ct + 4 * g) = o / by;
        }
    }
    if (U > 1 || t.runs == 1) return;
    if (w == 0 && g == 0) {
        __hip_atomic_store(&b.ml[slot * 32 + n], M, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(&b.ml[slot * 32 + 16 + n], L, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    // The last of a unit's runs to arrive folds them, in their order. Of many
    // the last of each group folds the group's to its first run's place, and the
    // last of those the groups': two short chains of loads for a long one (one
    // sequence of 20000 columns, 63 runs of a unit: 16.8 us against 18.3 and a
    // gap with a fold by a launch, 25 by one workgroup; at 16 runs one is as fast).
    const int per = a.Dh / 4;
    int n_part = t.runs, step = a.Hkv;
    uint32_t *counter = b.arrived + p.slot;
    if (t.runs > KV8_RUNS) {
        int lg = 3;
        while (t.runs > 1 << (2 * lg)) lg++;
        const int x0 = p.x >> lg << lg, n = min(1 << lg, t.runs - x0);
        const int64_t at = p.slot + (int64_t)x0 * a.Hkv;
        if (!kv8_arrive(b.arrived + at, n)) return;
        for (int i = (int)threadIdx.x; i < rows * per; i += 64 * KV8_NW) {
            const int row = i / per, d = 4 * (i - row * per);
            const Kv8Sum r = kv8_fold(a, b, at, n, a.Hkv, row, d);
            kv8_put(b.part + (at * 16 + row) * a.Dh + d, r.o);
            if (d == 0) sm[0][row] = r.top, sl[0][row] = r.sum;
        }
        __syncthreads();   // every thread has read the group's maxima and sums
        if ((int)threadIdx.x < rows) {
            __hip_atomic_store(&b.ml[at * 32 + threadIdx.x], sm[0][threadIdx.x], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(&b.ml[at * 32 + 16 + threadIdx.x], sl[0][threadIdx.x], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        n_part = (t.runs + (1 << lg) - 1) >> lg;
        step = a.Hkv << lg;
        counter += KV8_UNITS;
    }
    if (!kv8_arrive(counter, n_part)) return;
    for (int i = (int)threadIdx.x; i < rows * per; i += 64 * KV8_NW) {
        const int row = i / per, d = 4 * (i - row * per);
        const Kv8Sum r = kv8_fold(a, b, p.slot, n_part, step, row, d);
        const float by = B::SEES == KV8_TREE && r.sum == 0.0f && kv8_blank(a, b, p, row) ? 1.0f : r.sum;
        *(kv8_f4 *)(kv8_out(a, b, p, t, row) + d) = r.o / by;
    }
}

// Many rows (prompts): a wave a unit, KV8_NW row tiles of one kv head side by
// side in a workgroup, so that they find K and V in the caches; nothing is cut
// or folded. 2.6 us a step and pair of waves of a SIMD at dim 128; the loads alone
// take 2.2, all but the loads 2.4, all but the matrix products 2.5. 500 rows
// behind 1500 (64 heads on 8) 98 us. (K and V loaded once for the four and put
// in shared memory: 2.8 us a step; that in steps of 128 columns: spills.) Grid: (ids of KV8_NW row tiles, kv heads), kv heads fastest, so
// that with 8 of them an XCD's L2 holds one head's K and V.
template <int D, bool FULL, int U, class B>
__device__ __forceinline__ void kv8_attn_rows(const Kv8Args &a, const B &b) {
    typedef Kv8Wave<B, D, FULL, B::SEES != KV8_TREE> Wave;
    __shared__ Kv8Rel rel[KV8_NW];
    serve_args<128>();
    kv8_check(a, B::SEES == KV8_TREE ? KV8_NODES : 0x7FFFFFFF);
    Kv8Plan p;
    const int id = (int)blockIdx.x / a.Hkv, gran = KV8_NW * b.TT;
    p.hk = (int)blockIdx.x - id * a.Hkv;
    p.s = kv8_find(a, id, gran, 1, p.k, p.len, p.r0, p.r1);
    if (p.s < 0 || (B::SEES == KV8_TREE && p.r1 - p.r0 > KV8_NODES)) return;
    p.k = p.k * KV8_NW + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    if ((int64_t)p.k * b.TT >= p.r1 - p.r0) return;
    const Kv8Tile t = kv8_tile(a, b, p, 1);
    const int lane = (int)threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    Wave W;
    int32_t ek;
    W.start(a, p, t, 0, t.steps, 1, ek);
    W.init(a, b, p, t);
    W.walk(a, b, p, t, 0, t.steps, 1, ek, &rel[threadIdx.x >> 6]);
    const float l = kv8_sum_g(W.l);
    if (n >= t.nt * (b.H / a.Hkv)) return;
    const float inv = B::SEES == KV8_TREE && l == 0.0f && kv8_blank(a, b, p, n) ? 0.0f : 1.0f / l;   // sees nothing: 0
    float *o = kv8_out(a, b, p, t, n) + 4 * g;
#pragma unroll
    for (int ct = 0; ct < Wave::NC; ct++)
        if (FULL || 16 * ct < a.Dh) *(kv8_f4 *)(o + 16 * ct) = W.O[ct] * inv;
}

#define KV8_KERNEL(name, run, U, B, D, FULL) \
    extern "C" __global__ __launch_bounds__(64 * KV8_NW, 2) void name(Kv8Args a, B b) { run<D, FULL, U>(a, b); }
#define KV8_KERNEL4(name, run, U, B)           \
    KV8_KERNEL(name##_128, run, U, B, 128, true)    \
    KV8_KERNEL(name##_to128, run, U, B, 128, false) \
    KV8_KERNEL(name##_64, run, U, B, 64, true)      \
    KV8_KERNEL(name##_to64, run, U, B, 64, false)
#ifdef KV8_KERNELS
KV8_KERNEL4(sepia_kv8_attn, kv8_attn_run, 1, Kv8Attn)
KV8_KERNEL4(sepia_kv8_rows, kv8_attn_rows, KV8_NW, Kv8Attn)
#endif
