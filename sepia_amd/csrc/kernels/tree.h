// tree.h -- what a target accepts of trees of drafted tokens (kv8_attn.h's
// words), and the paged 8-bit cache (kv8.h) made to follow it.
#pragma once
#include "kv8.h"

// ------------------------------------------------------------- accept ------
// Row 0 of a sequence is kept. Below a kept row the lowest child is kept that
// was drafted with the row's sampled token; a child of row p is a row whose
// path's rows before it are p's and p. One wave a sequence, lane i its row i:
// a level is a ballot, at most 63 of them. Bound by the launch and two dependent
// loads: 4.0-4.3 us by events around the launch, for one sequence as for 250 of 7072
// rows (2.5 in a trace, which leaves the launch out).
extern "C" __global__ __launch_bounds__(64) void sepia_tree_accept(TreeCall a) {
    serve_args<64>();
    const int s = (int)blockIdx.x, i = (int)threadIdx.x;
    const int32_t r0 = a.starts[s], r1 = a.starts[s + 1], m = r1 - r0;
    if (r0 < 0 || r1 < r0 || r1 > a.n || m > KV8_NODES) {
        sepia_report_error(nullptr, KV8_ERR_SEQ, i);
        return;
    }
    if (m == 0) {
        if (i == 0) a.counts[s] = 0, a.next[s] = -1;
        return;
    }
    const int row = r0 + min(i, m - 1);
    const uint64_t before = a.tree[row] & ((1ull << i) - 1);
    const int32_t token = a.drafted[row], sampled = a.sampled[row];
    uint64_t kept = 1, path = 1;   // kept: the rows so far; path: the last one's children's rows before them
    int at = 0;
    int32_t wanted = __builtin_amdgcn_readlane(sampled, 0);
    while (true) {
        const uint64_t hit = __ballot(i > at && i < m && before == path && token == wanted && wanted >= 0);
        if (!hit) break;
        at = __builtin_ctzll(hit);
        wanted = __builtin_amdgcn_readlane(sampled, at);
        kept |= 1ull << at;
        path |= 1ull << at;
    }
    const int n = __builtin_popcountll(kept);
    if (kept >> i & 1) a.kept[r0 + __builtin_popcountll(kept & ((1ull << i) - 1))] = i;
    if (i >= n && i < m) a.kept[r0 + i] = -1;
    if (i == 0) a.counts[s] = n, a.next[s] = wanted;
}

// --------------------------------------------------------------- keep ------
// The cache's position len + i takes what position len + kept[i] holds. A page
// that a row moves to gets the largest of its tokens' scales as its scale, so
// that no code grows; codes become rint(c old / new), the quotient and the
// product in double. kept rises, so every row moves down or stays.
// Unit: (sequence, kv head, K or V), a workgroup. All loads of the unit are done
// before its first store. K moves by 16 dims of a token; V, whose tokens lie
// side by side, by 16 slots of a dim, into which the moved tokens' bytes are
// gathered. Bound by a chain of five dependent loads (the sequence, kept, the
// table, scales, codes): 4.4 us for one sequence of 25 rows (8 kv heads of 128), 8.3
// for 61 of 1145 (16 kv heads, 1952 workgroups in one round).
#define KEEP_NT 256
struct KeepRow {
    int32_t page, slot;   // where the token lies
    double ratio;         // its scale over its page's to come
};
extern "C" __global__ __launch_bounds__(KEEP_NT) void sepia_kv8_keep(Kv8Args a, const int32_t *__restrict__ kept) {
    __shared__ KeepRow from[2 * KV8_NODES];   // of the positions from the first page's beginning on
    __shared__ int32_t to[8];                 // the pages, by their order
    serve_args<64>();
    kv8_check(a, KV8_NODES);
    const int lane = (int)threadIdx.x & 63, hk = (int)blockIdx.y, side = (int)blockIdx.z;
    int32_t k_unit = 0, len, r0, r1;
    int s = (int)blockIdx.x;
    if (a.extra) {   // ids are sequences
        if (!kv8_seq(a, s, len, r0, r1)) return;
    } else {
        s = kv8_find(a, blockIdx.x, a.gran, 0, k_unit, len, r0, r1);
        if (s < 0 || k_unit) return;
    }
    const int m = r1 - r0;
    if (m < 1 || m > KV8_NODES) return;
    const int32_t src = lane < m ? kept[r0 + lane] : -1;
    const uint64_t none = __ballot(src < 0);
    const int count = none ? __builtin_ctzll(none) : 64;
    const int32_t last = __shfl_up(src, 1);
    if (__ballot(lane < count && (src >= m || (lane > 0 && src <= last)))) {
        sepia_report_error(nullptr, KV8_ERR_SEQ, (int)threadIdx.x);
        return;
    }
    const uint64_t moved = __ballot(lane < count && src != lane);
    if (!moved) return;
    const int first = __builtin_ctzll(moved);   // rows before it stay where they are
    const int page0 = (len + first) >> a.lg, base = page0 << a.lg, P = a.P();
    const int end = len + count, pages = ((end - 1) >> a.lg) - page0 + 1;   // at most 5
    // rows in front of page0 take part in nothing
    const bool mine = lane < count && len + lane >= base;
    const int here = mine ? ((len + lane) >> a.lg) - page0 : -1;
    const int page_to = kv8_page(a, s, mine ? page0 + here : page0);
    const int page_from = kv8_page(a, s, mine ? (len + src) >> a.lg : page0);
    if (__ballot(page_to < 0 || page_from < 0)) {
        sepia_report_error(nullptr, KV8_ERR_PAGE, (int)threadIdx.x);
        return;
    }
    const float old = *a.scale(__builtin_amdgcn_readfirstlane(kv8_page(a, s, page0)), side, hk);   // of the first page
    const float scale = *a.scale(page_from, side, hk);
    float now[5] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f}, target = 1.0f;
#pragma unroll
    for (int j = 0; j < 5; j++) {
        if (j >= pages) break;
        const bool in = here == j;
        now[j] = kv8_wave_max(in ? scale : 0.0f);
        if (j == 0 && base < len) now[0] = fmaxf(now[0], old);
        if (__ballot(in && scale != scale) || (j == 0 && base < len && old != old)) now[j] = NAN;
        if (in) target = now[j];
    }
    // 1 where the scale stays, or is none
    const auto ratio = [](float s, float n) { return s < n && n < INFINITY ? (double)s / (double)n : 1.0; };
    // the tokens of the first page that stay where they are, when its scale changes
    const bool again = now[0] != old && len + first > base;
    if (threadIdx.x < 64) {
        const int held = len - base;   // the cached tokens of the first page
        if (held > 0 && lane < held) from[lane] = KeepRow{kv8_page(a, s, page0), lane, ratio(old, now[0])};
        if (mine) from[len + lane - base] = KeepRow{page_from, (len + src) & (P - 1), ratio(scale, target)};
        if (mine && ((len + lane) & (P - 1)) == 0) to[here] = page_to;
        if (lane == 0) to[0] = kv8_page(a, s, page0);
    }
    __syncthreads();
    // positions from base on that change
    const int n = end - base, begin = again ? 0 : len + first - base;
    uint4 got[4];
    if (side == 0) {
        const int pieces = a.Dh / 16;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int item = (int)threadIdx.x + i * KEEP_NT + begin * pieces;
            if (item >= n * pieces) continue;
            const KeepRow f = from[item / pieces];
            const uint4 x = *(const uint4 *)(a.k_codes(f.page, hk) + f.slot * a.Dh + 16 * (item % pieces));
            got[i] = f.ratio == 1.0 ? x : make_uint4(kv8_again(x.x, f.ratio), kv8_again(x.y, f.ratio), kv8_again(x.z, f.ratio), kv8_again(x.w, f.ratio));
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int item = (int)threadIdx.x + i * KEEP_NT + begin * pieces;
            if (item >= n * pieces) continue;
            const int t = item / pieces;
            *(uint4 *)(a.k_codes(to[t >> a.lg], hk) + (t & (P - 1)) * a.Dh + 16 * (item % pieces)) = got[i];
        }
    } else {
        const int p0 = begin / 16, p1 = (n + 15) / 16;   // pieces of 16 slots of a dim
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int item = (int)threadIdx.x + i * KEEP_NT;
            if (item >= (p1 - p0) * a.Dh) continue;
            const int d = item % a.Dh, t0 = 16 * (p0 + item / a.Dh);
            const uint4 was = *(const uint4 *)(a.v_codes(to[t0 >> a.lg], hk) + ((int64_t)d << a.lg) + (t0 & (P - 1)));
            uint32_t w[4] = {was.x, was.y, was.z, was.w};
#pragma unroll
            for (int j = 0; j < 16; j++) {
                if (t0 + j < begin || t0 + j >= n) continue;
                const KeepRow f = from[t0 + j];
                const int8_t c = a.v_codes(f.page, hk)[((int64_t)d << a.lg) + f.slot];
                const uint32_t r = (uint32_t)(int32_t)__builtin_rint((double)c * f.ratio) & 0xFFu;
                w[j / 4] = (w[j / 4] & ~(0xFFu << (8 * (j % 4)))) | r << (8 * (j % 4));
            }
            got[i] = make_uint4(w[0], w[1], w[2], w[3]);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int item = (int)threadIdx.x + i * KEEP_NT;
            if (item >= (p1 - p0) * a.Dh) continue;
            const int d = item % a.Dh, t0 = 16 * (p0 + item / a.Dh);
            *(uint4 *)(a.v_codes(to[t0 >> a.lg], hk) + ((int64_t)d << a.lg) + (t0 & (P - 1))) = got[i];
        }
    }
    if (threadIdx.x < 64) {
#pragma unroll
        for (int j = 0; j < 5; j++)
            if (j < pages && lane == j) *a.scale(to[j], side, hk) = now[j];
    }
}
