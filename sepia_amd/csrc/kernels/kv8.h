// kv8.h -- a paged key/value cache held in 8 bits: its layout, appending to it
// and reading it back (attention over it: kv8_attn.h).
//
// Page p of the pool holds P tokens (16, 32 or 64) of every kv head: K codes
// int8 [head][token][dim], then V codes int8 [head][dim][token], and a scale
// f32 [K, V][head]; a cached value is code * scale. A table row gives a
// sequence's pages in order.
//
// Appending new rows to a page (unit: page, K or V, head): with y the row's
// values (K with norm weights w: x w / sqrt(mean(x^2) + eps)) and a the
// largest |y|, the scale becomes max(old scale, a (1 / 127)) (no old scale
// where the unit begins at the page's first token); if it grew, the codes before the
// unit become rint(c old / new); the new codes are rint(y / scale), at most
// 127 in magnitude. Norms, quotients and roundings are double, so that a code
// next to a rounding border does not depend on the order of a sum; a, 1 / 127
// and their product are rounded to f32. A value that is not finite makes
// the scale NaN, and with it every value of the unit's page and head.
#pragma once
#include "common.h"
#include "kv8_map.h"

#define KV8_ERR_PAGE 6u   // device error: a page of the table outside the pool
#define KV8_ERR_SEQ 7u    // device error: lens or starts that do not fit the call

// What every kernel is given (the host's struct in serve.c mirrors it).
struct Kv8Args {
    int8_t *codes;
    float *scales;
    const int32_t *table, *lens, *starts;
    int64_t n_pages;
    int32_t n_seqs, max_pages, Hkv, Dh, lg, n;   // n: rows of the call
    uint32_t head_bytes, page_bytes;             // of a head's K or V in a page, of a page
    __device__ __forceinline__ int P() const { return 1 << lg; }
    __device__ __forceinline__ int8_t *k_codes(uint32_t page, int hk) const {
        return codes + (uint64_t)hk * head_bytes + (uint64_t)page * page_bytes;
    }
    __device__ __forceinline__ int8_t *v_codes(uint32_t page, int hk) const {
        return codes + (uint64_t)(Hkv + hk) * head_bytes + (uint64_t)page * page_bytes;
    }
    __device__ __forceinline__ float *scale(uint32_t page, int side, int hk) const {
        return scales + (side * Hkv + hk) + (uint64_t)page * (2u * (uint32_t)Hkv);
    }
};

// That sequence's length and rows; 0 where they cannot be used.
__device__ __forceinline__ int kv8_seq(const Kv8Args &a, int s, int32_t &len, int32_t &r0, int32_t &r1) {
    len = a.lens[s];
    r0 = a.starts[s];
    r1 = a.starts[s + 1];
    return kv8_seq_ok(len, r0, r1, a.n, (int64_t)a.max_pages << a.lg);
}
// The sequence that owns `id`, its length and rows; -1 if there is none, or
// one that cannot be used. 64 sequences a look: one round for up to 64 of
// them, with everything about the one found already loaded, two for 4096.
__device__ __forceinline__ int kv8_find(const Kv8Args &a, int64_t id, int gran, int extra, int32_t &len, int32_t &r0, int32_t &r1) {
    const int lane = (int)(threadIdx.x & 63);
    int lo = 0, n = a.n_seqs;
    while (true) {
        const int step = (n + 63) / 64, i = lane * step, s = lo + min(i, n - 1);
        r0 = a.starts[s];
        r1 = a.starts[s + 1];
        len = a.lens[s];
        const int c = __builtin_popcountll(__ballot(i < n && kv8_first_id(r0, s, gran, extra) <= id));
        if (c == 0) return -1;
        if (step == 1) {
            r0 = __builtin_amdgcn_readlane(r0, c - 1);
            r1 = __builtin_amdgcn_readlane(r1, c - 1);
            len = __builtin_amdgcn_readlane(len, c - 1);
            return kv8_seq_ok(len, r0, r1, a.n, (int64_t)a.max_pages << a.lg) ? lo + c - 1 : -1;
        }
        lo += (c - 1) * step;
        n = min(step, n - (c - 1) * step);
    }
}
// The grid's last workgroup reports sequences that cannot be used (others
// pass them over, or, where starts fall, may not find them at all). It is the
// last since that seldom has anything else to do.
__device__ __forceinline__ void kv8_check(const Kv8Args &a) {
    if (blockIdx.x + 1 != gridDim.x || blockIdx.y || blockIdx.z) return;
    bool bad = false;
    int32_t len, r0, r1;
    for (int s = (int)threadIdx.x; s < a.n_seqs; s += (int)blockDim.x) bad |= !kv8_seq(a, s, len, r0, r1);
    if (bad) sepia_report_error(nullptr, KV8_ERR_SEQ, 0);
}
// The pool's page of entry `i` of a sequence's table row, -1 if it has none.
__device__ __forceinline__ int kv8_page(const Kv8Args &a, int s, int i) {
    const int32_t p = a.table[(int64_t)s * a.max_pages + i];
    return (uint32_t)p < (uint64_t)a.n_pages ? p : -1;
}

// ------------------------------------------------------------- append ------
__device__ __forceinline__ uint32_t kv8_code(double y, double inv) {
    const double c = __builtin_rint(y * inv);
    return (uint32_t)(int32_t)__builtin_fmax(-127.0, __builtin_fmin(127.0, c)) & 0xFFu;
}
__device__ __forceinline__ uint32_t kv8_again(uint32_t word, double ratio) {
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < 4; i++)
        r |= ((uint32_t)(int32_t)__builtin_rint((double)(int8_t)(word >> (8 * i)) * ratio) & 0xFFu) << (8 * i);
    return r;
}

// The unit's scale from each wave's largest value (bad: one is not finite),
// and what its codes are multiplied with: the new rows' 1 / scale, the old
// codes' old / new (1 where the scale did not grow).
struct Kv8Scale {
    double inv, ratio;
};
__device__ __forceinline__ Kv8Scale kv8_rescale(float *scale, bool fresh, float most, bool bad) {
    __shared__ float red[4];
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) most = fmaxf(most, __shfl_xor(most, o, 64));
    if (__ballot(bad)) most = INFINITY;
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = most;
    const float old = fresh ? 0.0f : *scale;
    __syncthreads();   // every wave has the old scale, and the maxima
    for (unsigned w = 0; w < blockDim.x / 64; w++) most = fmaxf(most, red[w]);
    float s = fmaxf(old, most * (1.0f / 127.0f));
    if (!(s < INFINITY) || old != old) s = NAN;
    if (threadIdx.x == 0) *scale = s;
    Kv8Scale r;
    r.inv = s > 0.0f ? 1.0 / (double)s : 0.0;
    r.ratio = s > old && old > 0.0f ? (double)old / (double)s : 1.0;
    return r;
}

// Grid (ids, Hkv, 2: K and V), a wave for each 16 tokens of a page; gran = P,
// extra = 2.
extern "C" __global__ __launch_bounds__(256, 4) void sepia_kv8_append(Kv8Args a, const float *__restrict__ k,
                                                                   const float *__restrict__ v,
                                                                   const float *__restrict__ norm, float eps) {
    const int hk = (int)blockIdx.y, lane = (int)(threadIdx.x & 63), slot0 = (int)(threadIdx.x >> 6) * 16;
    kv8_check(a);
    int32_t len, r0, r1;
    const int s = kv8_find(a, blockIdx.x, a.P(), 2, len, r0, r1);
    Kv8Unit u;
    if (s < 0) return;
    if (!kv8_unit(len, r0, r1, (int)(blockIdx.x - kv8_first_id(r0, s, a.P(), 2)), a.lg, &u)) return;
    const int page = kv8_page(a, s, u.page);
    if (page < 0) {
        sepia_report_error(nullptr, KV8_ERR_PAGE, (int)threadIdx.x);
        return;
    }
    const int64_t ld = (int64_t)a.Hkv * a.Dh;
    float most = 0.0f;
    bool bad = false;
    if (blockIdx.z == 0) {
        // K: 8 lanes a token, 8 tokens a pass; lane j of a token holds dims
        // 32 i + 4 j .. + 3, so that every access of the eight is a whole line
        const int j = lane & 7;
        float x[2][16], w[16];
        double rms[2];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int d = 32 * i + 4 * j;
            float4 t = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
            if (norm && d < a.Dh) t = *(const float4 *)(norm + d);
            w[4 * i] = t.x, w[4 * i + 1] = t.y, w[4 * i + 2] = t.z, w[4 * i + 3] = t.w;
        }
#pragma unroll
        for (int p = 0; p < 2; p++) {
            const int slot = slot0 + 8 * p + (lane >> 3);
            const bool on = slot >= u.s0 && slot < u.s1;
            const float *row = k + (int64_t)(u.row + (on ? slot - u.s0 : 0)) * ld + (int64_t)hk * a.Dh;
            double ss = 0.0;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int d = 32 * i + 4 * j;
                float4 t = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (on && d < a.Dh) t = *(const float4 *)(row + d);
                x[p][4 * i] = t.x, x[p][4 * i + 1] = t.y, x[p][4 * i + 2] = t.z, x[p][4 * i + 3] = t.w;
#pragma unroll
                for (int c = 0; c < 4; c++) ss = __builtin_fma((double)x[p][4 * i + c], (double)x[p][4 * i + c], ss);
            }
#pragma unroll
            for (int o = 1; o <= 4; o <<= 1) ss += __shfl_xor(ss, o, 64);
            rms[p] = norm ? 1.0 / __builtin_sqrt(ss / a.Dh + (double)eps) : 1.0;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const float y = on ? (float)((double)x[p][i] * rms[p] * (double)w[i]) : 0.0f;
                most = fmaxf(most, fabsf(y));
                bad |= !(fabsf(y) < INFINITY);
            }
        }
        const Kv8Scale sc = kv8_rescale(a.scale(page, 0, hk), u.s0 == 0, most, bad);
        int8_t *c0 = a.k_codes(page, hk);
#pragma unroll
        for (int p = 0; p < 2; p++) {
            const int slot = slot0 + 8 * p + (lane >> 3);
            const bool on = slot >= u.s0 && slot < u.s1, again = slot < u.s0 && sc.ratio != 1.0;
            uint32_t *c = (uint32_t *)(c0 + slot * a.Dh);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (32 * i + 4 * j >= a.Dh) continue;
                if (on) {
                    uint32_t word = 0;
#pragma unroll
                    for (int b = 0; b < 4; b++)
                        word |= kv8_code((double)x[p][4 * i + b] * rms[p] * (double)w[4 * i + b], sc.inv) << (8 * b);
                    c[8 * i + j] = word;
                } else if (again) {
                    c[8 * i + j] = kv8_again(c[8 * i + j], sc.ratio);
                }
            }
        }
    } else {
        // V: lane j holds dims 2 j and 2 j + 1 of 16 tokens, whose codes are 32
        // bytes of the page in a row
        const int d = 2 * lane;
        float x[2][16];
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int slot = slot0 + i;
            float2 t = make_float2(0.0f, 0.0f);
            if (slot >= u.s0 && slot < u.s1 && d < a.Dh)
                t = *(const float2 *)(v + (int64_t)(u.row + slot - u.s0) * ld + (int64_t)hk * a.Dh + d);
            x[0][i] = t.x, x[1][i] = t.y;
            most = fmaxf(most, fmaxf(fabsf(t.x), fabsf(t.y)));
            bad |= !(fabsf(t.x) < INFINITY) || !(fabsf(t.y) < INFINITY);
        }
        const Kv8Scale sc = kv8_rescale(a.scale(page, 1, hk), u.s0 == 0, most, bad);
        if (d >= a.Dh || slot0 >= u.s1 || (slot0 + 16 <= u.s0 && sc.ratio == 1.0)) return;
        const bool whole = slot0 >= u.s0 && slot0 + 16 <= u.s1;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            uint4 *c = (uint4 *)(a.v_codes(page, hk) + ((int64_t)(d + e) << a.lg) + slot0);
            const uint4 was = whole ? make_uint4(0, 0, 0, 0) : *c;
            const uint32_t old[4] = {was.x, was.y, was.z, was.w};
            uint32_t now[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t kept = sc.ratio != 1.0 ? kv8_again(old[i], sc.ratio) : old[i];
                now[i] = 0;
#pragma unroll
                for (int b = 0; b < 4; b++) {
                    const int slot = slot0 + 4 * i + b;
                    const uint32_t byte = slot < u.s0 ? kept >> (8 * b) : slot < u.s1 ? kv8_code((double)x[e][4 * i + b], sc.inv) : old[i] >> (8 * b);
                    now[i] |= (byte & 0xFFu) << (8 * b);
                }
            }
            *c = make_uint4(now[0], now[1], now[2], now[3]);
        }
    }
}

// ---------------------------------------------------------------- read -----
// Rows of the cache as f32 (code * scale): the same units, a wave for each 16
// tokens of a page.
extern "C" __global__ __launch_bounds__(256) void sepia_kv8_read(Kv8Args a, float *__restrict__ k,
                                                                 float *__restrict__ v) {
    const int hk = (int)blockIdx.y, lane = (int)(threadIdx.x & 63), slot0 = (int)(threadIdx.x >> 6) * 16;
    kv8_check(a);
    int32_t len, r0, r1;
    const int s = kv8_find(a, blockIdx.x, a.P(), 2, len, r0, r1);
    Kv8Unit u;
    if (s < 0) return;
    if (!kv8_unit(len, r0, r1, (int)(blockIdx.x - kv8_first_id(r0, s, a.P(), 2)), a.lg, &u)) return;
    const int page = kv8_page(a, s, u.page);
    if (page < 0) {
        sepia_report_error(nullptr, KV8_ERR_PAGE, (int)threadIdx.x);
        return;
    }
    const int64_t ld = (int64_t)a.Hkv * a.Dh;
    const float sc = *a.scale(page, (int)blockIdx.z, hk);
    float *out = (blockIdx.z ? v : k) + (int64_t)hk * a.Dh;
    if (blockIdx.z == 0) {
        const int j = lane & 7;
#pragma unroll
        for (int p = 0; p < 2; p++) {
            const int slot = slot0 + 8 * p + (lane >> 3);
            if (slot < u.s0 || slot >= u.s1) continue;
            const uint32_t *c = (const uint32_t *)(a.k_codes(page, hk) + slot * a.Dh);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int d = 32 * i + 4 * j;
                if (d >= a.Dh) continue;
                const uint32_t w = c[8 * i + j];
                *(float4 *)(out + (int64_t)(u.row + slot - u.s0) * ld + d) =
                    make_float4((float)(int8_t)w * sc, (float)(int8_t)(w >> 8) * sc, (float)(int8_t)(w >> 16) * sc,
                                (float)(int8_t)(w >> 24) * sc);
            }
        }
        return;
    }
    const int d = 2 * lane;
    if (d >= a.Dh || slot0 + 16 <= u.s0 || slot0 >= u.s1) return;
    const int8_t *c = a.v_codes(page, hk) + ((int64_t)d << a.lg) + slot0;
    const uint4 e = *(const uint4 *)c, f = *(const uint4 *)(c + a.P());
    const uint32_t we[4] = {e.x, e.y, e.z, e.w}, wf[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int slot = slot0 + i;
        if (slot < u.s0 || slot >= u.s1) continue;
        *(float2 *)(out + (int64_t)(u.row + slot - u.s0) * ld + d) = make_float2(
            (float)(int8_t)(we[i / 4] >> (8 * (i % 4))) * sc, (float)(int8_t)(wf[i / 4] >> (8 * (i % 4))) * sc);
    }
}
