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
#include "serve.h"
#include "serve_layout.h"

#define KV8_ERR_PAGE 6u   // device error: a page of the table outside the pool
#define KV8_ERR_SEQ 7u    // device error: lens or starts that do not fit the call

// What every kernel is given.
struct Kv8Args : Kv8Call {
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

// The sequence that owns `id`, which of its units that is, its length and rows;
// -1 if there is none, or one that cannot be used. 64 sequences a look: one round for up to 64 of
// them, with everything about the one found already loaded, two for 4096.
__device__ __forceinline__ int kv8_find(const Kv8Args &a, int64_t id, int gran, int extra, int32_t &k, int32_t &len, int32_t &r0,
                                        int32_t &r1) {
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
            const int found = lo + c - 1;
            return kv8_place(id, r0, found, gran, extra, &k) && kv8_seq_ok(len, r0, r1, a.n, (int64_t)a.max_pages << a.lg) ? found : -1;
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

// 1 / v for a positive v of f32's range, within a rounding or two of 2^-53.
__device__ __forceinline__ double kv8_rcp(double v) {
    double r = __builtin_amdgcn_rcp(v);
    r = __builtin_fma(__builtin_fma(-v, r, 1.0), r, r);
    return __builtin_fma(__builtin_fma(-v, r, 1.0), r, r);
}
// Sum over the 8 lanes of a token; every lane gets it.
__device__ __forceinline__ double kv8_sum8(double v) {
#define KV8_SWAP(ctrl)                                                                                                  \
    {                                                                                                                   \
        const uint64_t b = __builtin_bit_cast(uint64_t, v);                                                             \
        const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, ctrl, 0xF, 0xF, true);           \
        const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), ctrl, 0xF, 0xF, true);   \
        v += __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);                                                       \
    }
    KV8_SWAP(0xB1)    // lanes 1 0 3 2
    KV8_SWAP(0x4E)    // lanes 2 3 0 1
    KV8_SWAP(0x141)   // the half row mirrored: the other four lanes
#undef KV8_SWAP
    return v;
}
// The largest of a value over the wave; every lane gets it.
__device__ __forceinline__ float kv8_wave_max(float v) {
#define KV8_ROR(n)                                                                                                   \
    v = fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x120 | n, 0xF, 0xF, true)))
    KV8_ROR(8);
    KV8_ROR(4);
    KV8_ROR(2);
    KV8_ROR(1);
#undef KV8_ROR
    const auto a = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    v = fmaxf(__builtin_bit_cast(float, (uint32_t)a[0]), __builtin_bit_cast(float, (uint32_t)a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)b[0]), __builtin_bit_cast(float, (uint32_t)b[1]));
}

// The unit's scale from its waves' largest values (bad: one is not finite; old:
// the scale there was, 0 for none), and what its codes are multiplied with: the
// new rows' 1 / scale, the old codes' old / new (1 where the scale did not
// grow). `waves` waves are a unit.
struct Kv8Scale {
    double inv, ratio;
};
__device__ __forceinline__ Kv8Scale kv8_rescale(float *scale, float old, float most, bool bad, int wave, int waves, bool mine) {
    __shared__ float red[4];
    const int w0 = wave & ~(waves - 1);
    most = kv8_wave_max(most);
    if (__ballot(bad)) most = INFINITY;
    if ((threadIdx.x & 63) == 0) red[wave] = most;
    __syncthreads();   // every wave has the old scale, and the maxima
    for (int w = 0; w < waves; w++) most = fmaxf(most, red[w0 + w]);
    float s = fmaxf(old, most * (1.0f / 127.0f));
    if (!(s < INFINITY) || old != old) s = NAN;
    if (mine && wave == w0 && (threadIdx.x & 63) == 0) *scale = s;
    Kv8Scale r;
    r.inv = s > 0.0f ? kv8_rcp((double)s) : 0.0;
    r.ratio = s > old ? (double)old * r.inv : 1.0;   // 0 behind a scale of 0, whose codes stand for 0
    return r;
}

// Grid (ids, kv heads / what a workgroup takes of them, 2: K and V), a wave for
// each 16 tokens of a page: four heads a workgroup with pages of 16, two of 32,
// one of 64. What bounds it is the chain of dependent loads (arguments,
// lengths, table entry, the old scale and codes) and the launch: 4.7 us for one
// token (8 heads of 128), 8.1 for 61 sequences' tokens (16 heads), 18.1 for 5157
// rows of prompts (8 heads; 53 MB, 2.9 TB/s), in calls that append the rows over
// themselves, so that no scale grows; 5.0, 9.7 and 18 where all of them do and the
// codes before are rounded anew. Twice as many waves of half the
// work took 11.3 us for the 61 and as long for the prompts; four waves a SIMD in
// the place of three spilled and took 8.9 and 20.6.
extern "C" __global__ __launch_bounds__(256, 3) void sepia_kv8_append(Kv8Args a, const float *__restrict__ k,
                                                                   const float *__restrict__ v,
                                                                   const float *__restrict__ norm, float eps) {
    serve_args<64>();
    const int waves = a.P() / 16, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = (int)(threadIdx.x & 63);
    const int head = (int)blockIdx.y * (4 / waves) + wave / waves, slot0 = (wave & (waves - 1)) * 16;
    const int hk = min(head, a.Hkv - 1);
    const bool mine = head < a.Hkv;   // else the wave only keeps the others company at the barrier
    kv8_check(a);
    int32_t k_unit, len, r0, r1;
    const int s = kv8_find(a, blockIdx.x, a.gran, a.extra, k_unit, len, r0, r1);
    Kv8Unit u;
    if (s < 0) return;
    if (!kv8_unit(len, r0, r1, k_unit, a.lg, &u)) return;
    // The rows are asked for before the table's entry is waited for.
    const int page = kv8_page(a, s, u.page);
    const int64_t ld = (int64_t)a.Hkv * a.Dh;
    float most = 0.0f;
    bool bad = false;
    if (blockIdx.z == 0) {
        // K: 8 lanes a token, 8 tokens a pass; lane j of a token holds dims
        // 32 i + 4 j .. + 3, so that every access of the eight is a whole line.
        // A pass without new tokens is passed over.
        const int j = lane & 7;
        float x[2][16], w[16];
        double rms[2] = {1.0, 1.0};
        bool some[2];
#pragma unroll
        for (int i = 0; i < 16; i++) w[i] = 1.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int d = 32 * i + 4 * j;
            if (!norm) break;
            const float4 t = *(const float4 *)(norm + (d < a.Dh ? d : 0));
            w[4 * i] = t.x, w[4 * i + 1] = t.y, w[4 * i + 2] = t.z, w[4 * i + 3] = t.w;
        }
#pragma unroll
        for (int p = 0; p < 2; p++) {
            some[p] = mine && slot0 + 8 * p < u.s1 && slot0 + 8 * p + 8 > u.s0;
            if (!some[p]) continue;
            const int slot = max(u.s0, min(u.s1 - 1, slot0 + 8 * p + (lane >> 3)));   // rows that repeat change nothing
            const float *row = k + (int64_t)(u.row + slot - u.s0) * ld + (int64_t)hk * a.Dh;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int d = 32 * i + 4 * j;
                float4 t = *(const float4 *)(row + (d < a.Dh ? d : 0));
                if (d >= a.Dh) t = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                x[p][4 * i] = t.x, x[p][4 * i + 1] = t.y, x[p][4 * i + 2] = t.z, x[p][4 * i + 3] = t.w;
            }
        }
        if (page < 0) {
            sepia_report_error(nullptr, KV8_ERR_PAGE, (int)threadIdx.x);
            return;
        }
        const float old = u.s0 == 0 ? 0.0f : *a.scale(page, 0, hk);
#pragma unroll
        for (int p = 0; p < 2; p++) {
            if (!some[p]) continue;
            if (norm) {
                double ss[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
                for (int i = 0; i < 16; i++) ss[i & 3] = __builtin_fma((double)x[p][i], (double)x[p][i], ss[i & 3]);
                rms[p] = rsqrt(kv8_sum8((ss[0] + ss[1]) + (ss[2] + ss[3])) / a.Dh + (double)eps);
            }
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const float y = (float)((double)x[p][i] * rms[p] * (double)w[i]);
                most = fmaxf(most, fabsf(y));
                bad |= !(fabsf(y) < INFINITY);
            }
        }
        const Kv8Scale sc = kv8_rescale(a.scale(page, 0, hk), old, most, bad, wave, waves, mine);
        if (!mine) return;
        uint32_t *codes = (uint32_t *)(a.k_codes(page, hk) + (slot0 + (lane >> 3)) * a.Dh) + j;
        if (sc.ratio != 1.0 && slot0 < u.s0) {   // the codes before the unit, all asked for before one is waited for
            uint32_t c[2][4];
#pragma unroll
            for (int p = 0; p < 2; p++)
#pragma unroll
                for (int i = 0; i < 4; i++) c[p][i] = codes[2 * p * a.Dh + (32 * i + 4 * j < a.Dh ? 8 * i : 0)];
#pragma unroll
            for (int p = 0; p < 2; p++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (slot0 + 8 * p + (lane >> 3) < u.s0 && 32 * i + 4 * j < a.Dh)
                        codes[2 * p * a.Dh + 8 * i] = kv8_again(c[p][i], sc.ratio);
        }
#pragma unroll
        for (int p = 0; p < 2; p++) {
            if (!some[p]) continue;
            const int slot = slot0 + 8 * p + (lane >> 3);
            const bool on = slot >= u.s0 && slot < u.s1;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                uint32_t word = 0;
#pragma unroll
                for (int b = 0; b < 4; b++)
                    word |= kv8_code((double)x[p][4 * i + b] * rms[p] * (double)w[4 * i + b], sc.inv) << (8 * b);
                if (on && 32 * i + 4 * j < a.Dh) codes[2 * p * a.Dh + 8 * i] = word;
            }
        }
    } else {
        // V: lane j has dims 2 j and 2 j + 1 of 16 tokens, whose codes are 32
        // bytes of the page in a row
        const int d = 2 * lane, dd = d < a.Dh ? d : 0;
        // a slot's row, or the nearest of the unit's: loads without branches are
        // in flight together
        const float *rows = v + (int64_t)hk * a.Dh + dd;
        float x[2][16];
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const float2 t = *(const float2 *)(rows + (int64_t)(u.row + max(0, min(u.s1 - 1, slot0 + i) - u.s0)) * ld);
            x[0][i] = t.x, x[1][i] = t.y;
        }
        if (page < 0) {
            sepia_report_error(nullptr, KV8_ERR_PAGE, (int)threadIdx.x);
            return;
        }
        const float old = u.s0 == 0 ? 0.0f : *a.scale(page, 1, hk);
        uint4 *codes[2], was[2];
        const bool whole = slot0 >= u.s0 && slot0 + 16 <= u.s1;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            codes[e] = (uint4 *)(a.v_codes(page, hk) + ((int64_t)(dd + e) << a.lg) + slot0);
            if (!whole) was[e] = *codes[e];
        }
        if (d < a.Dh) {
#pragma unroll
            for (int i = 0; i < 16; i++) {   // rows that repeat change nothing
                most = fmaxf(most, fmaxf(fabsf(x[0][i]), fabsf(x[1][i])));
                bad |= !(fabsf(x[0][i]) < INFINITY) || !(fabsf(x[1][i]) < INFINITY);
            }
        }
        const Kv8Scale sc = kv8_rescale(a.scale(page, 1, hk), old, most, bad, wave, waves, mine);
        if (!mine || d >= a.Dh || slot0 >= u.s1 || (slot0 + 16 <= u.s0 && sc.ratio == 1.0)) return;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            uint32_t now[4] = {was[e].x, was[e].y, was[e].z, was[e].w};
            if (sc.ratio != 1.0)   // the old codes are the first; what lies behind the new ones stays
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int n = u.s0 - slot0 - 4 * i;   // old codes of the word
                    if (n <= 0) continue;
                    const uint32_t keep = n >= 4 ? 0u : ~0u << (8 * n);
                    now[i] = (kv8_again(now[i], sc.ratio) & ~keep) | (now[i] & keep);
                }
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int slot = slot0 + i;
                const uint32_t at = 0xFFu << (8 * (i % 4));
                if (slot >= u.s0 && slot < u.s1)
                    now[i / 4] = (now[i / 4] & ~at) | kv8_code((double)x[e][i], sc.inv) << (8 * (i % 4));
            }
            *codes[e] = make_uint4(now[0], now[1], now[2], now[3]);
        }
    }
}

// ---------------------------------------------------------------- read -----
// Rows of the cache as f32 (code * scale): the same units, a wave for each 16
// tokens of a page. Bound by its writes from some thousand rows on.
extern "C" __global__ __launch_bounds__(256) void sepia_kv8_read(Kv8Args a, float *__restrict__ k,
                                                                 float *__restrict__ v) {
    serve_args<64>();
    const int waves = a.P() / 16, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = (int)(threadIdx.x & 63);
    const int head = (int)blockIdx.y * (4 / waves) + wave / waves, slot0 = (wave & (waves - 1)) * 16;
    const int hk = head;
    kv8_check(a);
    if (head >= a.Hkv) return;
    int32_t k_unit, len, r0, r1;
    const int s = kv8_find(a, blockIdx.x, a.gran, a.extra, k_unit, len, r0, r1);
    Kv8Unit u;
    if (s < 0) return;
    if (!kv8_unit(len, r0, r1, k_unit, a.lg, &u)) return;
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
