// logits.h -- logits with penalties for a request's tokens, biases and grammar
// masks.
//
// With n the number of times that a token occurs in its row's list from the
// prompt's end on and on its path, and `seen` whether it occurs at all:
//   x = seen ? (x > 0 ? x / repetition : x repetition) : x
//   x = x - frequency n - (n > 0 ? presence : 0) + bias
//   x = allowed ? x : -inf
// Workgroup: (chunk of the vocabulary, row). It goes through the row's whole
// list and counts what falls into its chunk in shared memory (whole numbers, so
// the order does not matter), a word a token: the count, and in the highest bit
// that it was seen. In place only logits that change are written, by masks alone of
// many rows whole lines of memory with such a logit (sepia_logits_lines).
//
// Bound by memory where rows are many: 196 rows of 100003 with lists of up to 8000
// tokens, masks and biases (157 MB) 43 us with three states in turn, 35 with one,
// which the Infinity Cache holds in part; a plain copy of as much 33 and 26. One row 7
// us: the launch and four dependent loads (its sequence, the list's place, the list,
// the logits). (The logits that a list names loaded one by one, in front of the copy's
// stores: 55 and 41.)
#pragma once
#include "common.h"
#include "serve.h"
#include "serve_layout.h"

#define LOGITS_ERR 7u        // device error: lists, rows or masks that do not fit the call
#define LOGITS_SEEN 0x80000000u

typedef float logits_f4 __attribute__((ext_vector_type(4)));
typedef logits_f4 logits_f4u __attribute__((aligned(4)));

// The sequence that row r belongs to, -1 for none: starts rise, 64 looks at a time.
__device__ __forceinline__ int logits_seq(const LogitsArgs &a, int r) {
    if (!a.row_starts) return r;
    const int lane = (int)threadIdx.x & 63;
    int lo = 0, n = a.n_seqs;   // among the sequences [lo, lo + n) the last that begins at or before r
    while (true) {
        const int step = (n + 63) / 64, i = lane * step;
        const int c = __builtin_popcountll(__ballot(i < n && a.row_starts[lo + min(i, n - 1)] <= r));
        if (c == 0) return -1;
        lo += (c - 1) * step;
        n = min(step, n - (c - 1) * step);
        if (step == 1) break;
    }
    return a.row_starts[lo] <= r && a.row_starts[lo + 1] > r ? lo : -1;   // starts that fall: perhaps another
}
// The grid's last workgroup reports what does not fit; rows that it concerns are
// left as they are.
__device__ __forceinline__ void logits_check(const LogitsArgs &a) {
    if (blockIdx.x + 1 != gridDim.x || blockIdx.y + 1 != gridDim.y) return;
    bool bad = false;
    for (int s = (int)threadIdx.x; s < a.n_seqs; s += (int)blockDim.x) {
        if (a.row_starts) {
            const int r0 = a.row_starts[s], r1 = a.row_starts[s + 1];
            bad |= r0 < 0 || r1 < r0 || r1 > a.rows || (a.tree && r1 - r0 > KV8_NODES);
        }
        if (a.tokens) bad |= a.token_starts[s] < 0 || a.token_starts[s + 1] < a.token_starts[s] || a.token_starts[s + 1] > a.n_tokens;
    }
    for (int r = (int)threadIdx.x; r < a.rows; r += (int)blockDim.x) {
        if (a.bias_tokens) bad |= a.bias_starts[r] < 0 || a.bias_starts[r + 1] < a.bias_starts[r] || a.bias_starts[r + 1] > a.n_biases;
        if (a.mask_row) bad |= a.mask_row[r] >= a.n_masks;
    }
    if (__syncthreads_or(bad)) sepia_report_error(nullptr, LOGITS_ERR, (int)threadIdx.x);
}

// Four logits from element t on (at the vocabulary's end the last ones again).
// Offsets in 32 bits from a pointer in scalar registers: a row is at most 4 MB.
__device__ __forceinline__ logits_f4 logits_four(const float *x, uint32_t t, uint32_t vocab) {
    if (t + 4 <= vocab) return *(const logits_f4u *)((const char *)x + 4 * t);
    logits_f4 v;
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) v[j] = *(const float *)((const char *)x + 4 * min(t + j, vocab - 1));
    return v;
}
// A logit whose token's word is n. The quotient is the product with 1 / repetition in
// double: two roundings of 2^-53, so off by up to 2^-52 before it is rounded to f32.
__device__ __forceinline__ float logits_penal(float v, uint32_t n, float rep, double inv, float freq, float pres) {
    if (n == 0) return v;
    const float times = (float)(n & ~LOGITS_SEEN);
    v = v > 0.0f ? (float)((double)v * inv) : v * rep;
    return times > 0.0f ? v - freq * times - pres : v;
}

// NT threads, four tokens each, N times: their logits and mask are asked for behind
// the list's first tokens, LOGITS_BATCH a thread, and used when the list is counted.
// In place the tokens that the list and the path name, few of a row, are taken one by
// one, each by the thread that sets its bit first.
#define LOGITS_BATCH 8
template <int NT, int N>
__device__ __forceinline__ void logits_run(const LogitsArgs &a) {
    constexpr uint32_t CHUNK = 4 * N * NT;
    __shared__ alignas(16) uint32_t word[CHUNK];   // counts, then biases' places
    __shared__ uint32_t bits[CHUNK / 32];          // in place: tokens that are taken
    serve_args<184>();
    logits_check(a);
    const int r = (int)blockIdx.y;
    const uint32_t c0 = blockIdx.x * CHUNK, vocab = (uint32_t)a.vocab, wide = min(vocab - c0, CHUNK), tid = threadIdx.x;
    // What goes by the row is asked for before its sequence is looked for.
    const int32_t b0 = a.bias_tokens ? a.bias_starts[r] : 0, b1 = a.bias_tokens ? a.bias_starts[r + 1] : 0;
    const int32_t mask_row = !a.mask ? -1 : a.mask_row ? a.mask_row[r] : r;
    float rep = a.repetition ? a.repetition[r] : 1.0f, freq = a.frequency ? a.frequency[r] : 0.0f, pres = a.presence ? a.presence[r] : 0.0f;
    uint64_t path = a.tree ? a.tree[r] : 0;
    const int s = logits_seq(a, r);
    if (s < 0 || b0 < 0 || b1 < b0 || b1 > a.n_biases || mask_row >= a.n_masks + !a.mask) return;
    int32_t lo = 0, hi = 0, first = 0;
    if (a.tokens) {
        lo = a.token_starts[s];
        hi = a.token_starts[s + 1];
        if (lo < 0 || hi < lo || hi > a.n_tokens) return;
    }
    if (a.tree) {
        first = a.row_starts[s];
        if (a.row_starts[s + 1] - first > KV8_NODES || first < 0 || a.row_starts[s + 1] > a.rows) return;
        path &= (2ull << (r - first)) - 1;   // the row's own token too
    }
    const uint32_t *mask = mask_row >= 0 ? a.mask + (int64_t)mask_row * ((a.vocab + 31) / 32) : nullptr;
    if (!(rep > 0.0f)) rep = 1.0f;
    if (freq != freq) freq = 0.0f;
    if (pres != pres) pres = 0.0f;
    const double inv = 1.0 / (double)rep;
    const bool counts = (rep != 1.0f || freq != 0.0f || pres != 0.0f) && (hi > lo || path);
    const float *x = a.logits + r * a.stride;
    float *y = a.out + r * a.out_stride;
    const bool here = x == y;
    // Loads return in the order they are issued in: the list's first tokens and the
    // biases', then the mask (used at once, it would keep the list waiting for the
    // logits: 50 us in the place of 43) and the logits.
    const uint32_t n_list = counts ? (uint32_t)(hi - lo) : 0, n_bias = (uint32_t)(b1 - b0);
    const uint32_t late = a.prompt && counts ? (uint32_t)max(0, a.prompt[s]) : 0;
    const int32_t *list = a.tokens + lo, *bias = a.bias_tokens + b0;
    uint32_t token[LOGITS_BATCH], drafted = ~0u, biased = ~0u;
#pragma unroll
    for (uint32_t k = 0; k < LOGITS_BATCH; k++)
        if (k * NT < n_list) token[k] = (uint32_t)list[min(tid + k * NT, n_list - 1)];
    if (counts && tid < KV8_NODES && path >> tid & 1) drafted = (uint32_t)a.drafted[first + (int)tid];
    if (tid < n_bias) biased = (uint32_t)bias[tid];
    logits_f4 v[N];
    uint32_t allowed[N];   // the groups' words of the mask
    if (!here) {
#pragma unroll
        for (uint32_t k = 0; k < N; k++) allowed[k] = mask ? mask[min(c0 + 4 * (tid + k * NT), vocab - 1) / 32] : ~0u;
#pragma unroll
        for (uint32_t k = 0; k < N; k++) v[k] = logits_four(x, min(c0 + 4 * (tid + k * NT), vocab - 1), vocab);
    } else if (mask) {   // nothing but what it forbids is written
        uint32_t w[4 * N];
#pragma unroll
        for (uint32_t k = 0; k < 4 * N; k++) w[k] = mask[min(c0 + tid + k * NT, vocab - 1) / 32];
#pragma unroll
        for (uint32_t k = 0; k < 4 * N; k++)
            if (tid + k * NT < wide && !(w[k] >> (tid % 32) & 1)) y[c0 + tid + k * NT] = -INFINITY;
    }
    const auto allows = [&](uint32_t t) { return !mask || (mask[(c0 + t) / 32] >> (t % 32) & 1); };
    if (counts) {
#pragma unroll
        for (uint32_t k = 0; k < N; k++) *(uint4 *)&word[4 * (tid + k * NT)] = make_uint4(0, 0, 0, 0);
        if (here && tid < CHUNK / 32) bits[tid] = 0;
        __syncthreads();
        for (uint32_t i0 = 0; i0 < n_list; i0 += LOGITS_BATCH * NT) {
            if (i0)
#pragma unroll
                for (uint32_t k = 0; k < LOGITS_BATCH; k++)
                    if (i0 + k * NT < n_list) token[k] = (uint32_t)list[min(i0 + k * NT + tid, n_list - 1)];
#pragma unroll
            for (uint32_t k = 0; k < LOGITS_BATCH; k++) {
                if (i0 + k * NT >= n_list) break;
                const uint32_t i = i0 + k * NT + tid, t = token[k] - c0;
                if (t >= wide || i >= n_list) continue;
                if (i < late) atomicOr(&word[t], LOGITS_SEEN);
                else atomicAdd(&word[t], 1u);
            }
        }
        if (drafted - c0 < wide) atomicAdd(&word[drafted - c0], 1u);
        __syncthreads();
        if (here) {
            const auto take = [&](uint32_t t) { return t < wide && !(atomicOr(&bits[t / 32], 1u << (t % 32)) >> (t % 32) & 1); };
            const auto put = [&](uint32_t t, float x) {
                const float p = logits_penal(x, word[t], rep, inv, freq, pres);
                if (allows(t)) y[c0 + t] = p;
            };
            for (uint32_t i0 = 0; i0 < n_list; i0 += LOGITS_BATCH * NT) {
                if (n_list > LOGITS_BATCH * NT)
#pragma unroll
                    for (uint32_t k = 0; k < LOGITS_BATCH; k++)
                        if (i0 + k * NT < n_list) token[k] = (uint32_t)list[min(i0 + k * NT + tid, n_list - 1)];
#pragma unroll
                for (uint32_t k0 = 0; k0 < LOGITS_BATCH; k0 += 4) {
                    if (i0 + k0 * NT >= n_list) break;
                    bool mine[4];
                    float held[4];
#pragma unroll
                    for (uint32_t k = 0; k < 4; k++) {
                        mine[k] = i0 + (k0 + k) * NT < n_list && take(token[k0 + k] - c0);   // the last one again changes nothing
                        if (mine[k]) held[k] = x[token[k0 + k]];
                    }
#pragma unroll
                    for (uint32_t k = 0; k < 4; k++)
                        if (mine[k]) put(token[k0 + k] - c0, held[k]);
                }
            }
            if (take(drafted - c0)) put(drafted - c0, x[drafted]);
        }
    }
    if (!here)
#pragma unroll
        for (uint32_t k = 0; k < N; k++) {
            const uint32_t i = 4 * (tid + k * NT), t = c0 + i;
            if (t >= vocab) break;
            if (counts) {
                const uint4 n = *(const uint4 *)&word[i];
                v[k][0] = logits_penal(v[k][0], n.x, rep, inv, freq, pres);
                v[k][1] = logits_penal(v[k][1], n.y, rep, inv, freq, pres);
                v[k][2] = logits_penal(v[k][2], n.z, rep, inv, freq, pres);
                v[k][3] = logits_penal(v[k][3], n.w, rep, inv, freq, pres);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) v[k][j] = allowed[k] >> (t % 32 + j) & 1 ? v[k][j] : -INFINITY;
            if (t + 4 <= vocab) *(logits_f4u *)((char *)y + 4 * t) = v[k];
            else
                for (uint32_t j = 0; t + j < vocab; j++) y[t + j] = v[k][j];
        }
    // Biases: of a token's several the last counts, which has the largest place in
    // the list, from 1 on. They come on top of what has been written.
    if (n_bias == 0) return;
    bool some = false;
    for (uint32_t i = tid; i < n_bias; i += NT) some |= (i < NT ? biased : (uint32_t)bias[i]) - c0 < wide;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (!__syncthreads_or(some)) return;
    for (uint32_t i = tid; i < n_bias; i += NT) {
        const uint32_t t = (i < NT ? biased : (uint32_t)bias[i]) - c0;
        if (t < wide) word[t] = 0;
    }
    __syncthreads();
    for (uint32_t i = tid; i < n_bias; i += NT) {
        const uint32_t t = (i < NT ? biased : (uint32_t)bias[i]) - c0;
        if (t < wide) atomicMax(&word[t], i + 1);
    }
    __syncthreads();
    for (uint32_t i = tid; i < n_bias; i += NT) {
        const uint32_t t = (i < NT ? biased : (uint32_t)bias[i]) - c0;
        if (t < wide && word[t] == i + 1 && allows(t)) y[c0 + t] = y[c0 + t] + a.bias_values[b0 + (int64_t)i];
    }
}
extern "C" __global__ __launch_bounds__(LOGITS_NT, 8) void sepia_logits(LogitsArgs a) { logits_run<LOGITS_NT, LOGITS_MANY>(a); }
extern "C" __global__ __launch_bounds__(LOGITS_NT, 8) void sepia_logits_few(LogitsArgs a) { logits_run<LOGITS_NT, 1>(a); }

// Masks alone, in place: what they forbid is written, a token a lane, and no logit
// read.
extern "C" __global__ __launch_bounds__(LOGITS_NT, 8) void sepia_logits_mask(LogitsArgs a) {
    constexpr int N = LOGITS_MASK;
    serve_args<184>();
    logits_check(a);
    const int r = (int)blockIdx.y, c0 = (int)blockIdx.x * N * LOGITS_NT, tid = (int)threadIdx.x;
    const int32_t which = a.mask_row ? a.mask_row[r] : r;
    if (which < 0 || which >= a.n_masks || logits_seq(a, r) < 0) return;
    const uint32_t *mask = a.mask + (int64_t)which * ((a.vocab + 31) / 32);
    float *y = a.out + r * a.out_stride;
    uint32_t w[N];
#pragma unroll
    for (int k = 0; k < N; k++) w[k] = mask[min(c0 + tid + k * LOGITS_NT, a.vocab - 1) / 32];
#pragma unroll
    for (int k = 0; k < N; k++) {
        const int t = c0 + tid + k * LOGITS_NT;
        if (t < a.vocab && !(w[k] >> (t % 32) & 1)) y[t] = -INFINITY;
    }
}

// The same where the rows are more than the caches hold (LOGITS_MUCH): memory takes
// a line written in part no faster than one read and written whole, and these wait
// for nothing in the caches. Lines begin at multiples of 32 floats in memory; at the
// row's ends, whose lines are shared with other rows, single tokens are written. 200
// rows of 199999, of three states in turn, 48 us against 71 by single tokens; of one
// state, which the Infinity Cache holds, 48 against 28.
extern "C" __global__ __launch_bounds__(LOGITS_NT, 8) void sepia_logits_lines(LogitsArgs a) {
    constexpr int N = LOGITS_MASK / 4;
    serve_args<184>();
    logits_check(a);
    const int r = (int)blockIdx.y;
    const int32_t which = a.mask_row ? a.mask_row[r] : r;
    if (which < 0 || which >= a.n_masks || logits_seq(a, r) < 0) return;
    const int words = (a.vocab + 31) / 32;
    const uint32_t *mask = a.mask + (int64_t)which * words;
    float *y = a.out + r * a.out_stride;
    const int lead = (int)((uintptr_t)y / 4 % 32);   // floats of the first line in front of the row
    const int t0 = (int)blockIdx.x * N * 4 * LOGITS_NT + 4 * (int)threadIdx.x - lead;
    uint32_t f[N];
    logits_f4 v[N];
#pragma unroll
    for (int k = 0; k < N; k++) {
        const int t = t0 + 4 * k * LOGITS_NT, i = t >> 5;
        const uint64_t w = mask[max(0, min(i, words - 1))] | (uint64_t)mask[max(0, min(i + 1, words - 1))] << 32;
        f[k] = (uint32_t)(w >> (t & 31)) & 0xF;
    }
#pragma unroll
    for (int k = 0; k < N; k++) {
        const int t = t0 + 4 * k * LOGITS_NT;
        const bool in = t >= 0 && t + 4 <= a.vocab;
        if (!in) {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (t + j >= 0 && t + j < a.vocab && !(f[k] >> j & 1)) y[t + j] = -INFINITY;
            f[k] = 0xF;
        }
        const uint64_t some = __ballot(f[k] != 0xF);
        const bool dirty = (some >> ((int)threadIdx.x & 56) & 0xFF) != 0;   // the line of eight lanes
        if (!dirty || !in) f[k] = 0x10;   // is left
        else if (f[k]) v[k] = __builtin_nontemporal_load((const logits_f4 *)(y + t));
    }
#pragma unroll
    for (int k = 0; k < N; k++) {
        const int t = t0 + 4 * k * LOGITS_NT;
        if (f[k] == 0x10) continue;
#pragma unroll
        for (int j = 0; j < 4; j++) v[k][j] = f[k] >> j & 1 ? v[k][j] : -INFINITY;
        __builtin_nontemporal_store(v[k], (logits_f4 *)(y + t));
    }
}
