// sample.h -- the next token of each row of logits: temperature, top-k,
// top-p, min-p, and a draw by a given uniform number.
//
// With x the row's logits, m their maximum and T the temperature, a token's
// weight is w = e^((x - m) / T); -inf and NaN have none. The tokens are
// ordered by falling logit, equal ones by index. Kept are the first k of them
// (top-k), of these the shortest beginning whose weight reaches p of theirs
// (top-p), and of these the ones with w >= min-p: a beginning of the order
// each time. The draw is the first token whose cumulative weight exceeds u
// times the kept weight. T <= 0: the first token of the order.
//
// Weights are summed as integers in units of 2^-44 of the largest, so that
// every sum is exact and does not depend on its order: a row of up to 2^20
// tokens sums to less than 2^64, and a weight is within 2^-45 of its value
// (over n tokens the sums err by about sqrt(n) 2^-46, 10^-11 at most).
#pragma once
#include "common.h"

#define SAMPLE_ONE 17592186044416.0   // 2^44: the largest weight

struct SampleArgs {
    const float *logits, *u, *temperature, *top_p, *min_p;
    const int32_t *top_k;
    int32_t *token;
    float *prob;
    int64_t stride;
    int32_t vocab;
};

// Keys fall as logits rise: 0 is the largest. -0 and +0 are equal.
__device__ __forceinline__ uint32_t sample_key(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
    return (int32_t)b < 0 ? b : ~(b | 0x80000000u) & 0x7FFFFFFFu;
}
__device__ __forceinline__ float sample_logit(uint32_t key) {
    return __builtin_bit_cast(float, (int32_t)key < 0 ? key : ~key & 0x7FFFFFFFu);
}
__device__ __forceinline__ bool sample_on(float x) { return x > -INFINITY; }   // neither -inf nor NaN
__device__ __forceinline__ double sample_weight(float x, float m, double t) {
    return x == m ? 1.0 : exp(((double)x - (double)m) / t);
}
__device__ __forceinline__ uint64_t sample_mass(float x, float m, double t) {
    return (uint64_t)__builtin_rint(sample_weight(x, m, t) * SAMPLE_ONE);
}

#define SAMPLE_NT 1024
#define SAMPLE_BINS 2048
struct SampleLds {
    unsigned long long mass[SAMPLE_BINS];
    uint32_t count[SAMPLE_BINS];
    unsigned long long red[16];
    uint32_t redc[16];
    int32_t bin;
    unsigned long long below;
};

__device__ __forceinline__ unsigned long long sample_sum(unsigned long long v, SampleLds &L) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) L.red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
    for (int i = 0; i < SAMPLE_NT / 64; i++) v += L.red[i];
    return v;
}

// The first token of the order whose cumulative weight (by_count: place from
// 1) exceeds `over`; its key and index, and the cumulative weight up to and
// with it. There is one. A pass over the row settles 11, 11 and 10 bits of
// the key, then, among equal logits, 10 and 10 of the index.
struct SampleAt {
    uint32_t key;
    int32_t index;
    unsigned long long cum;
};
__device__ SampleAt sample_find(const SampleArgs &a, const float *x, float m, double t, bool by_count,
                                unsigned long long over, SampleLds &L) {
    SampleAt r;
    uint64_t prefix = 0;          // the settled bits of key << 20 | index
    int settled = 0;
    unsigned long long done = 0, mass = 0;   // what lies before the prefix: by the measure, and weight
    const int bits[5] = {11, 11, 10, 10, 10};
    for (int level = 0; level < 5; level++) {
        const int left = 52 - settled - bits[level];
        for (int i = threadIdx.x; i < SAMPLE_BINS; i += SAMPLE_NT) L.mass[i] = 0, L.count[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < a.vocab; i += SAMPLE_NT) {
            const uint64_t c = ((uint64_t)sample_key(x[i]) << 20) | (uint32_t)i;
            if (!sample_on(x[i]) || (settled && c >> (52 - settled) != prefix)) continue;
            const int b = (int)(c >> left) & ((1 << bits[level]) - 1);
            atomicAdd(&L.count[b], 1u);
            atomicAdd(&L.mass[b], (unsigned long long)sample_mass(x[i], m, t));
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            int b = 0;
            while (b < SAMPLE_BINS - 1) {
                const unsigned long long n = by_count ? L.count[b] : L.mass[b];
                if (done + n > over) break;
                done += n;
                mass += L.mass[b];
                b++;
            }
            L.bin = b;
            L.below = done;
            L.red[0] = mass;
        }
        __syncthreads();
        done = L.below;
        mass = L.red[0];
        prefix = (prefix << bits[level]) | (uint32_t)L.bin;
        settled += bits[level];
        __syncthreads();
    }
    r.key = (uint32_t)(prefix >> 20);
    r.index = (int32_t)(prefix & 0xFFFFF);
    r.cum = mass + sample_mass(x[r.index], m, t);
    return r;
}

extern "C" __global__ __launch_bounds__(SAMPLE_NT) void sepia_sample(SampleArgs a) {
    __shared__ SampleLds L;
    const int row = (int)blockIdx.x;
    const float *x = a.logits + (int64_t)row * a.stride;
    float m = -INFINITY;
    unsigned long long n = 0;
    for (int i = threadIdx.x; i < a.vocab; i += SAMPLE_NT) {
        m = fmaxf(m, x[i]);
        n += sample_on(x[i]);
    }
    n = sample_sum(n, L);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) L.redc[threadIdx.x >> 6] = __builtin_bit_cast(uint32_t, m);
    __syncthreads();
    for (int i = 0; i < SAMPLE_NT / 64; i++) m = fmaxf(m, __builtin_bit_cast(float, L.redc[i]));
    if (n == 0) {
        if (threadIdx.x == 0) {
            a.token[row] = -1;
            if (a.prob) a.prob[row] = 0.0f;
        }
        return;
    }
    const float temperature = a.temperature ? a.temperature[row] : 1.0f;
    const float top_p = a.top_p ? a.top_p[row] : 1.0f, min_p = a.min_p && a.min_p[row] > 0.0f ? fminf(a.min_p[row], 1.0f) : 0.0f;
    const int32_t k = a.top_k ? a.top_k[row] : 0;
    if (!(temperature > 0.0f)) {
        const SampleAt r = sample_find(a, x, m, 1.0, true, 0, L);
        if (threadIdx.x == 0) {
            a.token[row] = r.index;
            if (a.prob) a.prob[row] = 1.0f;
        }
        return;
    }
    const double t = (double)temperature;
    const unsigned long long floor_mass = min_p > 0.0f ? (unsigned long long)__builtin_ceil((double)min_p * SAMPLE_ONE) : 0;
    unsigned long long all = 0, over_min = 0;
    for (int i = threadIdx.x; i < a.vocab; i += SAMPLE_NT) {
        const unsigned long long w = sample_on(x[i]) ? sample_mass(x[i], m, t) : 0;
        all += w;
        over_min += w >= floor_mass ? w : 0;
    }
    unsigned long long kept = sample_sum(all, L);
    over_min = sample_sum(over_min, L);
    if (k > 0 && (unsigned long long)k < n) kept = sample_find(a, x, m, t, true, (unsigned long long)k - 1, L).cum;
    if (top_p < 1.0f) {
        // the last kept token is the first with cumulative weight >= p times the total
        const double want = __builtin_ceil((double)fmaxf(top_p, 0.0f) * (double)kept);
        kept = sample_find(a, x, m, t, false, want >= 1.0 ? (unsigned long long)want - 1 : 0, L).cum;
    }
    if (over_min < kept) kept = over_min;
    const float u = a.u[row];
    unsigned long long over = u > 0.0f ? (unsigned long long)((double)fminf(u, 1.0f) * (double)kept) : 0;
    if (over >= kept) over = kept - 1;
    const SampleAt r = sample_find(a, x, m, t, false, over, L);
    if (threadIdx.x == 0) {
        a.token[row] = r.index;
        if (a.prob) a.prob[row] = (float)(sample_weight(x[r.index], m, t) * SAMPLE_ONE / (double)kept);
    }
}
