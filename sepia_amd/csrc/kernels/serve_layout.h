// serve_layout.h -- what the serving kernels and their host (serve.c) have to
// agree on: the kernels' arguments, what lies in scratch, and the constants of
// both. Plain C.
#pragma once
#include <stdint.h>

// A cache call (kernels/kv8.h).
typedef struct {
    int8_t *codes;
    float *scales;
    const int32_t *table, *lens, *starts;
    int64_t n_pages;
    int32_t n_seqs, max_pages, Hkv, Dh, lg, n;   // lg: of a page's tokens; n: rows of the call
    uint32_t head_bytes, page_bytes;             // of a head's K or V in a page, of a page
    int32_t gran, extra;                         // the id space of the pages (kv8_map.h)
} Kv8Call;

// An attention call (kernels/kv8_attn.h).
#define KV8_NW 4         // waves of a workgroup: they take a unit's steps in turn
#define KV8_UNITS 8192   // arrival counters of a call, twice
typedef struct {
    const float *q, *rel, *tau;
    float *out;
    float *part, *ml;        // per run: O [16][Dh]; maxima [16], sums [16]
    uint32_t *arrived;       // at a group's first run's place: its runs that are done; KV8_UNITS on, at a unit's
                             // first run's place: its groups
    int32_t H, R, window, TT, budget;   // TT: tokens of a row tile
    float c;
} Kv8AttnCall;

// A sampling call (kernels/sample.h). Where a row has several chunks, scratch
// holds the rows' gathered tokens and then, [row][chunk], the chunks' bins.
#define SAMPLE_NT 512       // two workgroups a CU (of 1024 threads one: 36 against 26 us at 48 rows)
#define SAMPLE_BINS 1024    // two a thread
#define SAMPLE_MANY 16384   // gathered tokens of a row in scratch
typedef struct {
    unsigned long long mass[SAMPLE_BINS], over_min, best;
    uint32_t count[SAMPLE_BINS];
} SampleChunk;
typedef struct {
    unsigned long long list[SAMPLE_MANY];
    uint32_t n, arrived, unused[2];   // a multiple of 16 bytes: the bins behind are read by pairs of masses
} SampleRow;
typedef struct {
    const float *logits, *u, *temperature, *top_p, *min_p;
    const int32_t *top_k;
    int32_t *token;
    float *prob;
    SampleRow *rows;
    SampleChunk *bins;   // [row][chunk]
    int64_t stride;
    int32_t vocab, chunk, chunks;
} SampleArgs;
