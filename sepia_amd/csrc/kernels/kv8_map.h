// kv8_map.h -- where the rows of a call lie in a paged 8-bit key/value cache
// (kv8.h): plain integer code for the kernels, and for a CPU build that
// checks it.
//
// A call brings `n` new rows of several sequences back to back: sequence s
// has rows starts[s] .. starts[s + 1] - 1, at positions lens[s] + i. Work is
// cut into units of a sequence (the pages it touches, tiles of its rows)
// whose number only the device knows. The grid therefore counts in an id
// space that is fixed by n and the number of sequences alone: sequence s owns
// the ids from starts[s] / gran + extra s up to the next sequence's, which
// are at least as many as its units when a sequence of r rows has at most
// r / gran + extra units (pages touched: r / page + 2, and also r; row tiles of
// t rows: r / t + 1). An id past a sequence's last unit has no work.
#pragma once
#include <stdint.h>

#ifdef __HIPCC__
#define KV8_FN __device__ __forceinline__
#else
#define KV8_FN static inline
#endif

// The first id of sequence s.
KV8_FN int64_t kv8_first_id(int32_t start, int32_t s, int32_t gran, int32_t extra) {
    return (int64_t)(start / gran) + (int64_t)extra * s;
}
// The unit of sequence s that `id` stands for; 0 where the sequence's ids begin
// behind it, as they may for the one that a search finds where starts fall.
KV8_FN int kv8_place(int64_t id, int32_t start, int32_t s, int32_t gran, int32_t extra, int32_t *k) {
    const int64_t first = kv8_first_id(start, s, gran, extra);
    *k = (int32_t)(id - first);
    return id >= first;
}
// Ids of a call of n rows.
KV8_FN int64_t kv8_ids(int64_t n, int32_t n_seqs, int32_t gran, int32_t extra) {
    return n / gran + (int64_t)extra * n_seqs;
}
// Whether a sequence's length and rows can be used: the call's bounds, and
// every position within the table's row.
KV8_FN int kv8_seq_ok(int32_t len, int32_t r0, int32_t r1, int32_t n, int64_t capacity) {
    return len >= 0 && r0 >= 0 && r1 >= r0 && r1 <= n && (int64_t)len + (r1 - r0) <= capacity;
}

// Steps of 64 columns that columns 0 .. end - 1 lie in, end > 0 (up to 2^31 - 1).
KV8_FN int32_t kv8_steps(int32_t end) { return (end - 1) / 64 + 1; }

// Slots [s0, s1) of page `page` of the sequence that the k-th touched page's
// unit fills with the rows from r0 + (page << lg) + s0 - len on; 0 where there
// is no such unit.
typedef struct {
    int32_t page, s0, s1;
    int32_t row;   // the call's row of slot s0
} Kv8Unit;
KV8_FN int kv8_unit(int32_t len, int32_t r0, int32_t r1, int32_t k, int32_t lg, Kv8Unit *u) {
    if (r1 <= r0) return 0;
    const int32_t end = len + (r1 - r0), page = (len >> lg) + k;
    if (page > ((end - 1) >> lg)) return 0;
    const int32_t base = page << lg;
    u->page = page;
    u->s0 = len > base ? len - base : 0;
    u->s1 = end - base < (1 << lg) ? end - base : (1 << lg);
    u->row = r0 + (base + u->s0 - len);
    return 1;
}
