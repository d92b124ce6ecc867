/* serve.c -- the serving operators of include/sepia_hip_ext.h: the paged
 * 8-bit key/value cache (kernels/kv8.h) and sampling (kernels/sample.h). Host
 * checks and launches; what only the device knows (lengths, rows, the page
 * table) the kernels check. */
#include "internal.h"

#include <string.h>

#include "../../include/sepia_hip_ext.h"
#include "kernels/serve_layout.h"

#define LOG(...) sepia_log(__VA_ARGS__)
#define MAX_ROWS ((int64_t)1 << 24)     /* rows of a call: grids of fewer than 2^32 threads */
#define MAX_SAMPLES 65535              /* and of a sample call: the grid's second dimension */

/* What a call reads or writes of a buffer. */
typedef struct {
    SepiaGpuBuf *b;
    size_t off, n;
    const char *what;
} Part;
/* What a call writes (bit i of `written`: part i) while other workgroups read
 * the rest has to lie apart from all else, in one buffer or in two handles over
 * the same memory. */
static int apart(const char *op, const Part *p, int parts, unsigned written) {
    for (int i = 0; i < parts; i++) {
        if (!(written >> i & 1) || !p[i].b || !p[i].n) continue;
        const uintptr_t at = (uintptr_t)sepia_buf_dev(p[i].b) + p[i].off;
        for (int j = 0; j < parts; j++) {
            if (j == i || !p[j].b || !p[j].n) continue;
            const uintptr_t other = (uintptr_t)sepia_buf_dev(p[j].b) + p[j].off;
            if (at + p[i].n <= other || other + p[j].n <= at) continue;
            LOG("%s: %s overlaps %s", op, p[i].what, p[j].what);
            return 0;
        }
    }
    return 1;
}

/* Checks a cache and a call's rows, and fills the kernels' arguments; `write`:
 * the call writes to the pages. p: places for the cache's KV8_PARTS parts, then
 * the call's own (`parts` in all). */
enum { KV8_CODES, KV8_SCALES, KV8_TABLE, KV8_LENS, KV8_STARTS, KV8_PARTS };
static int kv8_args(const char *op, const SepiaKv8Cache *c, SepiaGpuBuf *lens, SepiaGpuBuf *starts, int64_t n,
                    int write, Part *p, int parts, unsigned written, Kv8Call *a) {
    if (!c || c->n_pages < 1 || c->max_pages < 1 || c->n_seqs < 1 || c->n_seqs > 65536 || c->n_kv_heads < 1 ||
        c->n_kv_heads > 65535 || n < 0 || n > MAX_ROWS || c->n_pages > 0x7FFFFFFF) {
        LOG("%s: invalid arguments", op);
        return 0;
    }
    if (c->page != 16 && c->page != 32 && c->page != 64) {
        LOG("%s: pages of %d tokens not supported (16, 32 or 64)", op, c->page);
        return 0;
    }
    if (c->head_dim < 16 || c->head_dim > 128 || c->head_dim % 16) {
        LOG("%s: head dim %d not supported (a multiple of 16 up to 128)", op, c->head_dim);
        return 0;
    }
    if (c->max_pages > 0x7FFFFFFF / c->page) {
        LOG("%s: %lld pages of %d tokens a sequence pass 2^31 - 1 positions", op, (long long)c->max_pages, c->page);
        return 0;
    }
    if (c->codes_off % 16 || c->scales_off % 4 || c->table_off % 4) {
        LOG("%s: the cache's offsets are not multiples of 16 (codes) and 4 bytes", op);
        return 0;
    }
    const size_t page = 2 * (size_t)c->n_kv_heads * (size_t)c->page * (size_t)c->head_dim;
    if ((size_t)c->n_pages > SIZE_MAX / page) {
        LOG("%s: invalid arguments", op);
        return 0;
    }
    const size_t cb = (size_t)c->n_pages * page, sb = (size_t)c->n_pages * 2 * (size_t)c->n_kv_heads * 4;
    const size_t tb = (size_t)c->n_seqs * (size_t)c->max_pages * 4, lb = (size_t)c->n_seqs * 4;
    if (!sepia_chk(c->codes, c->codes_off, cb, op, "codes") || !sepia_chk(c->scales, c->scales_off, sb, op, "scales") ||
        !sepia_chk(c->table, c->table_off, tb, op, "table") || !sepia_chk(lens, 0, lb, op, "lens") ||
        !sepia_chk(starts, 0, lb + 4, op, "starts"))
        return 0;
    p[KV8_CODES] = (Part){ c->codes, c->codes_off, cb, "codes" };
    p[KV8_SCALES] = (Part){ c->scales, c->scales_off, sb, "scales" };
    p[KV8_TABLE] = (Part){ c->table, c->table_off, tb, "table" };
    p[KV8_LENS] = (Part){ lens, 0, lb, "lens" };
    p[KV8_STARTS] = (Part){ starts, 0, lb + 4, "starts" };
    if (!apart(op, p, parts, written | (write ? 1u << KV8_CODES | 1u << KV8_SCALES : 0))) return 0;
    if (!sepia_need_batch(op) || !sepia_prep_in(c->table, c->table_off, tb, op) || !sepia_prep_in(lens, 0, lb, op) ||
        !sepia_prep_in(starts, 0, lb + 4, op))
        return 0;
    if (write ? !sepia_prep_out(c->codes, op) || !sepia_prep_out(c->scales, op)
              : !sepia_prep_in(c->codes, c->codes_off, cb, op) || !sepia_prep_in(c->scales, c->scales_off, sb, op))
        return 0;
    memset(a, 0, sizeof *a);
    a->codes = (int8_t *)sepia_buf_dev(c->codes) + c->codes_off;
    a->scales = (float *)(sepia_buf_dev(c->scales) + c->scales_off);
    a->table = (const int32_t *)(sepia_buf_dev(c->table) + c->table_off);
    a->lens = (const int32_t *)sepia_buf_dev(lens);
    a->starts = (const int32_t *)sepia_buf_dev(starts);
    a->n_pages = c->n_pages;
    a->n_seqs = c->n_seqs;
    a->max_pages = (int32_t)c->max_pages;
    a->Hkv = c->n_kv_heads;
    a->Dh = c->head_dim;
    a->lg = c->page == 16 ? 4 : c->page == 32 ? 5 : 6;
    a->n = (int32_t)n;
    a->head_bytes = (uint32_t)(c->page * c->head_dim);
    a->page_bytes = (uint32_t)page;
    return 1;
}

/* Units of pages, kv heads, K and V; a workgroup takes 64 tokens of the pages'
 * heads. A sequence of r > 0 rows touches at most r / page + 2 pages,
 * and at most r: the id space (kv8_map.h) that is the smaller for the call. */
static int kv8_pages(int k, const SepiaKv8Cache *c, int64_t n, Kv8Call *a, void **args, const char *op) {
    const int heads = 64 / c->page, few = n <= n / c->page + 2 * (int64_t)c->n_seqs;
    a->gran = few ? 1 : c->page;
    a->extra = few ? 0 : 2;
    const uint64_t ids = (uint64_t)(few ? n : n / c->page + 2 * (int64_t)c->n_seqs);
    return sepia_serve_launch(k, ids, (unsigned)((c->n_kv_heads + heads - 1) / heads), 2, 256, args, op);
}

int sepia_hip_kv8_append(const SepiaKv8Cache *c, SepiaGpuBuf *lens, SepiaGpuBuf *starts, int64_t n, SepiaGpuBuf *k,
                         SepiaGpuBuf *v, SepiaGpuBuf *k_norm, float eps) {
    const char *op = "kv8_append";
    Kv8Call a;
    if (!c || !lens || !starts || !k || !v) {
        LOG("%s: invalid arguments", op);
        return 0;
    }
    const size_t rows = n < 0 || n > MAX_ROWS ? 0 : (size_t)n * (size_t)c->n_kv_heads * (size_t)c->head_dim * 4;
    const size_t nb = (size_t)c->head_dim * 4;
    if (k_norm && !(eps >= 0.0f)) {
        LOG("%s: eps is negative or NaN", op);
        return 0;
    }
    if (c->n_kv_heads < 1 || c->head_dim < 1 || !sepia_chk(k, 0, rows, op, "k") || !sepia_chk(v, 0, rows, op, "v") ||
        (k_norm && !sepia_chk(k_norm, 0, nb, op, "k_norm"))) {
        if (c->n_kv_heads < 1 || c->head_dim < 1) LOG("%s: invalid arguments", op);
        return 0;
    }
    Part p[KV8_PARTS + 3] = { [KV8_PARTS] = { k, 0, rows, "k" }, { v, 0, rows, "v" }, { k_norm, 0, nb, "k_norm" } };
    if (!kv8_args(op, c, lens, starts, n, 1, p, KV8_PARTS + 3, 0, &a) || !sepia_prep_in(k, 0, rows, op) || !sepia_prep_in(v, 0, rows, op) ||
        (k_norm && !sepia_prep_in(k_norm, 0, nb, op)))
        return 0;
    if (n == 0) return 1;
    const float *kp = (const float *)sepia_buf_dev(k), *vp = (const float *)sepia_buf_dev(v);
    const float *np = (const float *)sepia_buf_dev(k_norm);
    void *args[] = { &a, &kp, &vp, &np, &eps };
    return kv8_pages(SK_KV8_APPEND, c, n, &a, args, op);
}

int sepia_hip_kv8_read(const SepiaKv8Cache *c, SepiaGpuBuf *first, SepiaGpuBuf *starts, int64_t n, SepiaGpuBuf *k,
                       SepiaGpuBuf *v) {
    const char *op = "kv8_read";
    Kv8Call a;
    if (!c || !first || !starts || !k || !v || k == v || c->n_kv_heads < 1 || c->head_dim < 1) {
        LOG("%s: invalid arguments", op);
        return 0;
    }
    const size_t rows = n < 0 || n > MAX_ROWS ? 0 : (size_t)n * (size_t)c->n_kv_heads * (size_t)c->head_dim * 4;
    if (!sepia_chk(k, 0, rows, op, "k") || !sepia_chk(v, 0, rows, op, "v")) return 0;
    Part p[KV8_PARTS + 2] = { [KV8_PARTS] = { k, 0, rows, "k" }, { v, 0, rows, "v" } };
    if (!kv8_args(op, c, first, starts, n, 0, p, KV8_PARTS + 2, 3u << KV8_PARTS, &a) || !sepia_prep_out(k, op) || !sepia_prep_out(v, op)) return 0;
    if (n == 0) return 1;
    float *kp = (float *)sepia_buf_dev(k), *vp = (float *)sepia_buf_dev(v);
    void *args[] = { &a, &kp, &vp };
    return kv8_pages(SK_KV8_READ, c, n, &a, args, op);
}

/* Units from which each has a wave of its own (a whole chip of them at two
 * workgroups a CU is 2048). Both kernels, wave a unit against cut into runs, us,
 * dim 128, 64 heads on 8: a chunk of 192, 256, 384, 512 rows (768 to 2048 units)
 * behind 200 columns 18, 23, 34, 40 against 20, 26, 38, 52, behind 1500 50, 53,
 * 81, 89 against 40, 50, 74, 100. Sequences of single tokens, ragged up to the
 * length: 128 (1024 units) of 500 columns 27 against 28, of 4000 138 against
 * 104, of 16000 554 against 324; 256 of 500 44 against 59, of 16000 841 against
 * 645; 1024 of 1000 227 against 480, since every run of a cut call looks through
 * all lengths. So a number of units says too little where contexts are long. */
#define KV8_ROWS 1024
#define KV8_BUDGET 512      /* runs of a call whose units alone leave the chip idle: two workgroups a CU */
_Static_assert(2 * (KV8_BUDGET * 3 / 2) + 64 <= KV8_UNITS && 2 * KV8_UNITS <= SEPIA_COUNTERS, "a counter for each slot, twice");

int sepia_hip_kv8_attn(const SepiaKv8Cache *c, SepiaGpuBuf *lens, SepiaGpuBuf *starts, int64_t n, SepiaGpuBuf *q,
                       SepiaGpuBuf *rel_logits, SepiaGpuBuf *tau, SepiaGpuBuf *out, int64_t n_heads,
                       int64_t rel_extent, int64_t window, float inv_head_dim) {
    const char *op = "kv8_attn";
    Kv8Call a;
    Kv8AttnCall b;
    if (!c || !lens || !starts || !q || !out || c->n_kv_heads < 1 || c->head_dim < 1 || n_heads < 1 ||
        n_heads > 65535 || n_heads % c->n_kv_heads || n_heads / c->n_kv_heads > 16 || window < 0 ||
        rel_extent < 0 || rel_extent > 0x7FFFFFFF || (rel_extent > 0) != (rel_logits != NULL) ||
        (rel_extent > 0 && n > 0 && n > INT64_MAX / 4 / n_heads / rel_extent)) {
        LOG("%s: invalid arguments", op);
        return 0;
    }
    const size_t rows = n < 0 || n > MAX_ROWS ? 0 : (size_t)n;
    const size_t qb = rows * (size_t)n_heads * (size_t)c->head_dim * 4, rb = rows * (size_t)n_heads * (size_t)rel_extent * 4;
    if (!sepia_chk(q, 0, qb, op, "q") || !sepia_chk(out, 0, qb, op, "out") ||
        (rel_logits && !sepia_chk(rel_logits, 0, rb, op, "rel_logits")) || (tau && !sepia_chk(tau, 0, rows * 4, op, "tau")))
        return 0;
    /* out may be q: a row of q is read by the workgroups whose last one writes it */
    const int same = sepia_buf_dev(q) == sepia_buf_dev(out);
    Part p[KV8_PARTS + 4] = { [KV8_PARTS] = { out, 0, qb, "out" }, { same ? NULL : q, 0, qb, "q" },
                              { rel_logits, 0, rb, "rel_logits" }, { tau, 0, rows * 4, "tau" } };
    if (!kv8_args(op, c, lens, starts, n, 0, p, KV8_PARTS + 4, 1u << KV8_PARTS, &a) || !sepia_prep_in(q, 0, qb, op) ||
        (rel_logits && !sepia_prep_in(rel_logits, 0, rb, op)) || (tau && !sepia_prep_in(tau, 0, rows * 4, op)) ||
        !sepia_prep_out(out, op))
        return 0;
    if (n == 0) return 1;
    memset(&b, 0, sizeof b);
    b.q = (const float *)sepia_buf_dev(q);
    b.rel = (const float *)sepia_buf_dev(rel_logits);
    b.tau = (const float *)sepia_buf_dev(tau);
    b.out = (float *)sepia_buf_dev(out);
    b.H = (int32_t)n_heads;
    b.R = (int32_t)rel_extent;
    b.window = window > 0x7FFFFFFF ? 0 : (int32_t)window;
    b.c = inv_head_dim;
    /* 16 rows a wave. Many units (row tile, kv head): a wave each. Few: cut
     * into runs of steps, whose partials are folded. */
    b.TT = (int32_t)(16 / (n_heads / c->n_kv_heads));
    const int dim = 2 * (c->head_dim <= 64) + (c->head_dim % 64 != 0);   /* which of the four kernels */
    const int64_t units = (n / b.TT > c->n_seqs ? n / b.TT : n < c->n_seqs ? n : c->n_seqs) * c->n_kv_heads;
    if (units >= KV8_ROWS) {
        void *args[] = { &a, &b };
        return sepia_serve_launch(SK_KV8_ROWS + dim, (uint64_t)(n / (4 * b.TT) + c->n_seqs) * (uint64_t)c->n_kv_heads,
                                  1, 1, 256, args, op);
    }
    /* Row tiles at most: sequences without rows have none. (4096 slots, a few in
     * use: 2.6 ms with all counted.) A call past the grid of the kernel above is
     * refused here too: whether it is does not go by the rows. */
    if ((uint64_t)(n / b.TT + c->n_seqs) * (uint64_t)c->n_kv_heads * 256 > UINT32_MAX) {
        LOG("%s: %lld row tiles and sequences of %d kv heads, more than a launch can have", op,
            (long long)(n / b.TT + c->n_seqs), c->n_kv_heads);
        return 0;
    }
    const int64_t ids = n / b.TT + (n < c->n_seqs ? n : c->n_seqs);
    const size_t per = 16 * (size_t)c->head_dim * 4, limit = sepia_scratch_limit();
    /* No more runs than places: a unit's last run is short, so as many fewer as
     * there are units (a whole round more for a few runs: 4 sequences of up to
     * 8000 columns, 8 kv heads and a band of 1024, 16.4 us against 18.2 with 512
     * runs). Half as many again as places where a run may be long, since units of
     * ragged lengths end unevenly (48 sequences of up to 12000 columns: 118.5 us
     * against 134.3 with 512; where runs are short they cost: 32 sequences in a
     * window of 512, 16 kv heads, 18.5 us against 28.5). None, and no scratch,
     * where a run has every step that the table or the window leaves a unit (as
     * long either way). What a unit may have is taken from the table's width: the
     * lengths are on the device. */
    int64_t steps = (c->max_pages * c->page + 63) / 64;   /* of a unit, at most */
    if (window > 0 && window / 64 + 2 < steps) steps = window / 64 + 2;
    int64_t budget = KV8_BUDGET - (units < KV8_BUDGET / 2 ? units : KV8_BUDGET / 2);
    if (units * steps / KV8_BUDGET > 64) budget = KV8_BUDGET * 3 / 2;
    if (steps <= KV8_NW) budget = 0;
    int64_t slots = 2 * budget + 64;
    while (budget && (size_t)slots * (per + 128) > limit) {
        budget /= 2;
        slots = 2 * budget + 64;
    }
    if (budget) {
        uint8_t *s = (uint8_t *)sepia_scratch((size_t)slots * (per + 128), op);
        if (!s) return 0;
        b.part = (float *)s;
        b.ml = (float *)(s + (size_t)slots * per);
        b.arrived = sepia_counters();   /* two for each slot, the second KV8_UNITS behind the first */
    }
    b.budget = (int32_t)budget;
    void *args[] = { &a, &b };
    return sepia_serve_launch(SK_KV8_ATTN + dim, (uint64_t)(budget + ids * c->n_kv_heads), 1, 1, 256, args, op);
}

#define SAMPLE_CHUNKS 16    /* chunks of a row at most */
#define SAMPLE_CHUNK 8192   /* logits of a chunk: at most, and 6145 at least, unless the chunks have to be fewer */
#define SAMPLE_PLACES 512   /* workgroups that the chip holds, two a CU */
int sepia_hip_sample(const SepiaSampleDesc *d, SepiaGpuBuf *logits, int64_t rows, int64_t vocab, int64_t stride,
                     SepiaGpuBuf *tokens, SepiaGpuBuf *prob) {
    const char *op = "sample";
    if (!d || !d->u || !logits || !tokens || rows < 0 || rows > MAX_SAMPLES || vocab < 1 || stride < vocab ||
        (rows > 0 && stride > INT64_MAX / 4 / rows)) {
        LOG("%s: invalid arguments", op);
        return 0;
    }
    if (vocab > (1 << 20)) {
        LOG("%s: %lld logits a row not supported (up to 2^20)", op, (long long)vocab);
        return 0;
    }
    const size_t lb = rows ? ((size_t)(rows - 1) * (size_t)stride + (size_t)vocab) * 4 : 0, rb = (size_t)rows * 4;
    SepiaGpuBuf *const in[] = { d->u, d->temperature, d->top_p, d->min_p, d->top_k };
    static const char *const names[] = { "u", "temperature", "top_p", "min_p", "top_k" };
    if (!sepia_chk(logits, 0, lb, op, "logits") || !sepia_chk(tokens, 0, rb, op, "tokens") ||
        (prob && !sepia_chk(prob, 0, rb, op, "prob")))
        return 0;
    Part p[8] = { { tokens, 0, rb, "tokens" }, { prob, 0, rb, "prob" }, { logits, 0, lb, "logits" } };
    for (int i = 0; i < 5; i++) {
        if (in[i] && !sepia_chk(in[i], 0, rb, op, names[i])) return 0;
        p[3 + i] = (Part){ in[i], 0, rb, names[i] };
    }
    if (!apart(op, p, 8, 3)) return 0;
    if (!sepia_need_batch(op) || !sepia_prep_in(logits, 0, lb, op)) return 0;
    for (int i = 0; i < 5; i++)
        if (in[i] && !sepia_prep_in(in[i], 0, rb, op)) return 0;
    if (!sepia_prep_out(tokens, op) || (prob && !sepia_prep_out(prob, op))) return 0;
    if (rows == 0) return 1;
    SampleArgs a;
    memset(&a, 0, sizeof a);
    a.logits = (const float *)sepia_buf_dev(logits);
    a.u = (const float *)sepia_buf_dev(d->u);
    a.temperature = (const float *)sepia_buf_dev(d->temperature);
    a.top_p = (const float *)sepia_buf_dev(d->top_p);
    a.min_p = (const float *)sepia_buf_dev(d->min_p);
    a.top_k = (const int32_t *)sepia_buf_dev(d->top_k);
    a.token = (int32_t *)sepia_buf_dev(tokens);
    a.prob = (float *)sepia_buf_dev(prob);
    a.stride = stride;
    a.vocab = (int32_t)vocab;
    /* chunks of a row: as many as the rows leave places for. Two more launches
     * cost 10 us, what one workgroup takes for 24000 logits: below three chunks
     * a row stays whole (1 row, 127 rows in chunks against whole: 33, 39 against
     * 27, 32 us of 11625 logits, 33, 48 against 32, 42 of 20000; 33, 52 against
     * 40, 54 of 32000). */
    int64_t chunks = (vocab + SAMPLE_CHUNK - 1) / SAMPLE_CHUNK;
    if (vocab < 3 * SAMPLE_CHUNK) chunks = 1;
    if (chunks > SAMPLE_PLACES / rows) chunks = SAMPLE_PLACES / rows;
    if (chunks > SAMPLE_CHUNKS) chunks = SAMPLE_CHUNKS;
    const size_t per = sizeof(SampleRow) + sizeof(SampleChunk) * (size_t)(chunks > 0 ? chunks : 1);
    if (chunks < 2 || (size_t)rows * per > sepia_scratch_limit()) chunks = 1;
    a.chunks = (int32_t)chunks;
    a.chunk = (int32_t)((vocab + chunks - 1) / chunks);
    void *args[] = { &a };
    if (chunks == 1) return sepia_serve_launch(SK_SAMPLE, 1, (unsigned)rows, 1, SAMPLE_NT, args, op);
    a.rows = (SampleRow *)sepia_scratch((size_t)rows * per, op);
    if (!a.rows) return 0;
    a.bins = (SampleChunk *)(a.rows + rows);
    for (int k = SK_SAMPLE_MAX; k <= SK_SAMPLE_PICK; k++)
        if (!sepia_serve_launch(k, (uint64_t)chunks, (unsigned)rows, 1, SAMPLE_NT, args, op)) return 0;
    return 1;
}
