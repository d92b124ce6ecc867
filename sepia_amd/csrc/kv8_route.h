/* kv8_route.h -- which of an attention call's kernels (kernels/kv8_attn.h) runs,
 * and into how many runs its units are cut: plain integer code for the host
 * (serve.c), and for a build that checks it. A unit is a (row tile, kv head).
 * The lengths are on the device: a unit's steps are counted from the table's
 * width and the window, so a table much wider than its sequences makes their
 * units look long. */
#ifndef SEPIA_KV8_ROUTE_H
#define SEPIA_KV8_ROUTE_H
#include <stdint.h>

#include "kernels/serve_layout.h"

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
/* Steps of 64 columns up to which a unit is short. Short units that are more than
 * the chip holds workgroups go two to a workgroup, one round for two (40 single
 * tokens, 16 kv heads, window 512: 25.5 us against 27.5 with one; 9 trees of 64
 * rows, dim 64, window 300: 17.9 against 22.2). Trees' units that are not short
 * are cut into runs up to KV8_TREES of them: a wave alone with the longest takes
 * that long (24 trees of up to 33 rows behind up to 6000 columns: 183 us against
 * 233 a wave a unit; 50 behind 4000 238 against 269; 100 behind 3000, 13000 units,
 * 448 against 444; 200 behind 2500 780 against 671), and of up to KV8_TREES / 32
 * sequences, which every workgroup walks through (300 of 9 rows 424 against 429,
 * 600 of 5 542 against 485). Where this rule goes wrong, for all that it does not know:
 * one tree of 25 rows behind 20001 columns, in a call of 1800 rows and 256 slots 116
 * us, of 257 slots 493 (a wave a unit); 250 of 9 rows ragged up to 12000 columns 930 and
 * 1094. And trees of 9 or 33 rows behind 200 columns whose table has room for 32768,
 * so that they look long: 40 of 9 21.5 us against 19.6 with a table of their width, 40
 * of 33 63.7 against 38.6 (dim 64: 29.7 against 22.5), 100 of 9 54 against 35. */
#define KV8_LONG 32
#define KV8_TREES 8192

enum { KV8_RUNS_FORM, KV8_ROWS_FORM, KV8_PAIR_FORM };   /* cut into runs, a wave a unit, two units a workgroup */
typedef struct {
    int form;
    int32_t window, sinks;   /* as the kernels take them: 0 for a window that nothing is outside of */
    int64_t units, steps;    /* steps of 64 columns of a unit, at most */
    int64_t budget;          /* KV8_RUNS_FORM: runs besides one a unit; 0: no unit is cut */
} Kv8Route;
/* n rows of n_seqs sequences in tiles of tt tokens, a table of max_pages pages of
 * `page` tokens a sequence (at most 2^31 - 1 tokens). tree: the rows are trees'.
 * pair: there are kernels of two units a workgroup. */
static inline Kv8Route kv8_route(int64_t n, int64_t n_seqs, int64_t kv_heads, int64_t tt, int64_t max_pages, int64_t page,
                                 int64_t window, int64_t sinks, int tree, int pair) {
    Kv8Route r = { KV8_RUNS_FORM, window > 0x7FFFFFFF ? 0 : (int32_t)window, 0, 0, 0, 0 };
    r.sinks = !r.window ? 0 : sinks > 0x7FFFFFFF ? 0x7FFFFFFF : (int32_t)sinks;   /* without a window all is seen */
    r.units = (n / tt > n_seqs ? n / tt : n < n_seqs ? n : n_seqs) * kv_heads;
    r.steps = (max_pages * page + 63) / 64;
    const int64_t wide = (int64_t)r.window / 64 + 2 + ((int64_t)r.sinks + 63) / 64 + tree;   /* a tree's rows end 63 columns apart */
    if (r.window > 0 && wide < r.steps) r.steps = wide;
    const int cut = tree && r.steps > KV8_LONG && r.units < KV8_TREES && n_seqs <= KV8_TREES / 32;
    if (r.units >= KV8_ROWS && !cut) {
        r.form = KV8_ROWS_FORM;
        return r;
    }
    if (pair && r.units > KV8_BUDGET && r.steps <= KV8_LONG) {
        r.form = KV8_PAIR_FORM;
        return r;
    }
    /* No more runs than places: a unit's last run is short, so as many fewer as
     * there are units (a whole round more for a few runs: 4 sequences of up to
     * 8000 columns, 8 kv heads and a band of 1024, 16.4 us against 18.2 with 512
     * runs). Half as many again as places where a run may be long, since units of
     * ragged lengths end unevenly (48 sequences of up to 12000 columns: 118.5 us
     * against 134.3 with 512; where runs are short they cost: 32 sequences in a
     * window of 512, 16 kv heads, 18.5 us against 28.5). Not for trees whose units
     * are likely to be as long as their neighbours, which 8 row tiles a sequence on
     * average are taken for (one tree of 60 rows behind 20001
     * columns 125.5 us against 144, 12 of up to 33 behind 6000 104.5 against 110;
     * 12 of up to 9 behind 20000 106 against 90, so they keep it). None, and no scratch,
     * where a run has every step that the table or the window leaves a unit (as
     * long either way). */
    r.budget = KV8_BUDGET - (r.units < KV8_BUDGET / 2 ? r.units : KV8_BUDGET / 2);
    const int even = tree && (n_seqs == 1 || n / tt >= 8 * n_seqs);
    if (r.units * r.steps / KV8_BUDGET > 64 && !even) r.budget = KV8_BUDGET * 3 / 2;
    if (r.steps <= KV8_NW) r.budget = 0;
    return r;
}
#endif
