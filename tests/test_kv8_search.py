"""The search for the sequence that an id belongs to (kv8_find in kernels/kv8.h, a wave's lanes counted one by one here),
in a CPU build of kernels/kv8_map.h: with starts that rise it finds the owner, and with starts that fall, which a call
may be handed, no unit of what it finds lies outside the sequence's pages, rows and table."""
import os

from test_kv8_map import KDIR, build

SEARCH = r'''
#include <stdio.h>
#include <stdlib.h>
#include "kv8_map.h"
/* kv8_find: 64 sequences a look; -1 where no sequence begins at or before the id */
static int find(const int *starts, int n_seqs, long id, int gran, int extra) {
    int lo = 0, n = n_seqs;
    while (1) {
        const int step = (n + 63) / 64;
        int c = 0;
        for (int lane = 0; lane < 64; lane++) {
            const int i = lane * step, s = lo + (i < n - 1 ? i : n - 1);
            c += i < n && kv8_first_id(starts[s], s, gran, extra) <= id;
        }
        if (c == 0) return -1;
        if (step == 1) return lo + c - 1;
        lo += (c - 1) * step;
        n = step < n - (c - 1) * step ? step : n - (c - 1) * step;
    }
}
static int starts[5001], lens[5000];
int main(void) {
    srand(3);
    long used = 0, passed = 0;
    for (int round = 0; round < 1500; round++) {
        const int lg = 4 + rand() % 3, P = 1 << lg, n_seqs = round % 10 ? 1 + rand() % 9 : 1 + rand() % 5000;
        const int falling = round & 1, n = 1 + rand() % 300;
        const long capacity = 640;
        int at = 0;
        for (int s = 0; s <= n_seqs; s++) {
            if (s < n_seqs) lens[s] = rand() % 400;
            starts[s] = falling ? rand() % (n + 1) : at;
            at += at < n && rand() % 3 ? rand() % (n - at + 1) / 2 : 0;
        }
        const int tile = 1 + rand() % 16;
        for (int space = 0; space < 3; space++) {   /* both id spaces of the pages, and the row tiles' */
            const int gran = space == 0 ? 1 : space == 1 ? P : 4 * tile, extra = space == 0 ? 0 : space == 1 ? 2 : 1;
            for (long id = 0; id < kv8_ids(n, n_seqs, gran, extra); id++) {
                const int s = find(starts, n_seqs, id, gran, extra);
                if (s < 0) continue;
                if (s >= n_seqs) return 1;
                const int r0 = starts[s], r1 = starts[s + 1];
                int k;
                if (!kv8_place(id, r0, s, gran, extra, &k)) {
                    if (!falling) return 2;
                    passed++;
                    continue;
                }
                if (!kv8_seq_ok(lens[s], r0, r1, n, capacity)) {
                    if (!falling) return 3;
                    continue;
                }
                if (space == 2) {   /* the four tiles of a workgroup: the first row, where there is one */
                    for (int w = 0; w < 4; w++) {
                        const long row = (long)(k * 4 + w) * tile;
                        if (row < r1 - r0 && (row < 0 || r0 + row >= n)) return 4;
                    }
                } else {
                    Kv8Unit u;
                    if (!kv8_unit(lens[s], r0, r1, k, lg, &u)) continue;
                    if (u.page < 0 || (long)(u.page + 1) * P > capacity || u.s0 < 0 || u.s0 >= u.s1 || u.s1 > P) return 5;
                    if (u.row < r0 || u.row + u.s1 - u.s0 > r1) return 6;
                }
                used++;
            }
        }
    }
    printf("%d\n", used > 10000 && passed > 1000);
    return 0;
}
'''


def test_search_stays_inside(tmp_path):
    r = build(tmp_path, SEARCH, "-fsanitize=address,undefined")
    assert r.returncode == 0 and r.stdout.strip() == "1", (r.returncode, r.stdout, r.stderr[-500:])


def test_steps_of_the_longest_sequences(tmp_path):
    """The attention's steps of 64 columns, up to the last length that a table can hold (2^31 - 16 tokens): no sum on the
    way passes 32 bits."""
    r = build(tmp_path, r'''
#include <stdio.h>
#include "kv8_map.h"
int main(void) {
    const int32_t top = 2147483647;
    for (int32_t end = 1; end < 5000; end++) {
        if (kv8_steps(end) != (end + 63) / 64) return 1;
        if (kv8_steps(top - end) != (int32_t)(((int64_t)top - end + 63) / 64)) return 2;
    }
    puts("ok");
    return 0;
}''', "-fsanitize=undefined", "-fno-sanitize-recover")
    assert r.returncode == 0 and r.stdout.strip() == "ok", (r.returncode, r.stderr[-300:])
    text = open(os.path.join(KDIR, "kv8_attn.h")).read()
    assert "steps = kv8_steps(len + (r1 - r0));" in text
