"""Which of an attention call's kernels runs (csrc/kv8_route.h), in a CPU build that ends at undefined arithmetic."""
import os

import pytest

from conftest import ROOT
from test_kv8_map import build

CALL = "n", "n_seqs", "kv_heads", "tt", "max_pages", "page", "window", "sinks", "tree", "pair"
FORMS = "runs", "rows", "pair"
TOP = 2 ** 31 - 1


def route(tmp_path, calls):
    """[(form, window, sinks, units, steps, budget)] of the calls, tuples of CALL."""
    rows = ",\n".join("{ %s }" % ", ".join("%dLL" % v for v in c) for c in calls)
    r = build(tmp_path, r'''
#include <stdio.h>
#include "kv8_route.h"
static const long long calls[][10] = { %s };
int main(void) {
    for (unsigned i = 0; i < sizeof calls / sizeof calls[0]; i++) {
        const long long *c = calls[i];
        const Kv8Route r = kv8_route(c[0], c[1], c[2], c[3], c[4], c[5], c[6], c[7], (int)c[8], (int)c[9]);
        printf("%%d %%d %%d %%lld %%lld %%lld\n", r.form, r.window, r.sinks, (long long)r.units, (long long)r.steps, (long long)r.budget);
    }
    return 0;
}''' % rows, "-I" + os.path.join(ROOT, "sepia_amd", "csrc"), "-fsanitize=undefined", "-fno-sanitize-recover")
    assert r.returncode == 0, r.stderr[-500:]
    out = [[int(v) for v in line.split()] for line in r.stdout.splitlines()]
    assert len(out) == len(calls)
    return [(FORMS[o[0]],) + tuple(o[1:]) for o in out]


def steps_of(max_pages, page, window, sinks, tree):
    """A unit's steps of 64 columns at most, in whole numbers of any size."""
    window = 0 if window > TOP else window
    wide = window // 64 + 2 + -(-min(sinks, TOP) // 64) + tree
    return min(-(-max_pages * page // 64), wide) if window else -(-max_pages * page // 64)


@pytest.mark.parametrize("sinks", [0, 1, 64, 65, TOP - 64, TOP - 63, TOP - 62, TOP - 1, TOP, TOP + 1, 2 ** 40, 2 ** 62])
def test_steps_of_many_sinks(tmp_path, sinks):
    """Sinks up to the largest number leave a unit the table's steps, so that long units are cut, and only short ones go
    two to a workgroup or (trees) a wave each."""
    calls = [(n, seqs, 8, 2, pages, 16, window, sinks, tree, 1)
             for n, seqs in ((1, 1), (25, 1), (160, 5), (300, 12), (600, 12), (4000, 300)) for pages in (8, 600, 2000, TOP // 16)
             for window in (1, 100, 5000, TOP - 1, TOP, 2 ** 40) for tree in (0, 1)]
    for c, (form, window, kept, units, steps, budget) in zip(calls, route(tmp_path, calls)):
        call = dict(zip(CALL, c))
        n, pages, tree = call["n"], call["max_pages"], call["tree"]
        assert window == (0 if call["window"] > TOP else call["window"]) and kept == (min(sinks, TOP) if window else 0)
        assert units == 8 * max(n // 2, min(n, call["n_seqs"]))
        assert steps == steps_of(pages, 16, call["window"], sinks, tree) and steps > 0, call
        long = steps > 32
        if units >= 1024 and not (tree and long and units < 8192 and call["n_seqs"] <= 256):
            assert form == "rows", call
        elif units > 512 and not long:
            assert form == "pair", call
        else:
            assert form == "runs" and (budget > 0) == (steps > 4), call


def test_routes(tmp_path):
    """Two rows a sequence's tile, 8 kv heads, tables of 9600 columns."""
    want = [
        ((64, 64, 8, 2, 600, 16, 512, 4, 0, 1), "runs"), ((65, 65, 8, 2, 600, 16, 512, 4, 0, 1), "pair"),
        ((65, 65, 8, 2, 600, 16, 512, 4, 0, 0), "runs"), ((65, 65, 8, 2, 600, 16, 5000, 4, 0, 1), "runs"),
        ((65, 65, 8, 2, 600, 16, 512, 2 ** 40, 0, 1), "runs"), ((127, 127, 8, 2, 600, 16, 512, 4, 0, 1), "pair"),
        ((128, 128, 8, 2, 600, 16, 512, 4, 0, 1), "rows"), ((300, 9, 8, 2, 600, 16, 0, 0, 1, 1), "runs"),
        ((300, 9, 8, 2, 600, 16, 300, 5, 1, 1), "rows"), ((300, 257, 8, 2, 600, 16, 0, 0, 1, 1), "rows"),
        ((2046, 9, 8, 2, 600, 16, 0, 0, 1, 1), "runs"), ((2048, 9, 8, 2, 600, 16, 0, 0, 1, 1), "rows"),
        ((200, 9, 8, 2, 600, 16, 300, 5, 1, 1), "pair"),
    ]
    assert [r[0] for r in route(tmp_path, [c for c, _ in want])] == [f for _, f in want]


def test_every_kernel_has_a_case(tmp_path):
    """The GPU tests' cases that are compared with the restatement reach all kernels of attention with sinks and over
    trees, and each of test_gpu_kv8_routes the one that it is meant for."""
    from test_gpu_kv8_masked import SINKS, TREES
    from test_gpu_kv8_routes import CASES, KERNELS
    cases = [("sinks",) + c for c in SINKS] + [("tree",) + c for c in TREES] + CASES
    calls, names = [], []
    for sees, H, heads, dim, page, lens, news, window, sinks, _ in cases:
        sees = sees.split("_")[0]
        n = H % 2 + sum(news) + H % 3
        pages = 1 + max(1, max(-(-(a + b) // page) for a, b in zip(lens, news)))   # test_gpu_kv8.make's table
        calls.append((n, len(lens), heads, 16 // (H // heads), pages, page, window, sinks, sees == "tree", 1))
        names.append((sees, ("" if dim % 64 == 0 else "to") + ("64" if dim <= 64 else "128")))
    reached = ["sepia_kv8_%s_%s_%s" % (sees, "attn" if r[0] == "runs" else r[0], dim) for (sees, dim), r in zip(names, route(tmp_path, calls))]
    assert set(reached) == set(KERNELS)
    assert reached[-len(CASES):] == ["sepia_kv8_" + c[0] for c in CASES]
