"""Where the rows of a cache call lie (kernels/kv8_map.h), in a CPU build: every new row falls to exactly one unit of
the id space that the grid counts in, units stay inside their page, and sequences that cannot be used are refused.
Also the serving structs' layout, and the calls' refusals before a device is there."""
import ctypes
import os
import subprocess
import sys

import pytest

from conftest import ROOT
from sepia_amd import hip

KDIR = os.path.join(ROOT, "sepia_amd", "csrc", "kernels")

MAP = r'''
#include <stdio.h>
#include <stdlib.h>
#include "kv8_map.h"
static int find(const int *starts, int n_seqs, long id, int gran, int extra) {   /* the last that begins at or before id */
    int s = -1;
    for (int i = 0; i < n_seqs; i++) if (kv8_first_id(starts[i], i, gran, extra) <= id) s = i;
    return s;
}
int main(void) {
    srand(7);
    for (int round = 0; round < 4000; round++) {
        const int lg = 4 + rand() % 3, P = 1 << lg, n_seqs = 1 + rand() % 9, before = rand() % 4, behind = rand() % 40;
        int starts[10], lens[9], n = before;
        for (int s = 0; s < n_seqs; s++) {
            lens[s] = rand() % 3 ? rand() % 300 : P * (rand() % 4);
            starts[s] = n;
            n += rand() % 4 ? rand() % 150 : 0;
        }
        starts[n_seqs] = n;
        n += behind;
        unsigned char *seen = calloc(n + 1, 1);
        const int gran = round % 2 ? P : 1, extra = round % 2 ? 2 : 0;   /* both id spaces of the pages */
        const long ids = kv8_ids(n, n_seqs, gran, extra);
        for (long id = 0; id < ids; id++) {
            const int s = find(starts, n_seqs, id, gran, extra);
            Kv8Unit u;
            if (s < 0) continue;
            if (!kv8_unit(lens[s], starts[s], starts[s + 1], (int)(id - kv8_first_id(starts[s], s, gran, extra)), lg, &u)) continue;
            if (u.s0 < 0 || u.s0 >= u.s1 || u.s1 > P) return 1;
            for (int i = u.s0; i < u.s1; i++) {
                const int row = u.row + i - u.s0;
                if (row < starts[s] || row >= starts[s + 1] || seen[row]++) return 2;
                if (lens[s] + row - starts[s] != (u.page << lg) + i) return 3;
            }
        }
        for (int r = 0; r < n; r++) if (seen[r] != (r >= starts[0] && r < starts[n_seqs])) return 4;
        free(seen);
    }
    if (!kv8_seq_ok(0, 0, 0, 0, 16) || !kv8_seq_ok(15, 3, 4, 4, 16) || kv8_seq_ok(16, 3, 4, 4, 16) || kv8_seq_ok(-1, 0, 1, 4, 16) ||
        kv8_seq_ok(0, 2, 1, 4, 16) || kv8_seq_ok(0, -1, 1, 4, 16) || kv8_seq_ok(0, 3, 5, 4, 16) ||
        kv8_seq_ok(2147483647, 0, 4, 4, 2147483647)) return 5;
    puts("ok");
    return 0;
}
'''


def build(tmp_path, text, *flags):
    c, exe = tmp_path / "t.c", tmp_path / "t"
    c.write_text(text)
    subprocess.run(["gcc", "-std=c11", "-O1", "-Wall", "-I" + hip.INCLUDE_DIR, "-I" + KDIR, *flags, "-o", str(exe), str(c)],
                   check=True)
    return subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)


def test_units_cover_every_row_once(tmp_path):
    r = build(tmp_path, MAP, "-fsanitize=address,undefined")
    assert r.returncode == 0 and r.stdout.strip() == "ok", (r.returncode, r.stderr[-500:])


def test_struct_layout(tmp_path):
    r = build(tmp_path, r'''
#include <stdio.h>
#include <stddef.h>
#include "sepia_hip_ext.h"
int main(void) {
    printf("%zu %zu %zu %zu %zu %zu %zu\n", sizeof(SepiaKv8Cache), offsetof(SepiaKv8Cache, n_seqs), offsetof(SepiaKv8Cache, page),
           offsetof(SepiaKv8Cache, codes), offsetof(SepiaKv8Cache, table_off), sizeof(SepiaSampleDesc), offsetof(SepiaSampleDesc, top_k));
    return 0;
}''')
    C, S = hip.Kv8Cache, hip.SampleDesc
    assert list(map(int, r.stdout.split())) == [ctypes.sizeof(C), C.n_seqs.offset, C.page.offset, C.codes.offset,
                                                C.table_off.offset, ctypes.sizeof(S), S.top_k.offset]


def test_code_object_has_every_serving_kernel():
    src = open(os.path.join(ROOT, "sepia_amd", "csrc", "sepia_hip.c")).read()
    import re
    names = re.findall(r'"(sepia_[a-z0-9_]+)"', src.split("serve_names[SK_COUNT]")[1].split("};")[0])
    blob = open(hip.SERVE_HSACO_PATH, "rb").read()
    assert len(names) >= 4
    for n in names:
        assert (n + ".kd").encode() in blob, n


@pytest.mark.skipif(os.path.exists("/dev/kfd"), reason="checks the no-device path")
def test_no_device():
    """Every call refuses with a log line and 0, whatever it is given, and never ends the process."""
    code = r'''
import ctypes
from sepia_amd import hip
L = hip.load()
c = hip.Kv8Cache(n_pages=4, max_pages=4, n_seqs=1, n_kv_heads=2, head_dim=64, page=16)
d = hip.SampleDesc()
B = ctypes.byref
for cache in (None, B(c), B(hip.Kv8Cache()), B(hip.Kv8Cache(n_pages=1, max_pages=1, n_seqs=1, n_kv_heads=1, head_dim=-16, page=16))):
    assert L.sepia_hip_kv8_append(cache, None, None, 1, None, None, None, 0.0) == 0
    assert L.sepia_hip_kv8_read(cache, None, None, 1, None, None) == 0
    assert L.sepia_hip_kv8_attn(cache, None, None, 1, None, None, None, None, 4, 0, 0, 1.0) == 0
for desc in (None, B(d)):
    assert L.sepia_hip_sample(desc, None, 1, 10, 10, None, None) == 0
print("ok")
'''
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=ROOT, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stderr
    assert r.stderr.count("sepia: hip:") == 14
