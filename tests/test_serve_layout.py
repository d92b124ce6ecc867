"""What the serving kernels and their host share (kernels/serve_layout.h), on the CPU: the arguments are the size of the
kernels' argument segments, and neither side has a copy of its own."""
import os
import re

import pytest

import test_kernarg_warm as warm
from conftest import ROOT
from sepia_amd import hip
from test_kv8_map import build

SIZES = r'''
#include <stdio.h>
#include "serve_layout.h"
int main(void) {
    printf("%zu %zu %zu\n", sizeof(Kv8Call), sizeof(Kv8AttnCall), sizeof(SampleArgs));
    return 0;
}'''


@pytest.mark.skipif(not os.path.exists(hip.SERVE_HSACO_PATH), reason="code object not built")
def test_arguments_are_the_kernels(tmp_path, monkeypatch):
    monkeypatch.setattr(warm, "HSACO", hip.SERVE_HSACO_PATH)
    seg = warm.kernel_segments(tmp_path)
    call, attn, sample = map(int, build(tmp_path, SIZES).stdout.split())
    want = {"sepia_kv8_append": call + 3 * 8 + 4, "sepia_kv8_read": call + 2 * 8}
    for k in seg:
        if k.startswith(("sepia_kv8_attn_", "sepia_kv8_rows_")):
            want[k] = call + attn
        if k.startswith("sepia_sample"):
            want[k] = sample
    assert set(want) == set(seg)
    for k, size in want.items():   # a kernel that asks for its grid has 256 bytes more, from a multiple of 8 on
        assert seg[k] in (size, -(-size // 8) * 8 + 256), (k, seg[k], size)


def test_bins_are_aligned(tmp_path):
    """Pairs of 8-byte masses are one load of 16 bytes: the bins behind any number of rows begin at a multiple of that."""
    r = build(tmp_path, r'''
#include <stdio.h>
#include <stddef.h>
#include "serve_layout.h"
int main(void) {
    for (int rows = 1; rows < 40; rows++)
        for (int chunk = 0; chunk < 3; chunk++)
            if ((rows * sizeof(SampleRow) + chunk * sizeof(SampleChunk) + offsetof(SampleChunk, mass)) % 16) return rows;
    return 0;
}''')
    assert r.returncode == 0


def test_one_definition():
    csrc = os.path.join(ROOT, "sepia_amd", "csrc")
    shared = open(os.path.join(csrc, "kernels", "serve_layout.h")).read()
    names = re.findall(r"#define (\w+)|\} (\w+);", shared)
    names = [a or b for a, b in names]
    assert len(names) >= 8
    files = [os.path.join(csrc, "serve.c")] + [os.path.join(csrc, "kernels", f) for f in
                                               ("kv8.h", "kv8_attn.h", "kv8_map.h", "sample.h", "serve.h", "sepia_serve.hip")]
    for f in files:
        text = open(f).read()
        for n in names:
            assert not re.search(r"#define %s\b|\} %s;|struct %s\b" % (n, n, n), text), (f, n)
