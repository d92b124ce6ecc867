"""The serving kernels' argument warm-up reads only inside each kernel's argument segment.

serve_args<BYTES>() (kernels/serve.h) reads a word of every 64-byte line of the first BYTES of the kernel's argument
segment, whose size the compiler records in the code object. CPU only: it reads the build's output."""
import os
import re

import pytest

import test_kernarg_warm as warm
from sepia_amd import hip

# the kernels that a file's warm-ups are compiled into, by the function that holds the call
HOLDERS = {"sepia_kv8_append": "sepia_kv8_append", "sepia_kv8_read": "sepia_kv8_read",
           "kv8_attn_run": "sepia_kv8_attn_", "kv8_attn_rows": "sepia_kv8_rows_", "sepia_sample_max": "sepia_sample_max", "sepia_sample_bins": "sepia_sample_bins",
           "sepia_sample_pick": "sepia_sample_pick", "sepia_sample": "sepia_sample"}


@pytest.mark.skipif(not os.path.exists(hip.SERVE_HSACO_PATH), reason="code object not built")
def test_serve_args_within_segment(tmp_path, monkeypatch):
    monkeypatch.setattr(warm, "HSACO", hip.SERVE_HSACO_PATH)
    seg = warm.kernel_segments(tmp_path)
    assert len(seg) == 14, sorted(seg)
    seen = set()
    for name in ("kv8.h", "kv8_attn.h", "sample.h"):
        text = open(os.path.join(warm.KDIR, name)).read()
        for m in re.finditer(r"serve_args<(\d+)>\(\);", text):
            holder = re.findall(r"void (\w+)\(", text[:m.start()])[-1]
            name = HOLDERS[holder]
            kernels = [k for k in seg if k == name or name[-1] == "_" and k.startswith(name)]
            assert kernels, holder
            for k in kernels:
                assert int(m.group(1)) <= seg[k], (k, m.group(1), seg[k])
            seen.add(holder)
    assert seen == set(HOLDERS)
