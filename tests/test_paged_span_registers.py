"""The kernel of few rows over a paged cache of 16 bits keeps its state in registers.  Where a change of its source makes
the compiler spill some, decoding slows down by up to a tenth (64 x 3000 keys, 24 heads over 8 of 128, fp16: 113 -> 125 us)
with the same results."""
from __future__ import annotations

import concurrent.futures as cf
import os
import re
import shutil
import subprocess

import pytest

from cdml import build as B

pytestmark = pytest.mark.skipif(not shutil.which(B.HIPCC), reason="no hipcc")


def spills(name):
    """{kernel: spilled registers} of the kernels of few rows in a source."""
    r = subprocess.run([B.HIPCC, *B.HIP_FLAGS, "--cuda-device-only", "-Rpass-analysis=kernel-resource-usage", "-c",
                        os.path.join(B.CSRC, name + ".hip"), "-o", os.devnull], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    kernel, found = None, {}
    for line in r.stderr.splitlines():
        if m := re.search(r"Function Name: (\S+)", line):
            kernel = m.group(1) if "paged_span_kernel" in m.group(1) else None
        elif kernel and (m := re.search(r"VGPRs Spill: (\d+)", line)):
            found[kernel] = int(m.group(1))
    return found


def test_no_spills():
    with cf.ThreadPoolExecutor(2) as ex:
        for found in ex.map(spills, ["paged_attn_bf16", "paged_attn_f16"]):
            assert len(found) == 6  # three head dims, aligned rows or not
            assert not any(found.values()), found
