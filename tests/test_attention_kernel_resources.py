"""The kernels of the attention library: those with copies straight into LDS wait for them with `s_waitcnt vmcnt(0)`, so that a spill
could not weaken a wait, but none of them has a reason to spill either.  Read from the metadata of the built library; and every
kernel in it has a form that the GPU tests launch."""
from __future__ import annotations

import collections
import os
import re
import shutil
import subprocess

import pytest

LLVM = "/opt/rocm/llvm/bin"
# types (f16, bf16; the rotation fp32 too) x widths x caches x scores
KERNEL_FORMS = {"qk_norm_rope_kernel": 9, "qk_norm_rope_any_kernel": 3, "attention_few_kernel": 36, "attention_rows_kernel": 48,
                "attention_join_kernel": 12}


def test_no_kernel_spills(tmp_path):
    from sonar_amd import _lib
    _lib.load_attention()
    if not os.path.exists(f"{LLVM}/llvm-objdump"):
        pytest.skip("llvm-objdump not available")
    lib = shutil.copy(_lib.attention_path(), tmp_path)
    subprocess.run([f"{LLVM}/llvm-objdump", "--offloading", lib], cwd=tmp_path, capture_output=True, check=True, timeout=60)
    seen = collections.Counter()
    for obj in tmp_path.glob("*gfx950*"):
        notes = subprocess.run([f"{LLVM}/llvm-readelf", "--notes", str(obj)], capture_output=True, text=True, timeout=60)
        for m in re.finditer(r"\.name:\s+(\S+).*?\.private_segment_fixed_size:\s+(\d+).*?\.vgpr_spill_count:\s+(\d+)", notes.stdout, re.S):
            kernel = re.search("|".join(sorted(KERNEL_FORMS, key=len, reverse=True)), m.group(1))
            assert kernel, m.group(1)
            seen[kernel.group(0)] += 1
            assert m.group(2) == "0" and m.group(3) == "0", f"{m.group(1)}: scratch {m.group(2)}, spills {m.group(3)}"
    assert dict(seen) == KERNEL_FORMS
