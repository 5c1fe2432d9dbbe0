"""The tiles of the int8 product wait for their copies with hand-counted `s_waitcnt vmcnt(N)`, as the library of the quantised
GEMMs does in places: a spill's own loads and stores would count too and weaken those waits.  No other kernel of the library
has a reason to spill either.  Read from the metadata of the built library."""
from __future__ import annotations

import os
import re
import shutil
import subprocess

import pytest

LLVM = "/opt/rocm/llvm/bin"


def test_no_kernel_spills(tmp_path):
    from sonar_amd import _lib
    _lib.load_layer()
    if not os.path.exists(f"{LLVM}/llvm-objdump"):
        pytest.skip("llvm-objdump not available")
    lib = shutil.copy(_lib._LAYER_PATH, tmp_path)
    subprocess.run([f"{LLVM}/llvm-objdump", "--offloading", lib], cwd=tmp_path, capture_output=True, check=True, timeout=60)
    seen = {}
    for obj in tmp_path.glob("*gfx950*"):
        notes = subprocess.run([f"{LLVM}/llvm-readelf", "--notes", str(obj)], capture_output=True, text=True, timeout=60)
        for m in re.finditer(r"\.name:\s+(\S+).*?\.private_segment_fixed_size:\s+(\d+).*?\.vgpr_spill_count:\s+(\d+)", notes.stdout, re.S):
            kernel = re.search(r"(int8_[a-z]+_kernel|topk_routing_kernel|rms_norm_quant(?:_any)?_kernel)", m.group(1))
            assert kernel, m.group(1)
            seen[kernel.group(1)] = seen.get(kernel.group(1), 0) + 1
            assert m.group(2) == "0" and m.group(3) == "0", f"{m.group(1)}: scratch {m.group(2)}, spills {m.group(3)}"
    assert seen.get("int8_tile_kernel") == 10 and len(seen) == 8 and sum(seen.values()) >= 80
