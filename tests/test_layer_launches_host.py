"""CPU: which kernels the layer library takes and launches.  Launches are counted by a stand-in for the runtime's launch
functions that the library finds first: no kernel runs."""
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

STAND_IN = """
int launches;
int __hipPushCallConfiguration(void) { return 0; }
int __hipPopCallConfiguration(void) { return 0; }
int hipLaunchKernel(const void *f, ...) { (void)f; ++launches; return 0; }
int hipFuncSetAttribute(const void *f, int attribute, int value) { (void)f; (void)attribute; (void)value; return 0; }
int hipGetLastError(void) { return 0; }
"""

CALLS = """
import ctypes, sys
sys.path.insert(0, sys.argv[1])
stand_in = ctypes.CDLL(sys.argv[2], mode=ctypes.RTLD_GLOBAL)
from sonar_amd import _lib
lib = _lib.load_layer()
launches = ctypes.c_int.in_dll(stand_in, "launches")
AT = 1 << 20   # a device address that nothing looks at
def product(m, n, k, scratch=1 << 60, a_len=1, at=AT):
    before = launches.value
    rc = lib.sonar_scaled_mm_int8(at, k, AT, k, AT, AT, a_len, AT, 1, None, AT if scratch else None, scratch, 1, m, n, k, None)
    return rc, launches.value - before, lib.sonar_layer_last_error().decode()
def form(number, splits=1):
    assert lib.sonar_debug_int8_form(number, splits) == 0
# calls that run: one kernel, a join behind it, copies of unaligned rows before it
assert product(1, 4096, 4096)[:2] == (0, 1) and product(64, 256, 14336)[:2] == (0, 2)
assert product(300, 4096, 4095)[:2] == (0, 2) and product(300, 4096, 4095, scratch=0)[:2] == (0, 1)
# more tiles than a launch takes: with aligned copies first, without, split, and where no tile takes the rows
side = 1 << 20
def refused(*args, **more):
    rc, launched, text = product(*args, **more)
    assert rc == _lib.E_INVALID and launched == 0 and "tiles" in text, (args, more, rc, launched, text)
refused(side, side, 17)
refused(side, side, 17, scratch=0)
refused(side, side, 16)
refused(side, 1 << 15, 8)
for number in (0, 4, 5, 6, 7, 8):
    form(number)
    refused(side, side, 17)
    refused(side, side, 16)
form(4, 8)
refused(1 << 17, 1 << 17, 8192)
refused(1 << 17, 1 << 17, 8191)
form(2)
rc, launched, text = product(17, 4096, 4095)
assert rc == _lib.E_INVALID and launched == 0 and "rows" in text
form(-1)
for args, more in (((4, 64, 131072), {}), ((4, 64, 4095), dict(a_len=3)), ((300, 4096, 4095), dict(at=None))):
    rc, launched, _ = product(*args, **more)
    assert rc == _lib.E_INVALID and launched == 0, args
print("done")
"""


def test_a_refused_product_launches_nothing(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not available")
    (tmp_path / "stand_in.c").write_text(STAND_IN)
    library = str(tmp_path / "stand_in.so")
    subprocess.run([gcc, "-shared", "-fPIC", "-o", library, str(tmp_path / "stand_in.c")], check=True, timeout=60)
    run = subprocess.run([sys.executable, "-c", CALLS, ROOT, library], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and run.stdout.strip() == "done", run.stderr[-2000:]


def test_the_rule_counts_what_aligned_copies_move():
    """Rows that are laid down for the tiles are written to whole rounds of K, 256 bytes at least, and multiplied over them: for a
    short K that is many times the operands.  What was measured to be fastest there, and near there."""
    from sonar_amd import _lib
    lib = _lib.load_layer()
    for m, n, k in ((64, 1 << 20, 33), (64, 200000, 33), (48, 400000, 200), (64, 200000, 513), (100, 6144, 300)):
        assert lib.sonar_debug_int8_choice(m, n, k, 0, None) == 0, (m, n, k)   # the general kernel, on the rows as they lie
        assert lib.sonar_scaled_mm_int8_scratch_bytes(m, n, k, 0) == 0
    for m, n, k in ((83, 802, 29), (113, 270, 164)):
        assert lib.sonar_debug_int8_choice(m, n, k, 0, None) == 3, (m, n, k)   # the stream in blocks of 32 rows
    for m, n, k in ((200, 100000, 100), (1000, 50000, 60), (1 << 18, 512, 40), (300, 4096, 4095)):
        assert lib.sonar_debug_int8_choice(m, n, k, 0, None) >= 4, (m, n, k)   # tiles of copies
