"""CPU: what the layer library launches, counted by a stand-in for the runtime's launch functions that the library finds first:
no kernel runs.  A call that is refused launches nothing, whatever it is refused for."""
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
