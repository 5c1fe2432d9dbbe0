"""CPU: a deployment that ships only libsonar_marlin.so and libsonar_marlin_torch.so has every op of theirs; an operator of
the layer library raises when it is called, and says what is missing."""
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LAYER = ("libsonar_layer.so", "libsonar_layer_torch.so")

CALLS = """
import sys
import torch
from sonar_amd import fused_moe, marlin_linear, marlin_utils, ops
missing = sys.argv[1:]
assert ops.__file__.startswith(sys.path[0])
torch.ops._C.marlin_gemm, torch.ops.sonar_amd.per_token_quant_int8, ops.marlin_gemm
x = torch.zeros((2, 16))
codes = torch.zeros((2, 16), dtype=torch.int8)
for call in (lambda: ops.rms_norm_per_token_quant(x, x[0], 1e-6), lambda: ops.topk_routing(x, 2),
             lambda: ops.scaled_mm_int8(codes, codes.t(), torch.ones(2), torch.ones(2), torch.float16)):
    try:
        call()
    except ImportError as e:
        assert missing and all(name in str(e) for name in missing) and "sonar_amd.build" in str(e), e
    except NotImplementedError:   # (the ops are there, and take GPU tensors)
        assert not missing
    else:
        raise AssertionError("no error")
weights, ids = fused_moe.fused_topk(x, x, 2, True)
assert ids.tolist() == [[0, 1]] * 2
print("done")
"""


@pytest.mark.parametrize("missing", [(), LAYER, LAYER[:1], LAYER[1:]], ids=lambda names: "+".join(names) or "none")
def test_gemms_without_the_layer_libraries(missing, tmp_path):
    from sonar_amd import _lib
    package = tmp_path / "sonar_amd"
    (package / "lib").mkdir(parents=True)
    for name in os.listdir(os.path.join(ROOT, "sonar_amd")):
        if name.endswith(".py"):
            shutil.copy(os.path.join(ROOT, "sonar_amd", name), package)
    lib = os.path.dirname(_lib.lib_path())
    for name in os.listdir(lib):
        if name.endswith(".so") and name not in missing:
            shutil.copy(os.path.join(lib, name), package / "lib")
    run = subprocess.run([sys.executable, "-c", f"import sys; sys.path.insert(0, {str(tmp_path)!r})\n" + CALLS, *missing], cwd=tmp_path,
                         capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.strip().endswith("done"), run.stderr[-2000:]
