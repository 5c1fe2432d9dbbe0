"""CPU: the operators around the GEMMs without a GPU - the C ABI's list and its refusals (they come before anything is
launched), the ops' schemas and fake results, the router as torch expressions, and the oracle's own values."""
import collections
import math
import os
import re
import shutil
import subprocess

import numpy as np
import pytest
import torch

from oracle import layer_oracle as lo

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAKE = 1 << 20   # a device address that no refused call looks at


def layer():
    from sonar_amd import _lib
    return _lib, _lib.load_layer()


def test_header_prototypes_and_exports_agree():
    _lib, lib = layer()
    header = open(os.path.join(ROOT, "include", "sonar_layer.h")).read()
    declared = set(re.findall(r"^(?:int|size_t|const char\*)\s+(sonar_\w+)\(", header, re.M))
    assert declared == set(_lib.LAYER_PROTOTYPES)
    for name in declared:
        assert getattr(lib, name)
    assert int(re.search(r"SONAR_SCORING_SIGMOID (\d)", header).group(1)) == _lib.SCORING_SIGMOID


# ---------------------------------------------------------------- refusals
def norm_call(lib, **change):
    a = dict(x=FAKE, x_stride=64, residual=FAKE, residual_stride=64, weight=FAKE, residual_out=FAKE, norm_out=None, q=FAKE,
             q_dtype=0, scales=FAKE, dtype=1, rows=4, cols=64, epsilon=1e-6)
    a.update(change)
    return lib.sonar_rms_norm_per_token_quant(*a.values(), None)


@pytest.mark.parametrize("change,message", [
    (dict(rows=-1), "rows"), (dict(rows=1 << 31), "rows"), (dict(cols=0), "cols"), (dict(cols=1 << 30), "cols"),
    (dict(dtype=3), "dtype"), (dict(q_dtype=2), "q_dtype"), (dict(x_stride=63), "x_row_stride"),
    (dict(residual_stride=63), "residual_row_stride"), (dict(epsilon=0.0), "epsilon"), (dict(epsilon=-1e-6), "epsilon"),
    (dict(epsilon=float("nan")), "epsilon"), (dict(epsilon=1e-39), "epsilon"), (dict(epsilon=float("inf")), "epsilon"),
    (dict(x=None), "NULL"), (dict(weight=None), "NULL"), (dict(q=None), "NULL"), (dict(scales=None), "NULL"),
    (dict(residual_out=None), "together"), (dict(residual=None), "together")])
def test_norm_refuses(change, message):
    _lib, lib = layer()
    rc = norm_call(lib, **change)
    assert rc == _lib.E_INVALID and message in lib.sonar_layer_last_error().decode()
    with pytest.raises(_lib.SonarMarlinError, match=message):
        _lib.check_layer(rc)


def mm_call(lib, **change):
    a = dict(a=FAKE, lda=128, b=FAKE, ldb=128, c=FAKE, a_scales=FAKE, a_len=8, b_scales=FAKE, b_len=16, bias=None, scratch=None,
             scratch_bytes=0, dtype=1, m=8, n=16, k=128)
    a.update(change)
    return lib.sonar_scaled_mm_int8(*a.values(), None)


@pytest.mark.parametrize("change,message", [
    (dict(dtype=2), "dtype"), (dict(m=-1), "size_m"), (dict(n=-1), "size_n"), (dict(m=1 << 31), "size_m"), (dict(k=-1), "size_k"),
    (dict(k=131072, lda=131072, ldb=131072), "131072"), (dict(a=None), "NULL"), (dict(b=None), "NULL"), (dict(c=None), "NULL"),
    (dict(a_scales=None), "NULL"), (dict(b_scales=None), "NULL"), (dict(lda=127), "strides"), (dict(ldb=127), "strides"),
    (dict(a_len=7), "a_scales"), (dict(a_len=0), "a_scales"), (dict(b_len=15), "b_scales"), (dict(b_len=17), "b_scales")])
def test_int8_product_refuses(change, message):
    _lib, lib = layer()
    assert mm_call(lib, **change) == _lib.E_INVALID and message in lib.sonar_layer_last_error().decode()


def route_call(lib, **change):
    a = dict(logits=FAKE, dtype=2, stride=64, bias=None, weights=FAKE, ids=FAKE, tokens=4, experts=64, topk=4, scoring=0,
             renormalize=1, groups=1, kept=1, factor=1.0)
    a.update(change)
    return lib.sonar_topk_routing(*a.values(), None)


@pytest.mark.parametrize("change,message", [
    (dict(tokens=-1), "tokens"), (dict(experts=0), "experts"), (dict(experts=1025, stride=1025), "experts"), (dict(topk=0), "topk"),
    (dict(topk=65), "topk"), (dict(experts=3, topk=4), "topk"), (dict(groups=8, kept=2, topk=17), "topk"), (dict(groups=0), "groups"),
    (dict(groups=7), "groups"), (dict(experts=128, stride=128, groups=128), "groups"), (dict(groups=8, kept=0), "kept_groups"),
    (dict(groups=8, kept=9), "kept_groups"), (dict(scoring=2), "scoring"), (dict(stride=63), "row_stride"), (dict(dtype=3), "dtype"),
    (dict(logits=None), "NULL"), (dict(weights=None), "NULL"), (dict(ids=None), "NULL")])
def test_router_refuses(change, message):
    _lib, lib = layer()
    assert route_call(lib, **change) == _lib.E_INVALID and message in lib.sonar_layer_last_error().decode()


def test_the_rule_of_the_int8_product():
    """Which form takes a call, at the borders of the rule, and that its scratch is what the form needs."""
    import ctypes
    _lib, lib = layer()
    def choice(m, n, k, aligned=1):
        splits = ctypes.c_int(0)
        return lib.sonar_debug_int8_choice(m, n, k, aligned, ctypes.byref(splits)), splits.value
    assert choice(1, 4096, 4096) == (2, 1) and choice(16, 4097, 4096) == (1, 1)
    assert choice(17, 4096, 6144) == (3, 1) and choice(32, 4112, 4096)[0] >= 4 and choice(32, 4112, 4096, 0) == (3, 1)
    assert choice(17, 28672, 100) == (3, 1)           # K is no multiple of 16: unaligned whatever the strides are
    assert choice(33, 100, 15) == (0, 1) and choice(77, 1537, 1003) == (3, 1) and choice(200, 1537, 1003) == (0, 1)
    assert choice(77, 1537, 4095)[0] >= 4 and choice(1 << 24, 1, 17)[0] >= 4
    assert choice(8192, 28672, 4096) == (8, 1) and choice(2048, 4096, 14336) == (7, 1)
    form, splits = choice(64, 256, 14336)
    assert form == 4 and splits > 1
    rows, cols = (64, 64, 128, 256, 256), (64, 128, 128, 128, 256)
    for m, n, k in ((1, 512, 4096), (64, 256, 14336), (200, 1024, 14336), (500, 4096, 4096), (70, 700, 1001), (3000, 3000, 8191)):
        for aligned in (0, 1):
            form, splits = choice(m, n, k, aligned)
            want = 0
            if form >= 4:
                tiles = -(-m // rows[form - 4]) * -(-n // cols[form - 4])
                want = tiles * rows[form - 4] * cols[form - 4] * 4 * splits if splits > 1 else 0
                want += 0 if aligned and k % 16 == 0 else (m + n) * (-(-k // 256) * 256)
            assert lib.sonar_scaled_mm_int8_scratch_bytes(m, n, k, aligned) == want, (m, n, k, aligned)
    assert lib.sonar_scaled_mm_int8_scratch_bytes(0, 8, 8, 1) == 0


def test_calls_without_rows_launch_nothing():
    _lib, lib = layer()
    assert norm_call(lib, rows=0, x=None, q=None) == 0
    assert mm_call(lib, m=0, a=None, a_len=1) == 0 and mm_call(lib, n=0, b_len=1) == 0
    assert route_call(lib, tokens=0, logits=None) == 0


# ---------------------------------------------------------------- ops
def test_schemas():
    import sonar_amd.ops  # noqa: F401
    for name, want in (
            ("rms_norm_per_token_quant", "(Tensor x, Tensor weight, Tensor? residual, float epsilon, ScalarType quant_dtype, "
             "bool with_norm) -> Tensor[]"),
            ("scaled_mm_int8", "(Tensor a, Tensor b, Tensor a_scales, Tensor b_scales, ScalarType out_dtype, Tensor? bias) -> Tensor"),
            ("topk_routing", "(Tensor logits, int topk, str scoring_func, bool renormalize, Tensor? bias, int num_expert_group, "
             "int topk_group, float routed_scaling_factor) -> (Tensor, Tensor)")):
        assert str(getattr(torch.ops.sonar_amd, name).default._schema) == f"sonar_amd::{name}{want}"


def test_fake_results():
    from torch._subclasses.fake_tensor import FakeTensorMode

    from sonar_amd import ops
    with FakeTensorMode():
        x = torch.empty((2, 3, 64), dtype=torch.bfloat16, device="cuda")
        w = torch.empty(64, dtype=torch.bfloat16, device="cuda")
        q, s, z, y = ops.rms_norm_per_token_quant(x, w, 1e-6, torch.float8_e4m3fn, x)
        assert (q.shape, q.dtype, s.shape, s.dtype, z.shape, z.dtype, y) == (
            x.shape, torch.float8_e4m3fn, (2, 3, 1), torch.float32, x.shape, x.dtype, None)
        q, s, z, y = ops.rms_norm_per_token_quant(x, w, 1e-6, with_norm=True)
        assert q.dtype == torch.int8 and z is None and y.shape == x.shape
        b = torch.empty((48, 64), dtype=torch.int8, device="cuda").t()
        c = ops.scaled_mm_int8(q, b, s, s.new_empty(48), torch.float16)
        assert c.shape == (2, 3, 48) and c.dtype == torch.float16
        weights, ids = ops.topk_routing(torch.empty((5, 16), device="cuda"), 3)
        assert weights.shape == ids.shape == (5, 3) and weights.dtype == torch.float32 and ids.dtype == torch.int32


def test_ops_do_not_run_on_cpu_tensors():
    from sonar_amd import ops
    with pytest.raises(NotImplementedError):
        ops.scaled_mm_int8(torch.zeros((2, 16), dtype=torch.int8), torch.zeros((16, 4), dtype=torch.int8), torch.ones(2), torch.ones(4),
                           torch.float16)


# ---------------------------------------------------------------- router, torch expressions against the oracle
def route_inputs(seed, tokens, experts, ties):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((tokens, experts)) * 2
    if ties:
        x = np.round(x)   # many equal logits
    x[:, rng.integers(0, experts)] = -np.inf
    x[0] = -np.inf
    if tokens > 2:
        x[1, experts // 2], x[2, 0] = np.nan, np.finfo(np.float32).min
    return x.astype(np.float32), (rng.standard_normal(experts) * 0.1).astype(np.float32)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("experts,groups,kept,topk", [(8, 1, 1, 2), (1, 1, 1, 1), (60, 4, 2, 6), (64, 64, 5, 5), (33, 3, 3, 33)])
def test_router_expressions_match_the_oracle(scoring, biased, experts, groups, kept, topk):
    from sonar_amd.fused_moe import grouped_topk
    x, bias = route_inputs(experts, 9, experts, ties=True)
    w, ids = grouped_topk(torch.empty(9, 4), torch.from_numpy(x), topk, True, groups, kept, scoring, 2.5,
                          torch.from_numpy(bias) if biased else None)
    want_w, want_ids = lo.topk_routing(x, topk, scoring, True, bias if biased else None, groups, kept, 2.5)
    assert np.array_equal(ids.numpy(), want_ids)
    np.testing.assert_allclose(w.numpy(), want_w, rtol=2 ** -22, atol=0)


def test_router_host_refusals():
    from sonar_amd.fused_moe import fused_topk, grouped_topk
    h, x = torch.empty(3, 4), torch.zeros(3, 8)
    with pytest.raises(AssertionError, match="tokens"):
        fused_topk(torch.empty(2, 4), x, 2, True)
    with pytest.raises(ValueError, match="scoring"):
        fused_topk(h, x, 2, True, "tanh")
    with pytest.raises(ValueError, match="topk"):
        fused_topk(h, x, 9, True)
    with pytest.raises(ValueError, match="groups"):
        grouped_topk(h, x, 2, True, 3, 1)
    with pytest.raises(ValueError, match="topk"):
        grouped_topk(h, x, 5, True, 4, 2)


# ---------------------------------------------------------------- the oracle
def test_oracle_values():
    # softmax of (ln 1, ln 2, ln 4, ln 1): 1/8, 1/4, 1/2, 1/8; the bias lifts expert 3, whose weight stays its score
    x = np.log([[1.0, 2.0, 4.0, 1.0]])
    w, ids = lo.topk_routing(x, 2)
    assert ids.tolist() == [[2, 1]] and np.allclose(w, [[0.5, 0.25]])
    w, ids = lo.topk_routing(x, 2, bias=[0, 0, 0, 0.5], renormalize=True, factor=2.0)
    assert ids.tolist() == [[3, 2]] and np.allclose(w, [[0.4, 1.6]])
    w, ids = lo.topk_routing(x, 2, groups=2, kept_groups=1)   # best group: experts 2 and 3
    assert ids.tolist() == [[2, 3]]
    w, ids = lo.topk_routing([[-math.inf] * 4], 2, renormalize=True)
    assert ids.tolist() == [[0, 1]] and w.tolist() == [[0, 0]]
    z, y = lo.rms_norm(np.array([[3.0, 4.0]]), np.array([1.0, 2.0]), 0.0)
    assert np.allclose(y, [[3 / np.sqrt(12.5), 8 / np.sqrt(12.5)]])
    assert lo.round_to(np.array([1 + 2 ** -8, 1 + 3 * 2 ** -8, 1 + 2 ** -8 + 2 ** -30]), "bf16").tolist() == [
        1.0, 1 + 2 ** -6, 1 + 2 ** -7]
    for dtype, tdt in (("bf16", torch.bfloat16), ("fp16", torch.float16)):
        v = torch.randn(1000, dtype=torch.float64) * 10 ** torch.linspace(-9, 4, 1000, dtype=torch.float64)
        v = v.float()
        assert np.array_equal(lo.round_to(v.double().numpy(), dtype), v.to(tdt).double().numpy())
    c = lo.scaled_mm_int8(np.array([[1, -2]], dtype=np.int8), np.array([[3, 4], [-128, 127]], dtype=np.int8), [0.5], [1.0, 2.0],
                          np.array([1.0, 0.0]))
    assert c.tolist() == [[-1.5, -382.0]]


KERNEL_FORMS = {"rms_norm_quant_kernel": 36, "rms_norm_quant_any_kernel": 6, "int8_general_kernel": 2, "topk_routing_kernel": 16, "int8_stream_kernel": 12,
                "int8_tile_kernel": 10, "int8_join_kernel": 10, "int8_pad_kernel": 1}


def test_library_holds_the_kernel_forms_the_gpu_tests_launch():
    """Every instantiation in the library has a case in the GPU tests: a new form gets one before its number is raised."""
    nm = shutil.which("nm") or shutil.which("llvm-nm")
    if nm is None:
        pytest.skip("nm not available")
    _lib, _ = layer()
    syms = subprocess.run([nm, _lib._LAYER_PATH], capture_output=True, text=True, timeout=120).stdout
    seen = collections.Counter(m.group(1) for m in re.finditer(r"__device_stub__([a-z_0-9]+)", syms))
    assert dict(seen) == KERNEL_FORMS
