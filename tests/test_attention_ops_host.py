"""CPU: the operators between the qkv and the output projection without a GPU - the C ABI's list and its refusals (they come before
anything is launched), the ops' schemas and fake results, the tables of the rotation, and the oracle's own values."""
import ctypes
import math
import os
import re
import shutil
import subprocess
import sys

import numpy as np
import pytest
import torch

from oracle import attention_oracle as ao

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAKE = 1 << 20   # a device address that no refused call looks at


def library():
    from sonar_amd import _lib
    return _lib, _lib.load_attention()


def test_header_prototypes_and_exports_agree():
    _lib, lib = library()
    header = open(os.path.join(ROOT, "include", "sonar_attention.h")).read()
    declared = re.findall(r"^(?:int|size_t|const char\*)\s+(sonar_\w+)\((.*?)\);", header, re.M | re.S)
    assert {name for name, _ in declared} == set(_lib.ATTENTION_PROTOTYPES)
    for name, arguments in declared:
        count = 0 if arguments.strip() == "void" else arguments.count(",") + 1
        assert getattr(lib, name) and count == len(_lib.ATTENTION_PROTOTYPES[name][1]), name
    assert int(re.search(r"SONAR_CACHE_FP8 (\d)", header).group(1)) == _lib.CACHE_FP8


# ---------------------------------------------------------------- refusals
def cache(_lib, scale=None, scale_len=0, data=FAKE, page=2048, slot=128, head=64):
    return _lib.KvCache(data, page, slot, head, scale, scale_len)


def rope_call(lib, _lib, **change):
    a = dict(q=FAKE, q_token=512, q_head=64, k=FAKE, k_token=512, k_head=64, v=FAKE, v_token=512, v_head=64, positions=FAKE,
             positions_64=1, cos_sin=FAKE, max_position=100, rotary_dim=64, half=1, q_weight=FAKE, k_weight=FAKE, epsilon=1e-6,
             q_out=FAKE, k_out=None, keys=cache(_lib), values=cache(_lib), cache_dtype=1, slots=FAKE, slots_64=1, pages=10, page_size=16,
             dtype=1, tokens=4, heads=4, kv_heads=2, head_dim=64)
    a.update(change)
    return lib.sonar_qk_norm_rope(*(ctypes.byref(v) if isinstance(v, _lib.KvCache) else v for v in a.values()), None)


@pytest.mark.parametrize("change,message", [
    (dict(dtype=3), "dtype"), (dict(heads=0), "heads"), (dict(kv_heads=0), "kv_heads"), (dict(head_dim=0), "head_dim"),
    (dict(head_dim=1025), "head_dim"), (dict(tokens=-1), "tokens"), (dict(tokens=1 << 31), "tokens"), (dict(tokens=1 << 28), "too many"),
    (dict(positions=None), "together"), (dict(cos_sin=None), "together"), (dict(rotary_dim=63), "rotary_dim"),
    (dict(rotary_dim=66), "rotary_dim"), (dict(rotary_dim=0), "rotary_dim"), (dict(epsilon=0.0), "epsilon"),
    (dict(epsilon=float("nan")), "epsilon"), (dict(values=None), "together"), (dict(cache_dtype=0), "cache_dtype"),
    (dict(dtype=2, cache_dtype=3), "cache_dtype"), (dict(cache_dtype=3), "scales"), (dict(page_size=0), "slots"), (dict(pages=-1), "pages"),
    (dict(pages=1 << 40), "pages"), (dict(q=None), "NULL"), (dict(k=None), "NULL"), (dict(q_out=None), "NULL"), (dict(v=None), "v and slots"),
    (dict(slots=None), "v and slots"), (dict(keys=None, values=None), "k_out")])
def test_rotation_refuses(change, message):
    _lib, lib = library()
    rc = rope_call(lib, _lib, **change)
    assert rc == _lib.E_INVALID and message in lib.sonar_attention_last_error().decode()
    with pytest.raises(_lib.SonarMarlinError, match=message):
        _lib.check_attention(rc)


def attention_call(lib, _lib, **change):
    a = dict(q=FAKE, q_token=512, q_head=64, keys=cache(_lib), values=cache(_lib), cache_dtype=1, pages=10, page_size=16, table=FAKE,
             table_stride=5, table_pages=5, lens=FAKE, starts=FAKE, out=FAKE, out_token=512, out_head=64, clear=1, scale=0.125, cap=0.0,
             window=0, causal=1, slopes=None, tree=None, tree_words=0, scratch=None, scratch_bytes=0, dtype=1, tokens=4, seqs=2, heads=4,
             kv_heads=2, head_dim=64, max_seq_len=80)
    a.update(change)
    return lib.sonar_paged_attention(*(ctypes.byref(v) if isinstance(v, _lib.KvCache) else v for v in a.values()), None)


@pytest.mark.parametrize("change,message", [
    (dict(dtype=2), "dtype"), (dict(cache_dtype=0), "cache_dtype"), (dict(cache_dtype=3), "scales"), (dict(kv_heads=3), "multiple"),
    (dict(heads=0), "heads"), (dict(head_dim=8), "head_dim"), (dict(head_dim=72), "head_dim"), (dict(head_dim=272), "head_dim"),
    (dict(tokens=-1), "tokens"), (dict(tokens=1 << 30), "too many"), (dict(seqs=-1), "seqs"), (dict(seqs=0), "seqs"),
    (dict(max_seq_len=-1), "max_seq_len"), (dict(max_seq_len=1 << 31), "max_seq_len"), (dict(window=-1), "window"),
    (dict(window=4, causal=0), "window"), (dict(page_size=0), "slots"), (dict(table_pages=1 << 30, page_size=4), "slots"),
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(cap=-1.0), "cap"),
    (dict(cap=float("inf")), "cap"), (dict(tree=FAKE, tree_words=0), "tree_words"), (dict(tree=FAKE, tree_words=1, window=3), "tree"),
    (dict(tree=FAKE, tree_words=1, slopes=FAKE), "tree"), (dict(q=FAKE + 8), "q must"), (dict(q_token=516), "q must"),
    (dict(out=FAKE + 4), "out must"), (dict(out_head=66), "out must"), (dict(q=None), "NULL"), (dict(out=None), "NULL"),
    (dict(starts=None), "NULL"), (dict(lens=None), "seq_lens"), (dict(table=None), "block_table"), (dict(table_stride=4), "block_table"),
    (dict(pages=0), "pages"), (dict(scratch=FAKE + 8), "scratch"), (dict(seqs=1 << 29), "workgroups"), (dict(keys=None), "NULL")])
def test_attention_refuses(change, message):
    _lib, lib = library()
    assert attention_call(lib, _lib, **change) == _lib.E_INVALID and message in lib.sonar_attention_last_error().decode()


def test_caches_are_refused():
    _lib, lib = library()
    for bad in (cache(_lib, page=2052), cache(_lib, slot=132), cache(_lib, head=68), cache(_lib, data=FAKE + 8), cache(_lib, slot=1 << 36),
                cache(_lib, page=1 << 36), cache(_lib, page=1 << 32), cache(_lib, slot=-128), cache(_lib, page=-2048)):
        for name in ("keys", "values"):
            assert attention_call(lib, _lib, **{name: bad}) == _lib.E_INVALID
    for bad in (cache(_lib), cache(_lib, FAKE, 3), cache(_lib, FAKE, 0), cache(_lib, FAKE, 1, slot=136)):
        good = cache(_lib, FAKE, 2)
        assert attention_call(lib, _lib, cache_dtype=3, keys=good, values=bad) == _lib.E_INVALID
    assert rope_call(lib, _lib, cache_dtype=3, keys=cache(_lib, FAKE, 1), values=cache(_lib, FAKE, 3)) == _lib.E_INVALID


def test_calls_without_tokens_launch_nothing():
    _lib, lib = library()
    assert rope_call(lib, _lib, tokens=0, q=None, k=None, positions=None) == 0
    assert attention_call(lib, _lib, tokens=0, q=None, seqs=0, lens=None) == 0
    assert lib.sonar_paged_attention_scratch_bytes(0, 4, 8, 8, 64, 1, 10000, 0) == 0


# ---------------------------------------------------------------- ops
def test_schemas():
    import sonar_amd.ops  # noqa: F401
    for name, want in (
            ("qk_norm_rope", "(Tensor query, Tensor key, Tensor? positions, Tensor? cos_sin_cache, Tensor? q_weight, Tensor? k_weight, "
             "float epsilon, bool is_neox) -> (Tensor, Tensor)"),
            ("qk_norm_rope_append", "(Tensor query, Tensor key, Tensor value, Tensor(a!) key_cache, Tensor(b!) value_cache, "
             "Tensor slot_mapping, Tensor? positions, Tensor? cos_sin_cache, Tensor? q_weight, Tensor? k_weight, float epsilon, "
             "bool is_neox, Tensor? k_scale, Tensor? v_scale) -> Tensor"),
            ("paged_attention_out", "(Tensor query, Tensor key_cache, Tensor value_cache, Tensor block_table, Tensor seq_lens, "
             "Tensor query_start_loc, float scale, bool causal, int window, float softcap, Tensor? alibi_slopes, Tensor? tree_mask, "
             "Tensor? k_scale, Tensor? v_scale, int? max_seq_len, Tensor(a!) out) -> ()")):
        assert str(getattr(torch.ops.sonar_amd, name).default._schema) == f"sonar_amd::{name}{want}"


def test_fake_results():
    from torch._subclasses.fake_tensor import FakeTensorMode

    from sonar_amd import ops
    with FakeTensorMode():
        q = torch.empty((5, 8, 64), dtype=torch.bfloat16, device="cuda")
        kv = torch.empty((5, 2, 64), dtype=torch.bfloat16, device="cuda")
        at = torch.empty(5, dtype=torch.int64, device="cuda")
        table = torch.empty((99, 64), device="cuda")
        a, b = ops.qk_norm_rope(q, kv, at, table)
        assert a.shape == q.shape and b.shape == kv.shape and a.dtype == b.dtype == q.dtype
        keys = torch.empty((9, 16, 2, 64), dtype=torch.bfloat16, device="cuda")
        assert ops.qk_norm_rope_append(q, kv, kv, keys, keys, at, at, table).shape == q.shape
        lens, starts, pages = (torch.empty(n, dtype=torch.int32, device="cuda") for n in (3, 4, (3, 7)))
        out = ops.paged_attention(q, keys, keys, pages, lens, starts)
        assert out.shape == q.shape and out.dtype == q.dtype
        assert ops.paged_attention(q, keys, keys, pages, lens, starts, out=out) is out


def test_ops_do_not_run_on_cpu_tensors():
    from sonar_amd import ops
    x = torch.zeros((2, 2, 64), dtype=torch.float16)
    with pytest.raises(NotImplementedError):
        ops.qk_norm_rope(x, x)


CALLS = """
import sys
import torch
from sonar_amd import ops
missing = sys.argv[1:]
assert ops.__file__.startswith(sys.path[0])
x = torch.zeros((2, 2, 16))
i = torch.zeros(2, dtype=torch.int32)
torch.ops._C.marlin_gemm, ops.marlin_gemm, torch.ops.sonar_amd.topk_routing.default
for call in (lambda: ops.qk_norm_rope(x, x), lambda: ops.qk_norm_rope_append(x, x, x, x[None], x[None], i),
             lambda: ops.paged_attention(x, x[None], x[None], i[None], i, i), lambda: ops.paged_attention(x, x[None], x[None], i[None], i, i, out=x)):
    try:
        call()
    except ImportError as e:
        assert missing and all(name in str(e) for name in missing) and "sonar_amd.build" in str(e), e
    except NotImplementedError:   # (the ops are there, and take GPU tensors)
        assert not missing
    else:
        raise AssertionError("no error")
print("done")
"""
ATTENTION = ("libsonar_attention.so", "libsonar_attention_torch.so")


@pytest.mark.parametrize("missing", [(), ATTENTION, ATTENTION[:1], ATTENTION[1:]], ids=lambda names: "+".join(names) or "none")
def test_the_rest_without_the_attention_libraries(missing, tmp_path):
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


# ---------------------------------------------------------------- tables of the rotation
def test_rotary_tables():
    from sonar_amd.rotary import rotary_cos_sin, rotary_rates
    t = rotary_cos_sin(8, 100000)
    assert t.dtype == torch.float32 and t.shape == (100000, 8)
    for at, i in ((0, 0), (1, 1), (99999, 0), (77777, 3)):   # far positions: angles in 64 bits
        angle = at * 10000.0 ** (-2 * i / 8)
        assert abs(t[at, i] - math.cos(angle)) <= 2 ** -24 and abs(t[at, 4 + i] - math.sin(angle)) <= 2 ** -24
    plain = rotary_rates(128, 500000.0)
    assert torch.allclose(rotary_rates(128, 500000.0, {"rope_type": "linear", "factor": 4.0}) * 4, plain, rtol=1e-15)
    llama3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 8192}
    got, length = rotary_rates(128, 500000.0, llama3), 2 * math.pi / plain
    assert torch.equal(got[length < 2048], plain[length < 2048]) and torch.allclose(got[length > 8192] * 8, plain[length > 8192], rtol=1e-15)
    between = (length > 2048) & (length < 8192)
    part = (8192 / length[between] - 1) / 3
    assert between.any() and torch.allclose(got[between], (1 - part) * plain[between] / 8 + part * plain[between], rtol=1e-14)
    yarn = {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 4096}
    got, plain = rotary_rates(64, 10000.0, yarn), rotary_rates(64, 10000.0)
    turns = 4096 * plain / (2 * math.pi)
    assert torch.equal(got[turns > 40], plain[turns > 40]) and torch.allclose(got[turns < 0.7] * 16, plain[turns < 0.7], rtol=1e-15)
    assert (got <= plain * (1 + 1e-15)).all() and (got[1:] < got[:-1]).all()
    assert torch.allclose(rotary_cos_sin(64, 1, scaling=yarn)[0, :32], torch.tensor(0.1 * math.log(16) + 1).expand(32))
    assert float(rotary_cos_sin(64, 1, scaling={**yarn, "attention_factor": 0.5})[0, 0]) == 0.5
    for bad in (lambda: rotary_rates(7), lambda: rotary_rates(0), lambda: rotary_rates(8, scaling={"rope_type": "other", "factor": 2.0, "original_max_position_embeddings": 1})):
        with pytest.raises(ValueError):
            bad()


# ---------------------------------------------------------------- the oracle
def test_oracle_values():
    table = np.array([[1.0, 0.0], [0.0, 1.0]])   # no turn; a quarter of one
    x = np.array([[[1.0, 2.0, 3.0]], [[1.0, 2.0, 3.0]]])
    got = ao.qk_norm_rope(x, np.array([0, 1]), table)
    assert got.tolist() == [[[1, 2, 3]], [[-2, 1, 3]]]
    wide = np.array([[0.0, 1.0, 1.0, 0.0]])   # pair 0 a quarter turn, pair 1 none
    y = np.array([[[1.0, 2.0, 3.0, 4.0]]])
    assert ao.qk_norm_rope(y, np.array([0]), wide, half=True).tolist() == [[[-3, 2, 1, 4]]]
    assert ao.qk_norm_rope(y, np.array([0]), wide, half=False).tolist() == [[[-2, 1, 3, 4]]]
    assert np.allclose(ao.qk_norm_rope(np.array([[[3.0, 4.0]]]), weight=[1.0, 2.0], epsilon=0.0), [[[3 / np.sqrt(12.5), 8 / np.sqrt(12.5)]]])
    assert np.isnan(ao.qk_norm_rope(x, np.array([0, 2]), table)[1, 0, :2]).all()
    c = ao.append(np.zeros((2, 2, 1, 1)), np.array([[[5.0]], [[6.0]], [[7.0]]]), [3, -1, 4])
    assert c.ravel().tolist() == [0, 0, 0, 5]
    # two keys in pages of one, scores ln 1 and ln 3: weights 1/4 and 3/4
    k = np.log(np.array([1.0, 3.0])).reshape(2, 1, 1, 1)[[1, 0]]
    v = np.array([4.0, 8.0]).reshape(2, 1, 1, 1)[[1, 0]]
    call = lambda **more: ao.paged_attention(np.ones((2, 1, 1)), k, v, np.array([[1, 0]]), [2], [0, 2], 1.0, **more)[0].ravel()  # noqa: E731
    assert np.allclose(call(), [4, 7]) and np.allclose(call(causal=False), [7, 7]) and np.allclose(call(window=1), [4, 8])
    assert np.allclose(call(slopes=[np.log(3.0)]), [4, 0.1 * 4 + 0.9 * 8])
    assert np.allclose(call(cap=1.0, causal=False), 8 - 4 / (1 + np.exp(np.tanh(np.log(3.0)))))
    assert np.allclose(call(tree=np.array([[0], [1]])), [0, 4]) and np.allclose(call(tree=np.array([[2], [3]])), [8, 7])
    # a page that no query sees is not looked at
    assert np.allclose(ao.paged_attention(np.ones((1, 1, 1)), k, v, np.array([[99, 0]]), [2], [0, 1], 1.0, window=1)[0], 8)


@pytest.mark.parametrize("change,message", [
    (dict(scale=1e-31), "scale"), (dict(scale=1e31), "scale"), (dict(cap=1e-50), "cap"), (dict(cap=1e-31), "cap"), (dict(cap=1e31), "cap")])
def test_scales_that_float32_does_not_hold_are_refused(change, message):
    _lib, lib = library()
    assert attention_call(lib, _lib, **change) == _lib.E_INVALID and message in lib.sonar_attention_last_error().decode()


@pytest.mark.parametrize("cache_dtype", [1, 3])
@pytest.mark.parametrize("tokens,seqs,heads,kv_heads", [(1, 1, 32, 8), (64, 64, 32, 8), (256, 256, 32, 8), (4096, 4096, 32, 8), (192, 24, 32, 8),
                                                       (1, 1, 128, 1), (8192, 1, 32, 8), (20000, 20000, 64, 8)])
def test_scratch_for_long_tables_is_bounded(tokens, seqs, heads, kv_heads, cache_dtype):
    """Sequences that might be very long do not take memory for it: at most 256 parts, and no call is
    refused for the parts that it might have."""
    _lib, lib = library()
    for longest in (100, 5000, 131072, 2 ** 30):
        size = lib.sonar_paged_attention_scratch_bytes(tokens, seqs, heads, kv_heads, 128, cache_dtype, longest, 0)
        assert size <= 256 * tokens * heads * (128 * 4 + 8) + 16


def test_default_rotary_scaling():
    from sonar_amd import rotary
    assert torch.equal(rotary.rotary_rates(64, 5e5, {"rope_type": "default"}), rotary.rotary_rates(64, 5e5))
