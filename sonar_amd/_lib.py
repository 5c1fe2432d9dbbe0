"""ctypes binding of the C ABIs in include/sonar_marlin.h, include/sonar_layer.h and
include/sonar_attention.h.

Loading fails loudly when the HIP library has not been built: there is no
fallback path."""
from __future__ import annotations

import ctypes
import os
from ctypes import POINTER, c_char_p, c_double, c_float, c_int, c_int64, c_size_t, c_void_p

_LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", "libsonar_marlin.so")
_LAYER_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", "libsonar_layer.so")
_ATTENTION_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", "libsonar_attention.so")

DTYPE_F16 = 0
DTYPE_BF16 = 1
DTYPE_F32 = 2
LAYOUT_GFX950 = 0
ADTYPE_INT8 = 0
ADTYPE_FP8 = 1
TYPE_UINT4B8 = 1125899907892224
TYPE_UINT4 = 1125899906843648
TYPE_UINT8B128 = 1125899923621888
TYPE_FLOAT8_E4M3FN = 2814749767172868
TYPE_FLOAT4_E2M1F = 562949953487106

OK = 0
E_INVALID = -1
E_UNSUPPORTED = -2
E_RUNTIME = -3

GROUPED_GENERAL, GROUPED_DECODE, GROUPED_MID, GROUPED_TILE = 1, 2, 3, 4   # what sonar_marlin_last_grouped_kernel answers

# name -> (restype, argtypes); must list every symbol include/sonar_marlin.h declares
PROTOTYPES = {
    "sonar_marlin_last_error": (c_char_p, []),
    "sonar_marlin_version": (c_char_p, []),
    "sonar_marlin_last_decode_launch": (c_int, [c_void_p, c_int]),
    "sonar_marlin_last_grouped_kernel": (c_int, []),
    "sonar_marlin_last_mid_strips": (c_int, []),
    "sonar_debug_tile_schedule": (c_int64, [c_int64, c_int64, c_int64, c_int64, c_void_p, c_int64]),
    "sonar_debug_moe_tile_schedule": (c_int64, [c_int64, c_int64, c_int64, c_int64, c_int, c_void_p, c_int64]),
    "sonar_debug_moe_pair_schedule": (c_int64, [c_int64, c_int64, c_int64, c_int64, c_int64, c_int, c_void_p, c_void_p, c_int64]),
    "sonar_debug_twin_schedule": (c_int64, [c_int64] * 4 + [c_int, c_int, c_void_p, c_int64]),
    "sonar_debug_moe_twin": (c_int, [c_int64] * 6 + [c_int] * 3),
    "sonar_debug_tile_estimate": (c_double, [c_int64] * 3),
    "sonar_debug_mid_beats_tiles": (c_int, [c_int64] * 4 + [c_int, c_int64]),
    "sonar_gptq_marlin_repack": (c_int, [c_void_p, c_void_p, c_void_p, c_int64, c_int64, c_int, c_void_p]),
    "sonar_awq_marlin_repack": (c_int, [c_void_p, c_void_p, c_int64, c_int64, c_int, c_void_p]),
    "sonar_gptq_marlin_moe_repack": (c_int, [c_void_p, c_void_p, c_void_p, c_int64, c_int64, c_int64, c_void_p]),
    "sonar_awq_marlin_moe_repack": (c_int, [c_void_p, c_void_p, c_int64, c_int64, c_int64, c_void_p]),
    "sonar_marlin_permute_scales": (c_int, [c_void_p, c_void_p, c_int64, c_int, c_void_p]),
    "sonar_load_gptq_linear": (c_int, [c_void_p] * 7 + [c_int64] * 4 + [c_int, c_int, c_void_p]),
    "sonar_sort_g_idx": (c_int, [c_void_p] * 3 + [c_int64, c_void_p]),
    "sonar_load_gptq_act_order": (c_int, [c_void_p] * 8 + [c_int64] * 4 + [c_int, c_void_p]),
    "sonar_awq_to_standard": (c_int, [c_void_p] * 4 + [c_int64] * 3 + [c_void_p]),
    "sonar_marlin_pack_zero_points": (c_int, [c_void_p, c_void_p, c_int64, c_int64, c_int64, c_int64, c_int, c_int,
                                              c_void_p]),
    "sonar_awq_to_gptq": (c_int, [c_void_p, c_void_p, c_int64, c_int64, c_void_p]),
    "sonar_awq_zeros_to_plain": (c_int, [c_void_p, c_void_p, c_int64, c_int64, c_void_p]),
    "sonar_marlin_to_gfx950": (c_int, [c_void_p, c_void_p, c_int64, c_int64, c_void_p]),
    "sonar_gfx950_to_marlin": (c_int, [c_void_p, c_void_p, c_int64, c_int64, c_void_p]),
    "sonar_marlin8_to_gfx950": (c_int, [c_void_p, c_void_p, c_int64, c_int64, c_void_p]),
    "sonar_gfx950_to_marlin8": (c_int, [c_void_p, c_void_p, c_int64, c_int64, c_void_p]),
    "sonar_gptq_marlin_repack_a8": (c_int, [c_void_p, c_void_p, c_int64, c_int64, c_int, c_void_p]),
    "sonar_awq_marlin_repack_a8": (c_int, [c_void_p, c_void_p, c_int64, c_int64, c_int, c_void_p]),
    "sonar_marlin_a8_to_gfx950": (c_int, [c_void_p, c_void_p, c_int64, c_int64, c_void_p]),
    "sonar_gfx950_to_marlin_a8": (c_int, [c_void_p, c_void_p, c_int64, c_int64, c_void_p]),
    "sonar_marlin_int4_fp8_preprocess": (c_int, [c_void_p, c_void_p, c_void_p, c_int64, c_int64, c_int64, c_void_p]),
    "sonar_per_token_quant_int8": (c_int, [c_void_p, c_int, c_int64, c_void_p, c_void_p, c_int64, c_int64, c_void_p]),
    "sonar_per_token_quant_int8_scaled": (c_int, [c_void_p, c_int, c_int64, c_void_p, c_void_p, c_void_p, c_int64, c_int64,
                                                   c_void_p]),
    "sonar_per_token_quant_fp8": (c_int, [c_void_p, c_int, c_int64, c_void_p, c_void_p, c_int64, c_int64, c_void_p]),
    "sonar_marlin_gemm_a8_scratch_bytes": (c_size_t, [c_int64, c_int64, c_int64, c_int64]),
    "sonar_marlin_gemm_a8": (c_int, [c_void_p, c_int64, c_int, c_void_p, c_void_p, c_int, c_void_p, c_void_p,
                                     c_void_p, c_void_p, c_void_p, c_size_t, c_int, c_int64, c_int64, c_int64,
                                     c_int64, c_int64, c_void_p]),
    "sonar_moe_wna16_marlin_gemm_a8": (c_int, [
        c_void_p, c_int, c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int64,
        c_void_p, c_void_p, c_void_p, c_int64, c_int64, c_int, c_int64, c_int, c_int64, c_int64, c_int64, c_int64,
        c_int64, c_void_p]),
    "sonar_marlin_dequant": (c_int, [c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_void_p, c_int,
                                     c_int64, c_int64, c_int64, c_int64, c_int, c_void_p]),
    "sonar_marlin_gemm_scratch_bytes": (c_size_t, [c_int64, c_int64, c_int64]),
    "sonar_marlin_gemm": (c_int, [c_void_p, c_int64, c_void_p, c_void_p, c_int, c_void_p, c_void_p,
                                  c_void_p, c_void_p, c_void_p, c_void_p, c_int64, c_void_p, c_size_t,
                                  c_int, c_int64, c_int64, c_int64, c_int64, c_int64, c_int, c_int,
                                  c_int, c_void_p]),
    "sonar_marlin_gemm_nvfp4": (c_int, [c_void_p, c_int64, c_void_p, c_void_p, c_int, c_void_p, c_void_p,
                                        c_void_p, c_void_p, c_int64, c_void_p, c_size_t,
                                        c_int, c_int64, c_int64, c_int64, c_int64, c_void_p]),
    "sonar_marlin_gemm_noalloc": (c_int, [c_void_p, c_int64, c_void_p, c_void_p, c_int, c_void_p, c_void_p,
                                          c_void_p, c_void_p, c_void_p, c_void_p, c_int64,
                                          c_int, c_int64, c_int64, c_int64, c_int64, c_int64, c_int, c_int,
                                          c_int, c_void_p]),
    "sonar_moe_marlin_gemm_scratch_bytes": (c_size_t, [c_int64, c_int64, c_int64, c_int64]),
    "sonar_moe_wna16_marlin_gemm": (c_int, [
        c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
        c_void_p, c_int64, c_void_p, c_size_t, c_void_p, c_int64, c_void_p, c_void_p, c_void_p,
        c_int64, c_int64, c_int, c_int64, c_int, c_int64, c_int64, c_int64, c_int64, c_int64,
        c_int, c_int, c_int, c_void_p]),
    "sonar_moe_wna16_marlin_gemm_nvfp4": (c_int, [
        c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_void_p, c_size_t, c_void_p, c_int64,
        c_void_p, c_void_p, c_void_p, c_int64, c_int64, c_int, c_int64, c_int, c_int64, c_int64, c_int64, c_int64,
        c_void_p]),
    "sonar_moe_wna16_marlin_gemm_gated": (c_int, [
        c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
        c_size_t, c_void_p, c_int64, c_void_p, c_void_p, c_void_p, c_int64, c_int64, c_int, c_int64, c_int, c_int64,
        c_int64, c_int64, c_int64, c_int64, c_int, c_void_p, c_int, c_float, c_float, c_void_p, c_void_p, c_void_p,
        c_void_p]),
    "sonar_moe_routed_gemm_applies": (c_int, [c_int64] * 7),
    "sonar_moe_routed_gemm": (c_int, [
        c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int64, c_int64, c_int, c_int64, c_int,
        c_int64, c_int64, c_int64, c_int64, c_int64, c_void_p, c_int, c_float, c_float, c_void_p, c_void_p]),
    "sonar_moe_align_block_size": (c_int, [c_void_p, c_int64, c_int64, c_int64, c_void_p, c_int64, c_void_p,
                                           c_int64, c_void_p, c_void_p, c_void_p, c_void_p]),
    "sonar_silu_and_mul": (c_int, [c_void_p, c_void_p, c_int64, c_int64, c_int, c_void_p]),
    "sonar_moe_activation": (c_int, [c_void_p, c_void_p, c_int64, c_int64, c_int, c_float, c_float, c_float, c_int,
                                     c_void_p]),
    "sonar_moe_sum": (c_int, [c_void_p, c_void_p, c_int64, c_int64, c_int64, c_int, c_void_p]),
}

# the same for include/sonar_layer.h
LAYER_PROTOTYPES = {
    "sonar_layer_last_error": (c_char_p, []),
    "sonar_rms_norm_per_token_quant": (c_int, [c_void_p, c_int64, c_void_p, c_int64, c_void_p, c_void_p, c_void_p, c_void_p,
                                               c_int, c_void_p, c_int, c_int64, c_int64, c_double, c_void_p]),
    "sonar_scaled_mm_int8_scratch_bytes": (c_size_t, [c_int64] * 3 + [c_int]),
    "sonar_debug_int8_choice": (c_int, [c_int64] * 3 + [c_int, c_void_p]),
    "sonar_debug_int8_form": (c_int, [c_int, c_int]),
    "sonar_scaled_mm_int8": (c_int, [c_void_p, c_int64, c_void_p, c_int64, c_void_p, c_void_p, c_int64, c_void_p, c_int64,
                                     c_void_p, c_void_p, c_size_t, c_int, c_int64, c_int64, c_int64, c_void_p]),
    "sonar_topk_routing": (c_int, [c_void_p, c_int, c_int64, c_void_p, c_void_p, c_void_p, c_int64, c_int64, c_int64, c_int,
                                   c_int, c_int64, c_int64, c_double, c_void_p]),
}
SCORING_SOFTMAX, SCORING_SIGMOID = 0, 1
CACHE_FP8 = 3


class KvCache(ctypes.Structure):
    """sonar_kv_cache"""
    _fields_ = [("data", c_void_p), ("page_stride", c_int64), ("slot_stride", c_int64), ("head_stride", c_int64),
                ("scale", c_void_p), ("scale_len", c_int64)]


# the same for include/sonar_attention.h
ATTENTION_PROTOTYPES = {
    "sonar_attention_last_error": (c_char_p, []),
    "sonar_qk_norm_rope": (c_int, [c_void_p, c_int64, c_int64] * 3 + [c_void_p, c_int, c_void_p, c_int64, c_int64, c_int, c_void_p,
                                   c_void_p, c_double, c_void_p, c_void_p, POINTER(KvCache), POINTER(KvCache), c_int, c_void_p, c_int,
                                   c_int64, c_int64, c_int, c_int64, c_int64, c_int64, c_int64, c_void_p]),
    "sonar_paged_attention_scratch_bytes": (c_size_t, [c_int64] * 5 + [c_int] + [c_int64] * 2),
    "sonar_paged_attention": (c_int, [c_void_p, c_int64, c_int64, POINTER(KvCache), POINTER(KvCache), c_int, c_int64, c_int64, c_void_p,
                                      c_int64, c_int64, c_void_p, c_void_p, c_void_p, c_int64, c_int64, c_int, c_double, c_double,
                                      c_int64, c_int, c_void_p, c_void_p, c_int64, c_void_p, c_size_t, c_int, c_int64, c_int64, c_int64,
                                      c_int64, c_int64, c_int64, c_void_p]),
}

_lib = None
_layer = None
_attention = None


class SonarMarlinError(RuntimeError):
    def __init__(self, code: int, message: str):
        super().__init__(message)
        self.code = code


def lib_path() -> str:
    return _LIB_PATH


def layer_path() -> str:
    return _LAYER_PATH


def attention_path() -> str:
    return _ATTENTION_PATH


def _open(path: str, prototypes) -> ctypes.CDLL:
    if not os.path.exists(path):
        raise ImportError(
            f"{path} is missing: build it with `python -m sonar_amd.build` "
            "(hipcc --offload-arch=gfx950); there is no fallback implementation")
    lib = ctypes.CDLL(path)
    for name, (restype, argtypes) in prototypes.items():
        fn = getattr(lib, name)  # AttributeError if the library does not export it
        fn.restype = restype
        fn.argtypes = argtypes
    return lib


def load() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        _lib = _open(_LIB_PATH, PROTOTYPES)
    return _lib


def load_layer() -> ctypes.CDLL:
    global _layer
    if _layer is None:
        _layer = _open(_LAYER_PATH, LAYER_PROTOTYPES)
    return _layer


def load_attention() -> ctypes.CDLL:
    global _attention
    if _attention is None:
        _attention = _open(_ATTENTION_PATH, ATTENTION_PROTOTYPES)
    return _attention


def _raise(rc: int, msg: bytes) -> None:
    text = msg.decode("utf-8", "replace")
    if rc == E_UNSUPPORTED:
        raise NotImplementedError(text)
    raise SonarMarlinError(rc, text)


def check(rc: int) -> None:
    if rc != OK:
        _raise(rc, load().sonar_marlin_last_error())


def check_layer(rc: int) -> None:
    if rc != OK:
        _raise(rc, load_layer().sonar_layer_last_error())


def check_attention(rc: int) -> None:
    if rc != OK:
        _raise(rc, load_attention().sonar_attention_last_error())
