"""Python op wrappers with the names and signatures of the reference's
aphrodite/_custom_ops.py (:1363-1461 repack, :1472-1543 marlin_gemm,
:3046-3141 moe_wna16_marlin_gemm).  Importing this module loads the HIP library
and the torch op registration layer; it raises if either is missing.  The
operators around the GEMMs are two libraries more, those of the attention another
two: without those the module serves the rest, and a call of theirs raises."""
from __future__ import annotations

import os

import torch

from . import _lib
from .scalar_type import ScalarType

_OPS_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", "libsonar_marlin_torch.so")
_LAYER_OPS_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", "libsonar_layer_torch.so")
_ATTENTION_OPS_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", "libsonar_attention_torch.so")


def _load_ops() -> None:
    if hasattr(torch.ops._C, "marlin_gemm") and hasattr(torch.ops._C, "marlin_to_gfx950"):
        return
    _lib.load()  # raises with build instructions when the HIP library is missing
    if not os.path.exists(_OPS_PATH):
        raise ImportError(f"{_OPS_PATH} is missing: build it with `python -m sonar_amd.build`")
    torch.ops.load_library(_OPS_PATH)


def _load_layer_ops() -> list[str]:
    """Loads the operators around the GEMMs; returns the files that this takes and that are missing."""
    if hasattr(torch.ops.sonar_amd, "scaled_mm_int8"):
        return []
    missing = [path for path in (_lib.layer_path(), _LAYER_OPS_PATH) if not os.path.exists(path)]
    if not missing:
        _lib.load_layer()
        torch.ops.load_library(_LAYER_OPS_PATH)
    return missing


def _load_attention_ops() -> list[str]:
    """The same for the operators between the qkv and the output projection."""
    if hasattr(torch.ops.sonar_amd, "paged_attention"):
        return []
    missing = [path for path in (_lib.attention_path(), _ATTENTION_OPS_PATH) if not os.path.exists(path)]
    if not missing:
        _lib.load_attention()
        torch.ops.load_library(_ATTENTION_OPS_PATH)
    return missing


_load_ops()
_LAYER_MISSING = _load_layer_ops()
_ATTENTION_MISSING = _load_attention_ops()


def _register_layer_fakes(reg, quant_fake) -> None:
    @reg("sonar_amd::rms_norm_per_token_quant")
    def _(x, weight, residual, epsilon, quant_dtype, with_norm):
        more = (residual is not None) + bool(with_norm)
        return [*quant_fake(quant_dtype)(x), *(torch.empty(x.shape, dtype=x.dtype, device=x.device) for _ in range(more))]

    @reg("sonar_amd::scaled_mm_int8")
    def _(a, b, a_scales, b_scales, out_dtype, bias):
        return torch.empty(a.shape[:-1] + (b.shape[1],), dtype=out_dtype, device=a.device)

    @reg("sonar_amd::topk_routing")
    def _(logits, topk, scoring_func, renormalize, bias, num_expert_group, topk_group, routed_scaling_factor):
        shape = (logits.shape[0], topk)
        return (torch.empty(shape, dtype=torch.float32, device=logits.device),
                torch.empty(shape, dtype=torch.int32, device=logits.device))


def _register_attention_fakes(reg) -> None:
    @reg("sonar_amd::qk_norm_rope")
    def _(query, key, positions, cos_sin_cache, q_weight, k_weight, epsilon, is_neox):
        return (torch.empty(query.shape, dtype=query.dtype, device=query.device),
                torch.empty(key.shape, dtype=query.dtype, device=query.device))

    @reg("sonar_amd::qk_norm_rope_append")
    def _(query, key, value, key_cache, value_cache, slot_mapping, positions, cos_sin_cache, q_weight, k_weight, epsilon, is_neox,
          k_scale, v_scale):
        return torch.empty(query.shape, dtype=query.dtype, device=query.device)

    @reg("sonar_amd::paged_attention")
    def _(query, key_cache, value_cache, block_table, seq_lens, query_start_loc, scale, causal, window, softcap, alibi_slopes,
          tree_mask, k_scale, v_scale, max_seq_len):
        return torch.empty(query.shape, dtype=query.dtype, device=query.device)

    @reg("sonar_amd::paged_attention_out")
    def _(query, key_cache, value_cache, block_table, seq_lens, query_start_loc, scale, causal, window, softcap, alibi_slopes,
          tree_mask, k_scale, v_scale, max_seq_len, out):
        return None


def _register_fakes() -> None:
    reg = torch.library.register_fake

    @reg("_C::gptq_marlin_repack")
    def _(b_q_weight, perm, size_k, size_n, num_bits, is_a_8bit=False):
        pack_factor = 32 // num_bits
        return torch.empty((size_k // 16, size_n * 16 // pack_factor), dtype=b_q_weight.dtype,
                           device=b_q_weight.device)

    @reg("_C::awq_marlin_repack")
    def _(b_q_weight, size_k, size_n, num_bits, is_a_8bit=False):
        pack_factor = 32 // num_bits
        return torch.empty((size_k // 16, size_n * 16 // pack_factor), dtype=b_q_weight.dtype,
                           device=b_q_weight.device)

    @reg("_C::marlin_int4_fp8_preprocess")
    def _(qweight, qzeros_or_none=None, inplace=False):
        return torch.empty_like(qweight)

    @reg("sonar_amd::marlin_linear")
    def _(input, weight, bias, scales, a_factor, global_scale, zeros, g_idx, perm, workspace, b_type_id, size_n, size_k,
          is_k_full, use_fp32_reduce, act):
        # with quantised activations the result has the type of 16-bit scales
        dtype = scales.dtype if act and scales.element_size() == 2 else input.dtype
        return torch.empty(input.shape[:-1] + (size_n,), dtype=dtype, device=input.device)

    def quant_fake(code_dtype):
        def fake(x):
            return (torch.empty(x.shape, dtype=code_dtype, device=x.device),
                    torch.empty(x.shape[:-1] + (1,), dtype=torch.float32, device=x.device))
        return fake

    reg("sonar_amd::per_token_quant_int8")(quant_fake(torch.int8))
    reg("sonar_amd::per_token_quant_fp8")(quant_fake(torch.float8_e4m3fn))
    if not _LAYER_MISSING:
        _register_layer_fakes(reg, quant_fake)
    if not _ATTENTION_MISSING:
        _register_attention_fakes(reg)

    @reg("sonar_amd::gptq_marlin_moe_repack")
    def _(b_q_weight, perm, size_k, size_n):
        return torch.empty((b_q_weight.shape[0], size_k // 16, size_n * 2), dtype=b_q_weight.dtype,
                           device=b_q_weight.device)

    @reg("sonar_amd::awq_marlin_moe_repack")
    def _(b_q_weight, size_k, size_n):
        return torch.empty((b_q_weight.shape[0], size_k // 16, size_n * 2), dtype=b_q_weight.dtype,
                           device=b_q_weight.device)

    @reg("sonar_amd::permute_scales")
    def _(s, grouped):
        return torch.empty_like(s)

    @reg("sonar_amd::pack_zero_points")
    def _(zp, awq_order, transposed, is_a_8bit):
        return zp.new_empty((zp.shape[1], zp.shape[0])) if transposed else torch.empty_like(zp)

    @reg("sonar_amd::awq_to_standard")
    def _(qweight, qzeros):
        k, words = qweight.shape
        return qweight.new_empty((k // 8, words * 8)), qzeros.new_empty((words, qzeros.shape[0]))

    @reg("sonar_amd::load_gptq_linear")
    def _(qweight, scales, zeros, grouped, transposed):
        k, n = qweight.shape[0] * 8, qweight.shape[1]
        return (qweight.new_empty((k // 16, n * 2)), torch.empty_like(scales),
                qweight.new_empty((0 if zeros is None else scales.shape[0], n // 8)),
                qweight.new_empty((torch.cuda.get_device_properties(qweight.device).multi_processor_count,)))

    @reg("sonar_amd::sort_g_idx")
    def _(g_idx):
        return torch.empty_like(g_idx), torch.empty_like(g_idx)

    @reg("sonar_amd::load_gptq_act_order")
    def _(qweight, scales, g_idx, grouped):
        k, n = qweight.shape[0] * 8, qweight.shape[1]
        return (qweight.new_empty((k // 16, n * 2)), torch.empty_like(scales), torch.empty_like(g_idx), torch.empty_like(g_idx),
                qweight.new_empty((torch.cuda.get_device_properties(qweight.device).multi_processor_count,)))

    @reg("sonar_amd::fused_moe")
    def _(output, hidden, w1, w2, bias1, bias2, scale1, scale2, global_scale1, global_scale2, topk_weights, topk_ids,
          g_idx1, g_idx2, perm1, perm2, zeros1, zeros2, cache13, cache2, b_type_id, num_experts, block_size,
          router_weight_on_input, is_k_full, activation, limit, alpha, beta):
        return None

    @reg("_C::marlin_to_gfx950")
    def _(b_q_weight, size_k, size_n):
        return torch.empty_like(b_q_weight)

    def gemm_fake(a, c, b_q_weight, b_bias, b_scales, a_scales, global_scale, b_zeros, g_idx, perm,
                  workspace, b_q_type_id, size_m, size_n, size_k, is_k_full=True, use_atomic_add=False,
                  use_fp32_reduce=False, is_zp_float=False):
        dtype = a.dtype
        if dtype not in (torch.half, torch.bfloat16):
            dtype = b_scales.dtype
        return torch.empty((size_m, size_n), device=a.device, dtype=dtype)

    reg("_C::marlin_gemm")(gemm_fake)
    reg("_C::gptq_marlin_gemm")(gemm_fake)

    @reg("_moe_C::moe_wna16_marlin_gemm")
    def _(input, output, b_qweight, b_bias, b_scales, a_scales, global_scale, b_qzeros, g_idx, perm,
          workspace, sorted_token_ids, expert_ids, num_tokens_past_padded, topk_weights, moe_block_size,
          top_k, mul_topk_weights, b_q_type, size_m, size_n, size_k, is_k_full, use_atomic_add,
          use_fp32_reduce, is_zp_float, thread_k=-1, thread_n=-1, blocks_per_sm=-1):
        return torch.empty((size_m * top_k, size_n), dtype=input.dtype, device=input.device)


try:
    _register_fakes()
except RuntimeError:
    # already registered by another import of the same ops (e.g. the reference's own wrappers)
    pass


def gptq_marlin_repack(b_q_weight: torch.Tensor, perm: torch.Tensor, size_k: int, size_n: int,
                       num_bits: int, is_a_8bit: bool = False) -> torch.Tensor:
    return torch.ops._C.gptq_marlin_repack(b_q_weight, perm, size_k, size_n, num_bits, is_a_8bit)


def awq_marlin_repack(b_q_weight: torch.Tensor, size_k: int, size_n: int, num_bits: int,
                      is_a_8bit: bool = False) -> torch.Tensor:
    return torch.ops._C.awq_marlin_repack(b_q_weight, size_k, size_n, num_bits, is_a_8bit)


def gptq_marlin_moe_repack(b_q_weight: torch.Tensor, perm: torch.Tensor, size_k: int, size_n: int,
                           num_bits: int, is_a_8bit: bool = False) -> torch.Tensor:
    num_experts = b_q_weight.shape[0]
    assert size_k % 16 == 0
    if num_bits == 4 and not is_a_8bit and b_q_weight.is_contiguous() and perm.is_contiguous():
        return torch.ops.sonar_amd.gptq_marlin_moe_repack(b_q_weight, perm, size_k, size_n)
    output = torch.empty((num_experts, size_k // 16, size_n * (num_bits // 2)),
                         device=b_q_weight.device, dtype=b_q_weight.dtype)
    for e in range(num_experts):
        output[e] = torch.ops._C.gptq_marlin_repack(b_q_weight[e], perm[e], size_k, size_n, num_bits, is_a_8bit)
    return output


def awq_marlin_moe_repack(b_q_weight: torch.Tensor, perm: torch.Tensor, size_k: int, size_n: int,
                          num_bits: int, is_a_8bit: bool = False) -> torch.Tensor:
    num_experts = b_q_weight.shape[0]
    assert size_k % 16 == 0
    if num_bits == 4 and not is_a_8bit and b_q_weight.is_contiguous():
        return torch.ops.sonar_amd.awq_marlin_moe_repack(b_q_weight, size_k, size_n)
    output = torch.empty((num_experts, size_k // 16, size_n * (num_bits // 2)),
                         device=b_q_weight.device, dtype=b_q_weight.dtype)
    for e in range(num_experts):
        output[e] = torch.ops._C.awq_marlin_repack(b_q_weight[e], size_k, size_n, num_bits, is_a_8bit)
    return output


def marlin_int4_fp8_preprocess(qweight: torch.Tensor, qzeros_or_none: torch.Tensor | None = None,
                               inplace: bool = False) -> torch.Tensor:
    """aphrodite/_custom_ops.py:1464-1469: 4-bit codes -> sign and magnitude of code - zero
    point, the form the fp8-activation kernels read."""
    return torch.ops._C.marlin_int4_fp8_preprocess(qweight, qzeros_or_none, inplace)


def per_token_quant_int8(x: torch.Tensor):
    """One scale per row, max(absmax, 1e-10) / 127, and int8 codes rounded half away from zero
    (the reference's Triton kernel, layers/quantization/utils/int8_utils.py:70-120).  Returns
    (int8 of x's shape, float32 (..., 1))."""
    return torch.ops.sonar_amd.per_token_quant_int8(x)


def per_token_quant_fp8(x: torch.Tensor):
    """Dynamic per-token float8_e4m3fn quantisation (QuantFP8(False, GroupShape.PER_TOKEN),
    layers/quantization/input_quant_fp8.py:188-204): scale = max(absmax / 448, 1 / (448 * 512))."""
    return torch.ops.sonar_amd.per_token_quant_fp8(x)


def _layer_op(name: str, missing: list[str] = _LAYER_MISSING):
    """An op of the layer library itself, not the name that looks for an overload at every call."""
    if not missing:
        return getattr(torch.ops.sonar_amd, name).default

    def absent(*args):
        raise ImportError(f"{' and '.join(missing)} missing: build with `python -m sonar_amd.build`; there is no "
                          f"other implementation of {name}")
    return absent


_rms_norm_per_token_quant = _layer_op("rms_norm_per_token_quant")
_scaled_mm_int8 = _layer_op("scaled_mm_int8")
_topk_routing = _layer_op("topk_routing")
_qk_norm_rope = _layer_op("qk_norm_rope", _ATTENTION_MISSING)
_qk_norm_rope_append = _layer_op("qk_norm_rope_append", _ATTENTION_MISSING)
_paged_attention = _layer_op("paged_attention", _ATTENTION_MISSING)
_paged_attention_out = _layer_op("paged_attention_out", _ATTENTION_MISSING)


def rms_norm_per_token_quant(x: torch.Tensor, weight: torch.Tensor, epsilon: float,
                             quant_dtype: torch.dtype = torch.int8, residual: torch.Tensor | None = None,
                             with_norm: bool = False):
    """Root-mean-square norm of the rows of x (float16, bfloat16, float32), with the residual's addition before it and
    8-bit codes with one scale a row behind it, in one launch (the reference's rms_norm_dynamic_per_token_quant):

      z = x + residual, rounded to x's type;  y = z / sqrt(mean(z^2) + epsilon) * weight in float32

    Returns (codes, scales, z, norm): the codes (quant_dtype: int8 or float8_e4m3fn, of x's shape) and float32 scales
    (..., 1) of y as per_token_quant_int8 / _fp8 make them, what `marlin_gemm` and `scaled_mm_int8` take as `a` and
    `a_scales`; z where a residual was given, the next residual, else None; y rounded to x's type where `with_norm`
    (for a router, which reads 16 bits), else None.  The codes are those of y itself, not of the rounded norm.
    epsilon is at least 2^-126, so that rows of zeros stay zeros.  A row with an infinity or a NaN in z has the scale NaN, and
    so has every row where the weight holds a NaN; the codes are then 0 (int8) or NaN (fp8)."""
    got = _rms_norm_per_token_quant(x, weight, residual, epsilon, quant_dtype, with_norm)
    return got[0], got[1], got[2] if residual is not None else None, got[-1] if with_norm else None


def scaled_mm_int8(a: torch.Tensor, b: torch.Tensor, a_scales: torch.Tensor, b_scales: torch.Tensor,
                   out_dtype: torch.dtype, bias: torch.Tensor | None = None) -> torch.Tensor:
    """Product of 8-bit integers with a scale for each token and channel (W8A8; the reference's cutlass_scaled_mm with
    int8 operands):  out = out_dtype((a @ b) * (a_scales * b_scales) + bias), the sum in 32-bit integers.

    a: int8 (..., K).  b: int8 (K, N), column by column: `weight.t()` of a checkpoint's (N, K) weight, read as it lies.
    a_scales: float32, one a token or one in all; b_scales: one a channel or one in all.  out_dtype: float16 or
    bfloat16; bias: (N,) of out_dtype.  K below 131072, where the sum could leave 32 bits."""
    return _scaled_mm_int8(a, b, a_scales, b_scales, out_dtype, bias)


def topk_routing(gating_output: torch.Tensor, topk: int, scoring_func: str = "softmax", renormalize: bool = False,
                 bias: torch.Tensor | None = None, num_expert_group: int = 1, topk_group: int = 1,
                 routed_scaling_factor: float = 1.0):
    """The experts of each token and their weights: (topk_weights float32, topk_ids int32), both (tokens, topk), as
    `fused_marlin_moe` takes them.  gating_output: the router's logits (tokens, experts), float16, bfloat16 or float32.

    Scores are softmax(logits) or sigmoid(logits) (`scoring_func`); experts are chosen by score + bias (float32,
    (experts,); the bias balances loads and is no part of a weight), in falling order, equal ones by the lower number.
    With num_expert_group > 1 neighbouring experts form groups, and only those of the topk_group best groups may be
    chosen; a group counts by its best expert or, with a bias, by the sum of its two best.  The weights are the scores of
    the chosen, divided by their sum if `renormalize`, times routed_scaling_factor.  A NaN logit counts as -inf; a token
    whose logits are all -inf gets the lowest experts that may be chosen, with softmax weights 0.  With a bias an expert of
    logit -inf has the score 0 and may still be chosen, by its bias: a bias of -inf leaves it out (a NaN bias does too).
    At most 1024 experts, 64 groups, 64 choices."""
    return _topk_routing(gating_output, topk, scoring_func, renormalize, bias, num_expert_group, topk_group,
                         routed_scaling_factor)


def qk_norm_rope(query: torch.Tensor, key: torch.Tensor, positions: torch.Tensor | None = None,
                 cos_sin_cache: torch.Tensor | None = None, q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
                 epsilon: float = 1e-6, is_neox: bool = True):
    """Norm of each query and key head and rotation by the token's position, in one launch: (query, key), new tensors of the inputs'
    shapes.

      y = x / sqrt(mean(x^2) + epsilon) * weight over head_dim, where a weight is given;
      the first rotary_dim numbers in pairs (a, b) -> (a cos - b sin, b cos + a sin), where a table is given

    all in float32, rounded once.  query: (tokens, heads, head_dim), key: (tokens, kv_heads, head_dim), float16, bfloat16 or float32,
    of any strides: views of the qkv projection's output are read as they lie.  positions: (tokens,), int64 or int32.
    cos_sin_cache: float32 (positions, rotary_dim), a position's cosines, then its sines (`rotary.rotary_cos_sin` makes one; a scaling
    for long contexts is in it).  is_neox: pairs are (i, i + rotary_dim / 2), else neighbours.  Weights: (head_dim,) of query's type.
    A position outside the table turns the token's rotated numbers into NaN.  head_dim at most 1024, epsilon at least 2^-126."""
    return _qk_norm_rope(query, key, positions, cos_sin_cache, q_weight, k_weight, epsilon, is_neox)


def qk_norm_rope_append(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                        slot_mapping: torch.Tensor, positions: torch.Tensor | None = None, cos_sin_cache: torch.Tensor | None = None,
                        q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, epsilon: float = 1e-6,
                        is_neox: bool = True, k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None) -> torch.Tensor:
    """`qk_norm_rope` whose keys go, with the values, to the pages of a cache: returns the queries.

    key_cache, value_cache: (pages, page_size, kv_heads, head_dim) of any strides but the last (a layout with the heads before the
    slots is a transposed view), of query's type or float8_e4m3fn.  An 8-bit cache holds codes that stand for code * scale: the nearest
    to y / scale, at most 448; k_scale and v_scale: float32, one positive number or one a kv head.  slot_mapping: (tokens,), int64 or int32:
    token t goes to slot s % page_size of page s // page_size, s = slot_mapping[t]; nowhere where s is negative or past the last page.
    Which of two tokens with the same slot stays is not defined, for each head anew.  Without a table and weights this is the plain append."""
    return _qk_norm_rope_append(query, key, value, key_cache, value_cache, slot_mapping, positions, cos_sin_cache, q_weight, k_weight,
                                epsilon, is_neox, k_scale, v_scale)


def paged_attention(query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, block_table: torch.Tensor,
                    seq_lens: torch.Tensor, query_start_loc: torch.Tensor, scale: float | None = None, causal: bool = True,
                    window: int = 0, softcap: float = 0.0, alibi_slopes: torch.Tensor | None = None,
                    tree_mask: torch.Tensor | None = None, k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                    max_seq_len: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of a ragged batch over a paged cache, which holds the batch's own keys and values already (`qk_norm_rope_append`):
    prompts, pieces of prompts, single tokens and trees of drafted tokens, in any mixture.

    query: (tokens, heads, head_dim), float16 or bfloat16; sequence i's queries are the tokens query_start_loc[i] up to
    query_start_loc[i + 1] (int32, (sequences + 1,), from 0 on), the last ones of its seq_lens[i] tokens (int32, (sequences,)).
    Caches as `qk_norm_rope_append` fills them, 16-byte aligned; block_table: int32 (sequences, pages), key p of sequence i is in page
    block_table[i, p // page_size].  heads is a multiple of the cache's kv heads, neighbours share one.  scale: head_dim ** -0.5.

      s = scale * (q . k);  softcap > 0: softcap * tanh(s / softcap);  alibi_slopes (float32, (heads,)): s - slope * |distance|
      out = softmax(s over the keys that the query sees) v

    causal: a query sees its own and earlier keys, with window > 0 the last `window` of them; not causal: every key of its sequence.
    tree_mask (int64, (tokens, words)): a query sees the keys before its sequence's queries, and of those the ones whose bits are set:
    bit c % 64 of word c // 64 is query c of the sequence (a draft's own bit among them); it takes the place of `causal` and goes with
    neither window nor slopes.  A query that sees no key gives zeros, as do tokens behind the last sequence; with `out`, those are left as
    they are.  One that sees a score of +infinity or NaN, or none but -infinity, gives NaN.  NaNs and infinities in what a query does not see do not reach it.  Pages that no query sees are not read; a
    page number outside the cache among the others makes the results of the queries that see a key of it NaN.

    max_seq_len: the longest sequence, if the caller knows: how far the keys may be split over workgroups is chosen for it, and for
    all of the block table without it (a captured call whose lengths change does without); results are right, if not the same bits, for
    any number.  scale, and softcap if not 0, from 1e-30 to 1e30; k_scale negative or NaN makes the results NaN.
    head_dim a multiple of 16, at most 256."""
    if scale is None:
        scale = query.shape[-1] ** -0.5
    if out is None:
        return _paged_attention(query, key_cache, value_cache, block_table, seq_lens, query_start_loc, scale, causal, window, softcap,
                                alibi_slopes, tree_mask, k_scale, v_scale, max_seq_len)
    _paged_attention_out(query, key_cache, value_cache, block_table, seq_lens, query_start_loc, scale, causal, window, softcap,
                         alibi_slopes, tree_mask, k_scale, v_scale, max_seq_len, out)
    return out


def marlin_gemm(a: torch.Tensor, c: torch.Tensor | None, b_q_weight: torch.Tensor,
                b_bias: torch.Tensor | None, b_scales: torch.Tensor, a_scales: torch.Tensor | None,
                global_scale: torch.Tensor | None, b_zeros: torch.Tensor | None,
                g_idx: torch.Tensor | None, perm: torch.Tensor | None, workspace: torch.Tensor,
                b_q_type: ScalarType, size_m: int, size_n: int, size_k: int, is_k_full: bool = True,
                use_atomic_add: bool = False, use_fp32_reduce: bool = False,
                is_zp_float: bool = False) -> torch.Tensor:
    return torch.ops._C.marlin_gemm(a, c, b_q_weight, b_bias, b_scales, a_scales, global_scale, b_zeros,
                                    g_idx, perm, workspace, b_q_type.id, size_m, size_n, size_k,
                                    is_k_full, use_atomic_add, use_fp32_reduce, is_zp_float)


gptq_marlin_gemm = marlin_gemm  # the op's older name

# a linear layer in one op call (no reference counterpart): torch_bindings.cpp says what each argument is
marlin_linear = torch.ops.sonar_amd.marlin_linear.default


def moe_wna16_marlin_gemm(input: torch.Tensor, output: torch.Tensor | None, b_qweight: torch.Tensor,
                          b_bias: torch.Tensor | None, b_scales: torch.Tensor,
                          a_scales: torch.Tensor | None, global_scale: torch.Tensor | None,
                          b_qzeros: torch.Tensor | None, g_idx: torch.Tensor | None,
                          perm: torch.Tensor | None, workspace: torch.Tensor,
                          sorted_token_ids: torch.Tensor, expert_ids: torch.Tensor,
                          num_tokens_past_padded: torch.Tensor, topk_weights: torch.Tensor,
                          moe_block_size: int, top_k: int, mul_topk_weights: bool,
                          b_q_type: ScalarType, size_m: int, size_n: int, size_k: int, is_k_full: bool,
                          use_atomic_add: bool, use_fp32_reduce: bool, is_zp_float: bool,
                          thread_k: int = -1, thread_n: int = -1, blocks_per_sm: int = -1) -> torch.Tensor:
    return torch.ops._moe_C.moe_wna16_marlin_gemm(
        input, output, b_qweight, b_bias, b_scales, a_scales, global_scale, b_qzeros, g_idx, perm,
        workspace, sorted_token_ids, expert_ids, num_tokens_past_padded, topk_weights, moe_block_size,
        top_k, mul_topk_weights, b_q_type.id, size_m, size_n, size_k, is_k_full, use_atomic_add,
        use_fp32_reduce, is_zp_float, thread_k, thread_n, blocks_per_sm)


def marlin_to_gfx950(b_q_weight: torch.Tensor, size_k: int, size_n: int) -> torch.Tensor:
    """Marlin tile order -> the order the gfx950 kernels stream (no reference counterpart)."""
    return torch.ops._C.marlin_to_gfx950(b_q_weight, size_k, size_n)


def marlin_weight_cache_clear() -> int:
    """Drops the converted weight copies the GEMM ops keep; returns how many there were."""
    return torch.ops._C.marlin_weight_cache_clear()


def marlin_weight_cache_invalidate(t: torch.Tensor) -> int:
    """Drops the converted copies made from the memory of `t` (a Marlin weight tensor or a
    tensor of float8_e8m0fnu block scales); returns how many.  Needed after the bytes of `t`
    were rewritten in place in a way its version counter does not show (`t.data.copy_(...)`,
    any write to an inference-mode tensor).  Weights that come out of the repack ops, and
    in-place ops on `t` itself, need no call."""
    return torch.ops._C.marlin_weight_cache_invalidate(t)
