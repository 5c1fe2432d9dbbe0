/*
 * sonar_layer.h - C ABI of the operators of a decoder layer around the quantised GEMMs of sonar_marlin.h
 * (MI355X, gfx950): the norm that leaves 8-bit codes, the product of 8-bit integers, the router of an expert layer.
 *
 * The conventions are those of sonar_marlin.h: plain device pointers, sizes and a HIP stream (void*; NULL is the null
 * stream), all work enqueued on that stream, no synchronisation with the host, 0 or a negative SONAR_E_* code, nothing
 * launched when a call fails.  sonar_layer_last_error() returns the calling thread's message.  The element types are
 * SONAR_DTYPE_F16 / _BF16 / _F32, the code types SONAR_ADTYPE_INT8 / _FP8.  Nothing is kept from one call to the next.
 *
 * Counterparts in the reference, which reaches them as ops of its own extension or as Triton kernels:
 *   sonar_rms_norm_per_token_quant -> _C::rms_norm_dynamic_per_token_quant
 *   sonar_scaled_mm_int8           -> _C::cutlass_scaled_mm with int8 operands
 *   sonar_topk_routing             -> _moe_C::topk_softmax, topk_sigmoid and grouped_topk
 */
#ifndef SONAR_LAYER_H_
#define SONAR_LAYER_H_

#include "sonar_marlin.h"

#ifdef __cplusplus
extern "C" {
#endif

const char* sonar_layer_last_error(void);

/* Root-mean-square norm with the residual's addition before it and per-token 8-bit codes behind it:
 *   z = T(x + residual) (x itself without a residual), y = z * r * weight in fp32, r = 1 / sqrt(mean(z^2) + epsilon),
 *   int8: scale = max(max|y|, 1e-10) / 127, code = y * (127 / max|y|) rounded half away from zero,
 *   fp8:  scale = max(max|y| / 448, 1 / (448 * 512)), code = float8_e4m3fn(clamp(y * (1 / scale), -448, 448)).
 * The codes and scales are those of sonar_per_token_quant_int8 / _fp8 of the fp32 numbers y where all of them are numbers.
 *   x             dtype[rows][x_row_stride]
 *   residual      dtype[rows][residual_row_stride] or NULL
 *   weight        dtype[cols]
 *   residual_out  dtype[rows][cols], z; needed with a residual, NULL without.  May be x or residual itself where that
 *                 has the row stride cols; no other overlap with the inputs.
 *   norm_out      dtype[rows][cols], y rounded once; or NULL
 *   q             int8 or float8_e4m3fn [rows][cols] (q_dtype: SONAR_ADTYPE_INT8 / _FP8)
 *   scales        float[rows]
 *   epsilon       at least 2^-126, so that rows of zeros stay zeros
 * A row of y with a NaN (z holds one or an infinity, or weight holds a NaN) has the scale NaN and codes 0 (int8) or NaN (fp8);
 * an infinite weight gives the scale infinity, or NaN where z is 0 at its column. */
int sonar_rms_norm_per_token_quant(const void* x, int64_t x_row_stride, const void* residual,
                                   int64_t residual_row_stride, const void* weight, void* residual_out,
                                   void* norm_out, void* q, int q_dtype, float* scales, int dtype,
                                   int64_t rows, int64_t cols, double epsilon, void* stream);

/* Product of 8-bit integers with a scale for each token and channel:
 *   c[m][n] = T(float(sum over k of a[m][k] * b[n][k]) * (a_scales[m] * b_scales[n]) + bias[n])
 * The sum is exact (int32, size_k < 131072), so the result does not depend on how it is split.
 *   a         int8[size_m][a_row_stride]
 *   b         int8[size_n][b_row_stride]: a weight as a checkpoint holds it, one row per output channel
 *   c         dtype[size_m][size_n] (SONAR_DTYPE_F16 / _BF16)
 *   a_scales  float[a_scales_len], a_scales_len 1 or size_m; b_scales likewise, 1 or size_n
 *   bias      dtype[size_n] or NULL
 *   scratch   device memory, 16-byte aligned, of sonar_scaled_mm_int8_scratch_bytes(...) bytes (may be 0): partial sums
 *             where K is split, aligned copies of rows that are not.  A smaller one or none is allowed and slower, with the
 *             same results.  Calls that overlap in time need scratches of their own.
 *   aligned   whether a, b and both row strides are multiples of 16 bytes, the strides below 2^23
 * size_m and size_n below 2^25.  A call of 2^22 tiles or more is refused: of 256 x 256 results, which are more than the card
 * holds, or, where size_k is below 16 and where rows that are not aligned have no scratch, of 64 x 64. */
size_t sonar_scaled_mm_int8_scratch_bytes(int64_t size_m, int64_t size_n, int64_t size_k, int aligned);
int sonar_scaled_mm_int8(const int8_t* a, int64_t a_row_stride, const int8_t* b, int64_t b_row_stride, void* c,
                         const float* a_scales, int64_t a_scales_len, const float* b_scales,
                         int64_t b_scales_len, const void* bias, void* scratch, size_t scratch_bytes, int dtype,
                         int64_t size_m, int64_t size_n, int64_t size_k, void* stream);

/* The experts of each token and their weights, from the router's logits x:
 *   s = softmax(x) or 1 / (1 + exp(-x)); a NaN logit counts as -infinity; +infinities share a softmax evenly, and a
 *       token whose logits are all -infinity has the scores 0
 *   choice c = s + bias, or, without a bias, x (the order of s)
 *   groups > 1: experts / groups neighbours form a group; its score is the largest c in it or, with a bias, the sum of
 *       its two largest; experts outside the kept_groups best groups are left out
 *   ids: the topk largest c in falling order; weights: s of them, divided by their sum if renormalize (and the sum is
 *       not 0), times factor
 * Equal choices and equal group scores go to the lowest index; a NaN bias counts as -infinity.
 *   logits   dtype[tokens][row_stride] (SONAR_DTYPE_F16, _BF16 or _F32)
 *   bias     float[experts] or NULL
 *   weights  float[tokens][topk], ids int32[tokens][topk]
 * At most 1024 experts, 64 groups, 64 choices a token; topk <= kept_groups * (experts / groups). */
#define SONAR_SCORING_SOFTMAX 0
#define SONAR_SCORING_SIGMOID 1
int sonar_topk_routing(const void* logits, int dtype, int64_t row_stride, const float* bias, float* weights,
                       int32_t* ids, int64_t tokens, int64_t experts, int64_t topk, int scoring,
                       int renormalize, int64_t groups, int64_t kept_groups, double factor, void* stream);

/* Diagnostics for tests.  sonar_debug_int8_choice: the number of the kernel form that sonar_scaled_mm_int8 takes for a call
 * (0 general, 1 and 2 streams of up to 16 rows, 3 streams of blocks of 32, 4 to 8 tiles of 64 x 64, 64 x 128, 128 x 128, 256 x 128, 256 x 256) and
 * in how many parts it splits K; runs on the host.  sonar_debug_int8_form: the calling thread's calls take that form (-1: the
 * rule's again); a call that a stream form has too many rows for is refused. */
int sonar_debug_int8_choice(int64_t size_m, int64_t size_n, int64_t size_k, int aligned, int* splits);
int sonar_debug_int8_form(int form, int splits);

#ifdef __cplusplus
}
#endif
#endif /* SONAR_LAYER_H_ */
