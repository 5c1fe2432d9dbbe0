/*
 * sonar_attention.h - C ABI of the operators of a decoder layer between its qkv projection and its output projection
 * (MI355X, gfx950): norms and position rotation of the heads, the append to a paged cache, attention over the pages.
 *
 * The conventions are those of sonar_marlin.h: plain device pointers, sizes and a HIP stream (void*; NULL is the null
 * stream), all work enqueued on that stream, no synchronisation with the host, 0 or a negative SONAR_E_* code, nothing
 * launched when a call fails.  sonar_attention_last_error() returns the calling thread's message.  The element types are
 * SONAR_DTYPE_F16 / _BF16 / _F32.  Strides count elements.  Nothing is kept from one call to the next.
 */
#ifndef SONAR_ATTENTION_H_
#define SONAR_ATTENTION_H_

#include "sonar_marlin.h"

#ifdef __cplusplus
extern "C" {
#endif

const char* sonar_attention_last_error(void);

/* A paged cache of keys or values: element (page, slot, head, d) lies at data + page * page_stride + slot * slot_stride +
 * head * head_stride + d.  `dtype` is the element type, or SONAR_CACHE_FP8 for float8_e4m3fn codes, which stand for
 * code * scale; `scale` holds 1 or kv_heads float32 numbers on the device (scale_len; NULL for 16- and 32-bit caches), which must be
 * positive: a negative or NaN scale of the keys makes attention's results NaN. */
#define SONAR_CACHE_FP8 3
typedef struct sonar_kv_cache {
  void* data;
  int64_t page_stride, slot_stride, head_stride;
  const float* scale;
  int64_t scale_len;
} sonar_kv_cache;

/* Norm of each query and key head and rotation by the token's position, in one pass; keys and values go to new rows or to
 * the pages of a cache.  For a head x of head_dim numbers:
 *   y = x * r * weight, r = 1 / sqrt(mean(x^2) + epsilon)   (x itself without a weight)
 *   the first rotary_dim numbers in pairs (a, b) -> (a cos - b sin, b cos + a sin): pairs (i, i + rotary_dim / 2) where
 *   `half`, else (2i, 2i + 1); cos and sin of pair i are cos_sin[position][i] and cos_sin[position][rotary_dim / 2 + i]
 * in fp32, rounded once.  Values are copied.  An 8-bit cache gets float8_e4m3fn(clamp(y * (1 / scale), -448, 448)), the
 * nearest code.  A position outside [0, max_position) turns the rotated numbers of its token into NaN.
 *   q, k, v        dtype (token, head, d) with strides; v NULL without a cache
 *   positions      int64 (positions_64) or int32 [tokens], cos_sin float[max_position][rotary_dim]; both NULL: no rotation
 *   q_weight, k_weight  dtype[head_dim] or NULL
 *   epsilon        at least 2^-126
 *   q_out          dtype[tokens][heads][head_dim];  k_out dtype[tokens][kv_heads][head_dim], NULL with a cache
 *   key_cache, value_cache  both or neither; cache_dtype: dtype or SONAR_CACHE_FP8 (not with F32)
 *   slots          int64 (slots_64) or int32 [tokens]: token t goes to slot slots[t] % page_size of page slots[t] / page_size;
 *                  numbers outside [0, pages * page_size) go nowhere.  Which of two tokens with one slot
 *                  stays is not defined, for each head anew.
 * tokens * (heads + 2 kv_heads) below 2^31, head_dim at most 1024. */
int sonar_qk_norm_rope(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k, int64_t k_token_stride,
                       int64_t k_head_stride, const void* v, int64_t v_token_stride, int64_t v_head_stride, const void* positions,
                       int positions_64, const float* cos_sin, int64_t max_position, int64_t rotary_dim, int half,
                       const void* q_weight, const void* k_weight, double epsilon, void* q_out, void* k_out,
                       const sonar_kv_cache* key_cache, const sonar_kv_cache* value_cache, int cache_dtype, const void* slots,
                       int slots_64, int64_t pages, int64_t page_size, int dtype, int64_t tokens, int64_t heads,
                       int64_t kv_heads, int64_t head_dim, void* stream);

/* Attention of a ragged batch over a paged cache that already holds the batch's own keys and values.  Sequence i has
 * seq_lens[i] keys, key p in slot p % page_size of page block_table[i][p / page_size]; its queries, the tokens starts[i] to
 * starts[i + 1] - 1, are its last ones: query j has the position seq_lens[i] - (starts[i + 1] - starts[i]) + j.  Query head h
 * reads kv head h / (heads / kv_heads).
 *   s = scale * (q . k);  cap > 0: s = cap * tanh(s / cap);  slopes: s -= slopes[h] * |query position - key position|
 *   out = sum over the keys that the query sees of softmax(s) * v, rounded once; a query that sees none gives zeros, one all of
 *   whose scores are -infinity, or one of them NaN or +infinity, NaN
 * A query at position t sees key p < seq_lens[i] where
 *   causal: p <= t, and with window > 0 also p > t - window (the last `window` keys, its own among them);
 *   tree_mask: p lies before the sequence's queries, or is its query c (p = seq_lens[i] - queries + c) and bit c % 64 of
 *   tree_mask[token][c / 64] is set, c < 64 * tree_words.  Neither slopes nor a window go with a tree mask, nor a window with causal = 0.
 * What lies in masked places, NaN included, does not reach the result.  Pages that no query sees are not read, and their
 * numbers not looked at; a number outside [0, pages) among the others makes the results of the queries that see a key of that page NaN,
 * and no others.  seq_lens are taken as at most table_pages * page_size.  Tokens from starts[seqs] on get zeros where clear_rest, else are left as they are.
 *   q, out      dtype (SONAR_DTYPE_F16 / _BF16) (token, head, d) with strides; q 16-byte aligned, its strides multiples of 8; out 8-byte
 *               aligned, its strides multiples of 4; out does not overlap the inputs
 *   caches      of dtype or SONAR_CACHE_FP8; 16-byte aligned, strides multiples of 16 bytes; page_size slots a page; 64 GiB at most
 *   block_table int32[seqs][table_stride], table_pages of a row in use;  seq_lens int32[seqs];  starts int32[seqs + 1], rising, from 0
 *   slopes      float[heads] or NULL;  tree_mask int64[tokens][tree_words] or NULL
 *   max_seq_len what the split of the keys is chosen for; longer sequences are right too, and much shorter ones, of up to 1024
 *               sequences, nearly as fast
 *   scratch     device memory, 16-byte aligned, of sonar_paged_attention_scratch_bytes(...) bytes (0 to 256 MiB); calls that overlap in
 *               time need scratches of their own
 * head_dim a multiple of 16, at most 256; scale, and cap if not 0, from 1e-30 to 1e30; tokens * heads below 2^31, table_pages * page_size below 2^31 - 1024. */
size_t sonar_paged_attention_scratch_bytes(int64_t tokens, int64_t seqs, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                           int cache_dtype, int64_t max_seq_len, int64_t window);
int sonar_paged_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, const sonar_kv_cache* key_cache,
                          const sonar_kv_cache* value_cache, int cache_dtype, int64_t pages, int64_t page_size,
                          const int32_t* block_table, int64_t table_stride, int64_t table_pages, const int32_t* seq_lens,
                          const int32_t* starts, void* out, int64_t out_token_stride, int64_t out_head_stride, int clear_rest,
                          double scale, double cap, int64_t window, int causal, const float* slopes, const int64_t* tree_mask,
                          int64_t tree_words, void* scratch, size_t scratch_bytes, int dtype, int64_t tokens, int64_t seqs,
                          int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t max_seq_len, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* SONAR_ATTENTION_H_ */
