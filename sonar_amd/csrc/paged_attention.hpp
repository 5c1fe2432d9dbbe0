// What the kernels of the attention over a paged cache share: the arguments, the search of a workgroup's rows, masks, page
// addresses, element types.
#pragma once

#include "common.hpp"
#include "lane_reduce.hpp"
#include "sonar_attention.h"

namespace sonar {

typedef float floatx16_t __attribute__((ext_vector_type(16)));
typedef short short4_t __attribute__((ext_vector_type(4)));
typedef short short8_t __attribute__((ext_vector_type(8)));

constexpr float kLog2E = 1.4426950408889634f;
constexpr float kInfinity = __builtin_inff();

struct CachePages {
  const char* data;
  long page, slot, head;   // strides in bytes
  const float* scale;      // NULL: 1
  int scale_heads;         // scale holds a number for each kv head
};

struct AttentionParams {
  const char* q;
  long q_token, q_head;   // strides in elements
  CachePages k, v;
  const int32_t* table;
  long table_stride;
  const int32_t *lens, *starts;
  char* out;
  long out_token, out_head;
  const float* slopes;
  const uint64_t* tree;
  float* part_o;    // [split][token][head][dim], not yet divided by the sum
  float2* part_ml;  // [split][token][head]: running maximum (of scores times log2 e) and sum
  float scale, cap;
  uint32_t page_magic;   // key / page_size = key * page_magic >> page_shift for keys below 2^31
  int page_shift, page_size, pages, table_pages;
  int window, tree_words, tokens, seqs, heads, kv_heads, group, dim;
  int blocks, splits, split_tiles;   // blocks of rows; at most `splits` parts of the keys, of `split_tiles` tiles at least
  bool causal, clear_rest;
};

// Rows are pairs (token, query head of the kv head), the head fastest.  A sequence's rows start a new block.
struct RowBlock {
  int seq;        // seqs: the tokens behind the last sequence
  int token;      // the sequence's first
  int first;      // row of the block's first one in its sequence
  int rows;       // of the sequence
  int len, past;  // keys of the sequence; position of its first query
};

// The sequence of block `b`: sequence i owns the numbers from starts[i] * group / ROWS + i on, which are as many as its blocks
// or one more.  A wavefront searches 64 places at a time.
template <int ROWS>
__device__ __forceinline__ RowBlock row_block(const AttentionParams& p, int b) {
  const int lane = threadIdx.x & 63;
  auto start = [&](int i) { return (int)min(max(p.starts[i], 0), p.tokens); };
  auto number = [&](int i) { return (int)((long)start(i) * p.group / ROWS) + i; };
  int low = 0, count = p.seqs + 1;
  while (count > 1) {
    const int step = (count + 63) / 64, i = lane * step;
    const uint64_t below = __ballot(i < count && number(low + min(i, count - 1)) <= b);
    const int last = max(__builtin_popcountll(below) - 1, 0) * step;
    low += last, count = min(step, count - last);
  }
  RowBlock r;
  r.seq = __builtin_amdgcn_readfirstlane(low);
  r.token = __builtin_amdgcn_readfirstlane(start(r.seq));
  const int end = r.seq < p.seqs ? __builtin_amdgcn_readfirstlane(start(r.seq + 1)) : p.tokens;
  r.first = (b - __builtin_amdgcn_readfirstlane(number(r.seq))) * ROWS;
  r.rows = max(end - r.token, 0) * p.group;
  r.len = r.seq < p.seqs ? (int)min((long)max(p.lens[r.seq], 0), (long)p.table_pages * p.page_size) : 0;
  r.past = r.len - (end - r.token);
  return r;
}

// Keys [low, high) that a query of tokens [t0, t1] of the sequence may see, t counted from its first query.
__device__ __forceinline__ void keys_seen(const AttentionParams& p, const RowBlock& r, int t0, int t1, int& low, int& high) {
  const bool bounded = p.causal && p.tree == nullptr;
  high = bounded ? min(r.len, max(r.past + t1 + 1, 0)) : r.len;
  low = bounded && p.window > 0 ? max(r.past + t0 - p.window + 1, 0) : 0;
}

// The part of the tiles [first, last) of a block that split s takes; false where there is none.  Sets how many parts there are.
__device__ __forceinline__ bool split_of(const AttentionParams& p, int s, int& first, int& last, int& parts) {
  const int tiles = last - first, each = max(p.split_tiles, (tiles + p.splits - 1) / p.splits);
  parts = max((tiles + each - 1) / each, 1);
  first += s * each;
  last = min(last, first + each);
  return s < parts;
}

// Which of the 64 keys from `base` on a query sees, a bit each.
struct Sight {
  int position, len, past, low_bound;
  const uint64_t* tree;   // the query's words, or NULL
  int words;
  bool causal;
  __device__ __forceinline__ static uint64_t below(int n) { return n <= 0 ? 0 : n >= 64 ? ~0ull : (1ull << n) - 1; }
  __device__ __forceinline__ uint64_t word(int w) const { return w < 0 ? ~0ull : w >= words ? 0 : tree[w]; }
  __device__ __forceinline__ uint64_t of(int base) const {
    uint64_t seen = below((causal && tree == nullptr ? min(len, position + 1) : len) - base) & ~below(low_bound - base);
    if (tree != nullptr) {
      const int from = base - past, w = from >> 6, s = from & 63;
      seen &= s == 0 ? word(w) : word(w) >> s | word(w + 1) << (64 - s);
    }
    return seen;
  }
};

__device__ __forceinline__ int page_of(const AttentionParams& p, int key) {
  return (int)((uint64_t)(uint32_t)key * p.page_magic >> p.page_shift);
}

// The number of a page as it may be used; `bad` where the table's is none.
__device__ __forceinline__ int page_number(const AttentionParams& p, int number, bool& bad) {
  if ((uint32_t)number < (uint32_t)p.pages) return number;
  bad = true;
  return 0;
}

template <typename T>
struct Element;
template <>
struct Element<__bf16> {
  typedef bf16x8_t eight;
  static constexpr uint16_t kExponent = 0x7f80;
  __device__ __forceinline__ static floatx16_t mfma32(eight a, eight b, floatx16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  __device__ __forceinline__ static floatx4_t mfma16(eight a, eight b, floatx4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  template <bool HIGH>
  __device__ __forceinline__ static uint32_t from_fp8(uint32_t v) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, 1.0f, HIGH));
  }
};
template <>
struct Element<_Float16> {
  typedef half8_t eight;
  static constexpr uint16_t kExponent = 0x7c00;
  __device__ __forceinline__ static floatx16_t mfma32(eight a, eight b, floatx16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  __device__ __forceinline__ static floatx4_t mfma16(eight a, eight b, floatx4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  template <bool HIGH>
  __device__ __forceinline__ static uint32_t from_fp8(uint32_t v) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v, 1.0f, HIGH));
  }
};

// Sixteen (eight) float8_e4m3fn codes as 16-bit numbers: exact.
template <typename T>
__device__ __forceinline__ u32x4_t widen(uint32_t a, uint32_t b) {
  typedef Element<T> E;
  return u32x4_t{E::template from_fp8<false>(a), E::template from_fp8<true>(a), E::template from_fp8<false>(b),
                 E::template from_fp8<true>(b)};
}

// Eight 16-bit numbers with 0 in the place of infinities and NaNs; `found` where there are some.
template <typename T>
__device__ __forceinline__ u32x4_t finite_part(u32x4_t v, bool& found) {
  constexpr uint32_t kLow = Element<T>::kExponent, kHigh = kLow << 16;
  u32x4_t out;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t keep = ((v[i] & kLow) == kLow ? 0 : 0xffffu) | ((v[i] & kHigh) == kHigh ? 0 : 0xffff0000u);
    found |= keep != ~0u;
    out[i] = v[i] & keep;
  }
  return out;
}

// Four keys (rows `pitch` apart) of sixteen neighbouring columns, turned: lane i of each 16 gets column i's four numbers.
// `at`: this lane's part, row i / 4, column 4 * (i % 4).
__device__ __forceinline__ short4_t turned(const char* at) {
  typedef __attribute__((address_space(3))) short4_t lds_short4;
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)at);
}

// `join` with lane l ^ 32's (HALVES) or l ^ 16's value
template <bool HALVES, typename F>
__device__ __forceinline__ float joined(float v, F join) {
  uint32_t one, other;
  sides<HALVES>(__builtin_bit_cast(uint32_t, v), one, other);
  return join(__builtin_bit_cast(float, one), __builtin_bit_cast(float, other));
}

}  // namespace sonar
