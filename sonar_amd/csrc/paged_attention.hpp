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

constexpr int kTile = 64;   // keys
constexpr int kTail = 32;   // rows
constexpr float kLog2E = 1.4426950408889634f;
constexpr float kInfinity = __builtin_inff();

struct CachePages {
  const char* data;
  uint32_t page, slot;     // strides in units of 16 bytes; no cache has 2^32 of them
  long head;               // in bytes
  const float* scale;      // NULL: 1
  int scale_heads;         // scale holds a number for each kv head
};

// What parts of the keys cost in the form for many rows (us, measured): what a compute unit's workgroups take for a tile, `period` of
// them together `whole`, one or two beside those `one` and `two`; and each part, to be written, read and joined.
struct PartsCost {
  int groups, period;   // workgroups without parts
  float whole, one, two, part;
  __host__ __device__ __forceinline__ float of(int tiles, int n) const {
#pragma clang fp contract(off)
    const int workgroups = (groups * n + 255) / 256, rest = workgroups % period;   // of one compute unit
    const float tile = (float)(workgroups / period) * whole + (rest == 0 ? 0.0f : rest == 1 ? one : two);
    return (float)((tiles + n - 1) / n) * tile + (n > 1 ? 5.0f + part * (float)n : 0.0f);
  }
};
// Tiles of a sequence of `keys` keys, the last `queries` of which see them: on average.
__host__ __device__ __forceinline__ int mean_tiles(int keys, int queries) {
  return (int)(((uint32_t)keys - (uint32_t)(queries < keys ? queries : keys) / 2 + kTile - 1) / kTile);
}
// More parts are taken where they are cheaper by 3 %.
constexpr float kWorth = 0.97f;

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
  float* part_o;    // [split][token][head][dim], not yet divided by the sum; with tails [split][seq][kv head][row of kTail][dim]
  float2* part_ml;  // the same without dim: running maximum (of scores times log2 e) and sum
  float scale, cap;
  uint32_t page_magic;   // key / page_size = key * page_magic >> page_shift for keys below 2^31
  int page_shift, page_size, pages, table_pages;
  int window, tree_words, tokens, seqs, heads, kv_heads, group, dim;
  int rows, blocks, splits, split_tiles;   // rows of a block, blocks of rows; at most `splits` parts of the keys, of `split_tiles` tiles at least
  int tails;                               // not 0: at most so many parts of the sequences' last rows, where those are no more than kTail
  int longest;                             // keys of a sequence at most, as far as the host knows
  int queries;                             // of a sequence, on average
  PartsCost cost;
  float few_share;                         // not 0: parts of few_tiles() tiles at least
  bool causal, clear_rest, by_dies;
};

// Rows are pairs (token, query head of the kv head), the head fastest.  A sequence's rows start a new block.
struct RowBlock {
  int seq;        // seqs: the tokens behind the last sequence
  int token;      // the sequence's first
  int first;      // row of the block's first one in its sequence
  int rows;       // of the sequence
  int len, past;  // keys of the sequence; position of its first query
  int longest;    // keys of the longest sequence, as far as they are known
};

// What workgroup `b` takes: a kv head and one of `items`.  Neighbouring workgroups run on different dies (8, in turn): each die gets
// items of its own with all their heads, one after the other.
__device__ __forceinline__ void item_of(const AttentionParams& p, int items, int b, int& item, int& kv_head) {
  const int whole = p.by_dies ? items / 8 * 8 : 0;
  if (b < whole * p.kv_heads) {
    kv_head = b / 8 % p.kv_heads, item = b / 8 / p.kv_heads * 8 + b % 8;
  } else {
    const int rest = b - whole * p.kv_heads;
    kv_head = rest % p.kv_heads, item = whole + rest / p.kv_heads;
  }
}

// The first token of sequence i, as far as there are tokens.
__device__ __forceinline__ int start_of(const AttentionParams& p, int i) { return min(max(p.starts[i], 0), p.tokens); }

// The last sequence i of [0, seqs] with number(i, its start) <= b, for numbers that rise from 0, and its sizes; its first row is left
// to the caller.  A wavefront looks at 64 places at a time; in the last round the lanes have the sizes too, so that a batch of up
// to 62 sequences takes one trip to memory.  Where parts are chosen by the longest length, those of up to 1024 sequences are read on the
// way (from 1025 on there are workgroups enough whatever the parts are).
template <typename F>
__device__ __forceinline__ RowBlock sequence_of(const AttentionParams& p, int b, F number) {
  const int lane = threadIdx.x & 63;
  const bool by_longest = p.splits > 1 && p.few_share == 0.0f && p.seqs <= 1024;
  int lens[4] = {};   // this lane's (some twice), the last one the largest of those from there on
  if (by_longest && p.seqs > 62) {
#pragma unroll
    for (int j = 0; j < 4; ++j) lens[j] = p.lens[min(lane + 64 * j, p.seqs - 1)];
    for (int i = lane + 256; i < p.seqs; i += 64) lens[3] = max(lens[3], p.lens[i]);
  }
  int low = 0, count = p.seqs + 1;
  while (count > 63) {
    const int step = (count + 63) / 64, i = low + min(lane * step, count - 1);
    const uint64_t below = __ballot(lane * step < count && number(i, start_of(p, i)) <= b);
    const int last = max(__builtin_popcountll(below) - 1, 0) * step;
    low += last, count = min(step, count - last);
  }
  const int i = low + lane;
  const int start = i <= p.seqs ? start_of(p, i) : p.tokens, len = i < p.seqs ? p.lens[i] : 0;
  const uint64_t below = __ballot(lane < count && number(i, start) <= b);
  const int found = max(__builtin_popcountll(below) - 1, 0);
  RowBlock r;
  r.seq = low + found;
  r.token = of_lane(start, found);
  const int end = r.seq < p.seqs ? of_lane(start, found + 1) : p.tokens;
  r.rows = max(end - r.token, 0) * p.group;
  r.len = (int)min((long)max(of_lane(len, found), 0), (long)p.table_pages * p.page_size);
  r.past = r.len - (end - r.token);
  r.longest = p.longest;
  if (by_longest) {
    auto larger = [](int a, int b) { return max(a, b); };
    r.longest = min(over_wave(p.seqs <= 62 ? len : max(max(lens[0], lens[1]), max(lens[2], lens[3])), 0, larger), p.longest);
  }
  return r;
}

// Block `b` of rows: sequence i owns the numbers from starts[i] * group / ROWS + i on, which are as many as its blocks or one more.
template <int ROWS>
__device__ __forceinline__ RowBlock row_block(const AttentionParams& p, int b) {
  auto number = [&](int i, int start) { return (int)((long)start * p.group / ROWS) + i; };
  RowBlock r = sequence_of(p, b, number);
  r.first = (b - number(r.seq, r.token)) * ROWS;
  return r;
}

// The last rows of sequence `i`, in blocks of p.rows.
__device__ __forceinline__ RowBlock last_rows(const AttentionParams& p, int i) {
  RowBlock r;
  r.seq = i, r.token = start_of(p, i), r.longest = p.longest;
  const int queries = max(start_of(p, i + 1) - r.token, 0);
  r.rows = queries * p.group, r.first = max(r.rows - 1, 0) / p.rows * p.rows;
  r.len = (int)min((long)max(p.lens[i], 0), (long)p.table_pages * p.page_size), r.past = r.len - queries;
  return r;
}
__device__ __forceinline__ bool is_tail(const RowBlock& r) { return r.rows - r.first <= kTail; }

// Keys [low, high) that a query of tokens [t0, t1] of the sequence may see, t counted from its first query.
__device__ __forceinline__ void keys_seen(const AttentionParams& p, const RowBlock& r, int t0, int t1, int& low, int& high) {
  const bool bounded = p.causal && p.tree == nullptr;
  high = bounded ? min(r.len, max(r.past + t1 + 1, 0)) : r.len;
  low = bounded && p.window > 0 ? max(r.past + t0 - p.window + 1, 0) : 0;
}

// Tiles of a part at least, of `tiles` in all, in the form for few rows.  `share`: kv heads and their blocks of rows over 4096.  With t tiles
// a workgroup takes some 0.6 t us, and joining the others 0.1 us a part, so that the square root of 0.15 times the tiles is about the
// best for one sequence (8000 keys: 4 tiles 17.2 us, 2 19.1); with more of them about 4096 workgroups, which even out (64 sequences
// of 800 to 4096 keys: 155 us with 8 tiles, 4 158, 16 164).
__host__ __device__ __forceinline__ int few_tiles(int tiles, float share) {
  const int for_many = (int)(share * (float)tiles);
  const int for_one = 2 + (tiles >= 59) + (tiles >= 105) + (tiles >= 165) + (tiles >= 239) + (tiles >= 325) + (tiles >= 425);   // 3 to 8 squared
  return for_many < for_one ? for_one : for_many > 8 ? 8 : for_many;
}

// Tiles of a part at least in the form for many rows.  Where the longest sequence is shorter than the host knew, the host's choice of
// parts is made anew: each lane prices a number of parts, of which there are no more than the host's.  (64 sequences of 800 to 4096 keys of
// one kv head that might have had 131072 take 28 us, with parts chosen for those 82; 32 of 33 tokens with 4096 keys 214 and 287.)
__device__ __forceinline__ int many_tiles(const AttentionParams& p, const RowBlock& r) {
  const int longest = (r.longest + kTile - 1) / kTile;
  int parts = p.splits;
  if (parts > 1 && longest < (p.longest + kTile - 1) / kTile) {
    const int tiles = max(mean_tiles(r.longest, p.queries), 1), lane = threadIdx.x & 63;
    const float time = p.cost.of(tiles, lane + 1);
    const int most = min(p.splits, tiles);
    float best = of_lane(time, 0);
    parts = 1;
    for (;;) {
      const uint64_t better = __ballot(lane >= parts && lane < most && time < kWorth * best);
      if (better == 0) break;
      parts = __builtin_ctzll(better) + 1;
      best = of_lane(time, parts - 1);
    }
  }
  return max(p.split_tiles, (longest + parts - 1) / parts);
}

// The part of the tiles [first, last) of a block that split s takes; false where there is none.  Sets how many parts there are.  Of how many
// tiles a part is, the lengths say that there are.
__device__ __forceinline__ bool split_of(const AttentionParams& p, const RowBlock& r, int s, int& first, int& last, int& parts) {
  const int tiles = last - first;
  // few rows: parts of each sequence's own size; many: of one size for all, so that what is short is not cut for nothing
  const int least = p.tails > 0 ? (is_tail(r) ? 4 : max(tiles, 1)) : p.few_share > 0.0f ? few_tiles(tiles, p.few_share) : many_tiles(p, r);
  const int most = p.tails > 0 ? p.tails : p.splits, each = max(least, (tiles + most - 1) / most);
  parts = max((tiles + each - 1) / each, 1);
  first += s * each;
  last = min(last, first + each);
  return s < parts;
}

// Where part `split` of a row lies.
__device__ __forceinline__ long part_at(const AttentionParams& p, const RowBlock& r, int split, int kv_head, int row) {
  if (p.tails > 0) return (((long)split * p.seqs + r.seq) * p.kv_heads + kv_head) * kTail + row - r.first;
  return ((long)split * p.tokens + r.token + row / p.group) * p.heads + kv_head * p.group + row % p.group;
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

// Whether query `t` of the sequence sees any key.
__device__ __forceinline__ bool sees_any(const AttentionParams& p, const RowBlock& r, int t) {
  if (p.tree == nullptr) {
    int low, high;
    keys_seen(p, r, t, t, low, high);
    return high > low;
  }
  uint64_t seen = r.past > 0 && r.len > 0;
  const uint64_t* words = p.tree + (long)(r.token + t) * p.tree_words;   // (of queries whose keys are 0 to len - 1)
  for (int w = 0; w < p.tree_words && 64 * w < r.len - r.past; ++w)
    seen |= words[w] & Sight::below(r.len - r.past - 64 * w) & ~Sight::below(-r.past - 64 * w);
  return seen != 0;
}

// What a row's sums are multiplied by.  A sum of 0 is that of a query without keys, whose result is 0, or of one all of whose scores
// are -infinity, whose result is NaN: the largest of finite scores has a weight of 1 or more.
__device__ __forceinline__ float row_scale(const AttentionParams& p, const RowBlock& r, int t, int kv_head, float sum) {
  if (sum == 0.0f) return sees_any(p, r, t) ? __builtin_nanf("") : 0.0f;
  return (p.v.scale == nullptr ? 1.0f : p.v.scale[p.v.scale_heads ? kv_head : 0]) / sum;
}

// A score where bit `i` of `seen` is set, else -infinity.
__device__ __forceinline__ float shown(float score, uint32_t seen, int i) {
  const uint32_t keep = (uint32_t)__builtin_amdgcn_sbfe((int)seen, i, 1);
  return __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, score) & keep) | (__builtin_bit_cast(uint32_t, -kInfinity) & ~keep));
}

__device__ __forceinline__ int page_of(const AttentionParams& p, int key) {
  return (int)((uint64_t)(uint32_t)key * p.page_magic >> p.page_shift);
}

// Where a key's row lies in a cache, in units of 16 bytes from a head's first page; `number`: its page's number, `bad` where that is none.
__device__ __forceinline__ uint32_t place_of(const AttentionParams& p, const CachePages& c, int key, int at, int number, bool& bad) {
  const bool known = (uint32_t)number < (uint32_t)p.pages;
  bad |= !known;
  return (known ? number : 0) * c.page + (key - at * p.page_size) * c.slot;
}
__device__ __forceinline__ const char* row_at(const char* base, uint32_t place) { return base + ((uint64_t)place << 4); }

template <typename T>
struct Element;
template <>
struct Element<__bf16> {
  typedef bf16x8_t eight;
  static constexpr uint16_t kExponent = 0x7f80;
  static constexpr float kRaise = 0.0f;   // weights are formed larger by 2 to this
  __device__ __forceinline__ static floatx16_t mfma32(eight a, eight b, floatx16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  __device__ __forceinline__ static floatx4_t mfma16(eight a, eight b, floatx4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  typedef bf16x2_t two;
  __device__ __forceinline__ static two pair(float a, float b) { return two{(__bf16)a, (__bf16)b}; }
  // `to` and two numbers, added in fp32 by one instruction
  __device__ __forceinline__ static float add(two v, float to) {
    return __builtin_amdgcn_fdot2_f32_bf16(v, two{(__bf16)1.0f, (__bf16)1.0f}, to, false);
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
  static constexpr float kRaise = 7.0f;   // so that they use the whole range, up to 2^15
  __device__ __forceinline__ static floatx16_t mfma32(eight a, eight b, floatx16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  __device__ __forceinline__ static floatx4_t mfma16(eight a, eight b, floatx4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  typedef half2_t two;
  __device__ __forceinline__ static two pair(float a, float b) { return two{(_Float16)a, (_Float16)b}; }
  __device__ __forceinline__ static float add(two v, float to) {
    return __builtin_amdgcn_fdot2(v, two{(_Float16)1.0f, (_Float16)1.0f}, to, false);
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

// Eight 16-bit numbers with 0 in the place of infinities and NaNs; `found` is not 0 where there are some.  (An exponent of ones and
// one more carry into the sign's place, in both halves of a word at once.)
template <typename T>
__device__ __forceinline__ u32x4_t finite_part(u32x4_t v, uint32_t& found) {
  constexpr uint32_t kOnes = Element<T>::kExponent * 0x10001u, kOne = kOnes & ~(kOnes << 1) & 0x7fff7fffu;
  u32x4_t out;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t special = ((v[i] & kOnes) + kOne) & 0x80008000u;
    found |= special;
    out[i] = v[i] & ~((special >> 15) * 0xffffu);
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
