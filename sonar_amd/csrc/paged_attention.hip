// Attention of a ragged batch over a paged cache: out = softmax(cap(scale * q k^T) - bias, what is masked left out) v.
//
// One pass over the keys with a running maximum m and sum l: a tile's scores s give p = 2^(s log2 e - m), out = out + p v,
// l = l + sum p, and where a score is above m by more than 8 (in powers of two) m rises to it, out and l shrinking with it.
// (Rising only then leaves p up to 2^8, which p's type and the sums hold as precisely.)  Products on the matrix
// instructions, sums in fp32; p is rounded to 16 bits for its product, by at most half a step of each.  For fp16 p is formed 2^7 times
// larger, the sums too: only what is below 2^-21 of the largest is then subnormal, and off by up to 2^-32 of it, so that 2^20 such
// keys together are off by less than half a step of the largest |v|.
//
// Both products are formed turned, k q^T and v^T p^T: a lane then holds scores of one query only, so that m, l and what
// out shrinks by are a lane's own numbers, and the scores lie where the second product takes them as its operand.  The keys of
// that product are in the order in which they fell there; v is read from LDS turned, four keys at a time, in the same order.
#include <algorithm>

#include "paged_attention.hpp"

namespace sonar {
char* last_error_buffer();
namespace {

// What turns a score q . k into a power of two: s * by, or capped cap * tanh of it as cap - 2 cap / (1 + e^2x); less the slope's part.
enum Scores { kPlain, kCapped, kSloped };   // (sloped ones may be capped too, and have slopes of 0 where the cap is large)
struct Score {
  float by, cap, slope;
  bool is_capped;
  __device__ __forceinline__ float capped(float s) const {
    return __builtin_fmaf(-2.0f * cap, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(s * by)), cap);
  }
  // The same for any cap: what is much smaller than it would be the difference of two large numbers above, off by 2^-22 of the cap.
  // Below an eighth of it four terms of tanh's series are off by 2^-29 of themselves.
  __device__ __forceinline__ float any_capped(float s) const {
    const float x = s * by * (0.5f / kLog2E), xx = x * x;
    const float series = __builtin_fmaf(xx, __builtin_fmaf(xx, __builtin_fmaf(xx, -17.0f / 315.0f, 2.0f / 15.0f), -1.0f / 3.0f), 1.0f);
    return fabsf(x) < 0.125f ? cap * (x * series) : capped(s);
  }
  __device__ __forceinline__ float sloped(float s, float distance) const { return __builtin_fmaf(-slope, fabsf(distance), s); }
};

__device__ __forceinline__ Score score_of(const AttentionParams& p, int kv_head, int head) {
  const float k_scale = p.k.scale == nullptr ? 1.0f : p.k.scale[p.k.scale_heads ? kv_head : 0];
  Score s;
  s.is_capped = p.cap > 0.0f;
  s.by = s.is_capped ? 2.0f * kLog2E * p.scale * k_scale / p.cap : p.scale * k_scale * kLog2E;
  // positive and finite, so that what is masked stays at -infinity and the largest product is the largest score
  s.by = k_scale >= 0.0f ? fminf(fmaxf(s.by, 0x1p-126f), 0x1p127f) : __builtin_nanf("");
  s.cap = p.cap * kLog2E;
  s.slope = p.slopes == nullptr ? 0.0f : p.slopes[head] * kLog2E;
  return s;
}

template <typename T>
using Four = T __attribute__((ext_vector_type(4)));
template <typename T>
__device__ __forceinline__ Four<T> four(float a, float b, float c, float d) {
  return Four<T>{(T)a, (T)b, (T)c, (T)d};
}

// The infinities and NaNs of v that were left out of the tiles in which some query's keys are masked: added to the results, which
// this workgroup has written, of the queries that see their keys (a product would have brought them to the others too, as
// 0 * NaN).  A thread a column; rare, so nothing here is fast.
template <typename T, bool FP8>
__device__ __forceinline__ void add_specials(const AttentionParams& p, const RowBlock& r, int kv_head, int split, int parts, int first,
                                             int last, int rows_end, int full_low, int full_high) {
  __threadfence();
  __syncthreads();
  const bool bounded = p.causal && p.tree == nullptr;
  for (int d = threadIdx.x; d < p.dim; d += blockDim.x)
    for (int tile = first; tile < last; ++tile) {
      if (tile * kTile >= full_low && tile * kTile + kTile <= full_high) continue;
      for (int key = tile * kTile; key < min(tile * kTile + kTile, r.len); ++key) {
        const int at = page_of(p, key);
        bool bad = false;
        const uint32_t place = place_of(p, p.v, key, at, p.table[(long)r.seq * p.table_stride + at], bad);
        const char* from = row_at(p.v.data + kv_head * p.v.head, place);
        float v;
        if (FP8) v = __builtin_amdgcn_cvt_f32_fp8((int)(uint8_t)from[d], 0);
        else v = (float)((const T*)from)[d];
        if (__builtin_isfinite(v)) continue;
        for (int row = r.first; row < rows_end; ++row) {
          const int t = row / p.group, head = kv_head * p.group + row % p.group;
          const long token = r.token + t;
          const Sight sight{r.past + t, r.len, r.past, bounded && p.window > 0 ? r.past + t - p.window + 1 : 0,
                            p.tree == nullptr ? nullptr : p.tree + token * p.tree_words, p.tree_words, p.causal};
          if (!(sight.of(key) & 1)) continue;
          if (parts > 1) {
            p.part_o[part_at(p, r, split, kv_head, row) * p.dim + d] += v;
          } else {
            T* to = (T*)p.out + token * p.out_token + head * p.out_head + d;
            *to = (T)((float)*to + v);
          }
        }
      }
    }
}

// NaN for the rows of the block that see a key whose page is none: `bad` pages were taken for the first one so far.  A thread a row; the
// keys are those of tiles [first, last), whose results this workgroup has written.
template <typename T>
__device__ __forceinline__ void spoil_rows(const AttentionParams& p, const RowBlock& r, int kv_head, int split, int parts, int first, int last,
                                           int rows_end) {
  __threadfence();
  __syncthreads();
  const bool bounded = p.causal && p.tree == nullptr;
  const int row = r.first + (int)threadIdx.x;
  if (row >= rows_end) return;
  const int t = row / p.group, end = min(last * kTile, r.len);
  const Sight sight{r.past + t, r.len, r.past, bounded && p.window > 0 ? r.past + t - p.window + 1 : 0,
                    p.tree == nullptr ? nullptr : p.tree + (long)(r.token + t) * p.tree_words, p.tree_words, p.causal};
  bool spoiled = false;
  for (int tile = first; tile < last && !spoiled; ++tile) {
    const uint64_t seen = sight.of(tile * kTile);
    for (int key = tile * kTile; key < min(tile * kTile + kTile, end) && seen != 0;) {
      const int at = page_of(p, key), next = (int)min((long)(at + 1) * p.page_size, (long)(tile * kTile + kTile));
      const bool known = (uint32_t)p.table[(long)r.seq * p.table_stride + at] < (uint32_t)p.pages;
      spoiled |= !known && (seen & Sight::below(next - tile * kTile) & ~Sight::below(key - tile * kTile)) != 0;
      key = next;
    }
  }
  if (!spoiled) return;
  if (parts > 1) {
    p.part_ml[part_at(p, r, split, kv_head, row)].y = __builtin_nanf("");
  } else {
    T* to = (T*)p.out + (long)(r.token + t) * p.out_token + (kv_head * p.group + row % p.group) * p.out_head;
    for (int d = 0; d < p.dim; ++d) to[d] = (T)__builtin_nanf("");
  }
}

// ---------------------------------------------------------------- many rows
// A workgroup takes 32 rows of a kv head for each of its WAVES wavefronts, and walks the keys in tiles of 64 that they share through
// LDS, two tiles there: while one is worked on, the next one is on its way.  Bound by the matrix pipes and the vector units together:
// 8192 tokens of 32 heads of 128 (8 kv heads) in bf16 take 550 us, 1000 TFLOP/s, with 48 % of the pipes' cycles.  Each step of the way
// there, at that size: copies through registers and products, weights, products one after the other 769; addresses found once a key
// 656; scores a half tile ahead 612; instructions in turn 586 (heads of 256: 466 to 365 for 4096 tokens); copies straight into
// LDS 574 (without them 489, without the reads of LDS too 442); wavefronts without rows copy only 567; first copies all at once and
// results through LDS 550.  Other orders of the instructions and the heads of an item on one die gave nothing.  Where a sequence
// has few rows (64 sequences of 800 to 4096 keys, 4 rows each) it is memory: 142 us, 4.6 TB/s, what a large copy reaches less 4 %.

// A row of a tile in LDS has no gap, as the copies straight into LDS leave none: its pieces of 16 bytes are swapped instead, by
// the row's number, so that the lanes which read at once find different banks: 16 lanes a piece of a row each of the keys, 32 lanes
// four pieces of four rows of the values.
template <int DP>
__device__ __forceinline__ int key_swap(int row) { return DP == 64 ? row >> 1 & 7 : row & 15; }
template <int DP>
__device__ __forceinline__ int value_swap(int row) { return DP == 64 ? (row >> 1 & 1) * 4 : (row & 3) * 4; }
template <int DP>
constexpr int rows_lds() { return 4 * kTile * DP * 2; }

// Asynchronous copy of 16 bytes a lane to LDS, lane after lane from byte `lds` on.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"   // m0 is a reserved register: that it changes is what the clobber says
__device__ __forceinline__ void copy_16_to_lds(uint32_t lds, const char* from) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(from) : "memory", "m0");
}
#pragma clang diagnostic pop

template <typename T, int DP, bool FP8, int SCORES, int WAVES>
__global__ __launch_bounds__(WAVES * 64, DP == 64 && !FP8 ? 3 : DP <= 128 ? 2 : 1) void attention_rows_kernel(const AttentionParams p) {
  typedef Element<T> E;
  typedef typename E::eight eight;
  constexpr int kRows = 32 * WAVES;
  constexpr int kSteps = DP / 16, kColumns = DP / 32, kPitch = DP * 2, kTileBytes = kTile * kPitch;
  constexpr int kLanes = FP8 ? DP / 16 : DP / 8;             // of a row, 16 bytes each
  constexpr int kGroup = 64 / kLanes;                        // rows that a wavefront copies at once
  constexpr int kPasses = kTile / (WAVES * kGroup);
  extern __shared__ __attribute__((aligned(16))) char lds[];
  char* const k_tiles = lds;
  char* const v_tiles = lds + 2 * kTileBytes;
  int* const flags = (int*)lds;   // behind the last tile

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int kv_head, split;
  RowBlock r;
  const int others = (int)blockIdx.x - p.blocks * p.splits * p.kv_heads;
  if (others < 0) {
    int item;
    item_of(p, p.blocks * p.splits, blockIdx.x, item, kv_head);
    split = item / p.blocks;
    // the blocks of the last tokens, which see the most keys, first
    r = row_block<kRows>(p, p.blocks - 1 - item % p.blocks);
  } else {   // the parts but the first of a sequence's last rows
    kv_head = others % p.kv_heads, split = 1 + others / p.kv_heads / p.seqs;
    r = last_rows(p, others / p.kv_heads % p.seqs);
    if (!is_tail(r)) return;
  }
  if (r.first < 0 || r.first >= r.rows || (r.seq == p.seqs && !p.clear_rest)) return;   // (negative where starts do not rise)

  const int row = r.first + wave * 32 + (lane & 31), half = lane >> 5;
  const int my_row = min(row, r.rows - 1), t = my_row / p.group, head = kv_head * p.group + my_row % p.group;
  const long token = r.token + t;
  const int wave_t0 = min(r.first + wave * 32, r.rows - 1) / p.group, wave_t1 = min(r.first + wave * 32 + 31, r.rows - 1) / p.group;
  const int block_t0 = r.first / p.group, block_t1 = min(r.first + kRows - 1, r.rows - 1) / p.group;
  const bool busy = r.first + wave * 32 < r.rows;   // (else the wavefront only copies)
  int low, high;
  keys_seen(p, r, block_t0, block_t1, low, high);
  int tile = low / kTile, last = high > low ? (high + kTile - 1) / kTile : low / kTile, parts;
  if (!split_of(p, r, split, tile, last, parts)) return;
  const int first_tile = tile;
  // tiles that every query of the wavefront (of the block) sees whole: from `full_low` up to `full_high`
  const bool bounded = p.causal && p.tree == nullptr;
  auto full_from = [&](int t1) { return bounded && p.window > 0 ? max(r.past + t1 - p.window + 1, 0) : 0; };
  auto full_to = [&](int t0) { return p.tree != nullptr ? min(r.len, r.past) : bounded ? min(r.len, r.past + t0 + 1) : r.len; };
  const int wave_full_low = full_from(wave_t1), wave_full_high = full_to(wave_t0);
  const int block_full_low = full_from(block_t1), block_full_high = full_to(block_t0);

  const Sight sight{r.past + t, r.len, r.past, bounded && p.window > 0 ? r.past + t - p.window + 1 : 0,
                    p.tree == nullptr ? nullptr : p.tree + token * p.tree_words, p.tree_words, p.causal};
  const Score score = score_of(p, kv_head, head);

  eight q[kSteps];
  {
    const T* from = (const T*)p.q + token * p.q_token + head * p.q_head;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int d = 16 * s + 8 * half;
      q[s] = eight{};
      if (d < p.dim) q[s] = *reinterpret_cast<const eight*>(from + d);
    }
  }

  // ---- copies of the tiles: lane l finds the places of key l, and the lanes that copy the key get them from it.  Tiles past the last
  // one find the last keys again, which nothing uses.  16-bit numbers go straight into LDS, 8-bit codes through registers.
  bool bad = false;
  int page_ahead = 0;        // the number of the page of this lane's key, a tile ahead of the places
  uint32_t places = 0;       // of its values
  uint32_t k_rows[kPasses], v_rows[kPasses];   // the places of the rows that this lane copies
  u32x4_t k_next[FP8 ? kPasses : 1], v_next[FP8 ? kPasses : 1];
  const int of_group = lane / kLanes, my_row_of_16 = wave * kGroup + of_group;   // (passes are 16 rows apart or more, but 8 in the widest form)
  const int k_chunk = FP8 ? lane % kLanes : lane % kLanes ^ key_swap<DP>(my_row_of_16);
  const int v_chunk = FP8 ? lane % kLanes : lane % kLanes ^ value_swap<DP>(my_row_of_16);
  constexpr bool kOdd = WAVES * kGroup == 8;   // every other pass is swapped by 8 pieces more
  const bool has_k = k_chunk * (FP8 ? 16 : 8) < p.dim, has_odd = (k_chunk ^ 8) * 8 < p.dim, has_v = v_chunk * (FP8 ? 16 : 8) < p.dim;
  const bool alike = p.k.page == p.v.page && p.k.slot == p.v.slot;
  const char* const k_base = p.k.data + kv_head * p.k.head + k_chunk * 16;
  const char* const v_base = p.v.data + kv_head * p.v.head + v_chunk * 16;
  const char* const k_odd = p.k.data + kv_head * p.k.head + (k_chunk ^ 8) * 16;
  const uint32_t k_lds = (uint32_t)(uintptr_t)(lds_void_t*)k_tiles + wave * 1024, v_lds = (uint32_t)(uintptr_t)(lds_void_t*)v_tiles + wave * 1024;
  const int32_t* const pages = p.table + (long)min(r.seq, p.seqs - 1) * p.table_stride;
  auto key_of = [&](int of_tile) { return min(max(of_tile * kTile + lane, low), high - 1); };
  auto look_up = [&](int of_tile) { page_ahead = pages[page_of(p, key_of(of_tile))]; };
  auto spread = [&](uint32_t (&rows)[kPasses], uint32_t place) {
#pragma unroll
    for (int i = 0; i < kPasses; ++i) rows[i] = __builtin_amdgcn_ds_bpermute(4 * ((i * WAVES + wave) * kGroup + of_group), (int)place);
  };
  auto find = [&](int of_tile) {   // the values' rows of the tile before, whose places are known, and the keys' of this one
    spread(v_rows, places);
    const int key = key_of(of_tile), at = page_of(p, key);
    const uint32_t of_keys = place_of(p, p.k, key, at, page_ahead, bad);
    places = alike ? of_keys : place_of(p, p.v, key, at, page_ahead, bad);
    spread(k_rows, of_keys);
  };
  auto fetch = [&](u32x4_t* to, const char* base, const uint32_t (&rows)[kPasses], bool has, uint32_t at, int first, int step) {
    if (!has) return;
#pragma unroll
    for (int i = first; i < kPasses; i += step) {
      if constexpr (FP8) to[i] = *reinterpret_cast<const u32x4_t*>(row_at(base, rows[i]));
      else copy_16_to_lds(__builtin_amdgcn_readfirstlane(at + i * (WAVES * 1024)), row_at(base, rows[i]));
    }
  };
  auto fetch_keys = [&](uint32_t at) {
    fetch(k_next, k_base, k_rows, has_k, at, 0, kOdd ? 2 : 1);
    if constexpr (kOdd) fetch(k_next, k_odd, k_rows, has_odd, at, 1, 2);
  };
  auto fetch_values = [&](uint32_t at) { fetch(v_next, v_base, v_rows, has_v, at, 0, 1); };
  uint32_t specials = 0;   // infinities and NaNs of v were left out of a tile that is masked for some query
  // What was fetched is in LDS when this ends, as far as this wavefront fetched it.
  auto keep = [&](char* to_k, char* to_v, bool sift) {
    if constexpr (FP8) {
      auto widened = [&](u32x4_t x, char* tiles, int swap, int i, bool sift) {
        char* row = tiles + my_row_of_16 * kPitch + i * (WAVES * kGroup * kPitch);
        u32x4_t y = widen<T>(x[2], x[3]);
        x = widen<T>(x[0], x[1]);
        if (sift) x = finite_part<T>(x, specials), y = finite_part<T>(y, specials);
        *reinterpret_cast<u32x4_t*>(row + 16 * (2 * k_chunk ^ swap)) = x;
        *reinterpret_cast<u32x4_t*>(row + 16 * (2 * k_chunk + 1 ^ swap)) = y;
      };
      if (has_k) {
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
          widened(k_next[i], to_k, key_swap<DP>(my_row_of_16), i, false);
          widened(v_next[i], to_v, value_swap<DP>(my_row_of_16), i, sift);
        }
      }
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      if (sift && has_v) {
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
          u32x4_t* at = reinterpret_cast<u32x4_t*>(to_v + (i * WAVES + wave) * 1024 + lane * 16);
          *at = finite_part<T>(*at, specials);
        }
      }
    }
  };

  // ---- 32 keys at a time: the scores of the next ones, the weights of these, the output of those before, which do not wait for
  // one another
  floatx16_t out[kColumns];
#pragma unroll
  for (int c = 0; c < kColumns; ++c) out[c] = floatx16_t{};
  float most = -kInfinity, sum = 0.0f;
  floatx16_t s[2];          // lane l has those of query l % 32 with the keys 8 (i / 4) + 4 (l / 32) + i % 4 of 32
  eight weights[2][2];      // of 32 keys
  // Half h of the tile `of_tile`: its scores become weights.  Meanwhile the scores of the half behind it are formed from k_from, and the
  // half before it, h ^ 1 of v_from, goes to the output with its weights.  The matrix pipes take 32 cycles for a product, and a
  // wavefront's instructions start in their order: so that pipes and vector units both have work, each product is followed by a
  // share of the other instructions, and its operands are read from LDS two products of its kind ahead.
  constexpr int kSlots = kSteps + 2 * kColumns, kTops = kSlots / 4;
  eight k_piece[kSteps], v_piece[2 * kColumns];
  const int k_place = (lane & 31) * kPitch + 16 * (half ^ key_swap<DP>(lane & 31)), v_row = 4 * half + (lane & 15) / 4;
  const int v_place = v_row * kPitch + (32 * (lane >> 4 & 1) + (lane & 3) * 8 ^ 16 * value_swap<DP>(v_row));
  // lane l reads key l % 32 of the half, numbers 16 d + 8 (l / 32)
  auto read_keys = [&](const char* tiles, int h, int d) {
    k_piece[d] = *reinterpret_cast<const eight*>(tiles + 32 * h * kPitch + (k_place ^ 32 * d));
  };
  // lane l reads column l % 16 of v for four keys at a time: keys 16 t + 8 u + 4 (l / 32), columns 32 c + 16 (l / 16 % 2)
  auto read_values = [&](const char* tiles, int h, int n) {
    const int t = n / kColumns, c = n % kColumns;
    const char* from = tiles + (32 * h + 16 * t) * kPitch + (v_place ^ 64 * c);
    const short4_t a = turned(from), b = turned(from + 8 * kPitch);
    v_piece[n] = __builtin_bit_cast(eight, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
  };
  auto step = [&](int of_tile, auto half_of_tile, const char* k_from, const char* v_from) {
    constexpr int h = decltype(half_of_tile)::value;
    const int base = of_tile * kTile + 32 * h;
#pragma unroll
    for (int n = 0; n < 2; ++n) read_values(v_from, h ^ 1, n), read_keys(k_from, h ^ 1, n);
    const bool masked = base < wave_full_low || base + 32 > wave_full_high;
    uint32_t seen = ~0u;
    if (masked) seen = (uint32_t)(sight.of(base) >> 4 * half);
    if (SCORES == kSloped) {
      const float distance = (float)(sight.position - base - 4 * half);
      if (score.is_capped) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[h][i] = score.any_capped(s[h][i]);
      } else {
        s[h] *= score.by;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) s[h][i] = score.sloped(s[h][i], distance - (float)(8 * (i / 4) + i % 4));
    }
    if (SCORES != kCapped && masked) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[h][i] = shown(s[h][i], seen, 8 * (i / 4) + i % 4);
    }
    // The weights are formed with the maximum so far, as if the scores had not risen past it, and anew in the rare case that they have:
    // so nothing waits for the comparison.
    const float before = sum;
    float top = -kInfinity;
    auto weight = [&](int e, float less) {
      return __builtin_amdgcn_exp2f(SCORES == kPlain ? __builtin_fmaf(s[h][e], score.by, -less) : s[h][e] - less);
    };
    auto put = [&](int e, float one, float two) {
      auto both = E::pair(one, two);
      asm volatile("" : "+v"(both));   // (or the weights would be formed where they are used, behind the products)
      weights[h][e / 8][e % 8] = both[0], weights[h][e / 8][e % 8 + 1] = both[1];
      sum = E::add(both, sum);
    };
    const float less = most == -kInfinity ? 0.0f : most - E::kRaise;
    float last_weight = 0.0f;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      const int n = i / 2;
      if (i % 2 == 0) {
        if (n + 2 < kSteps) read_keys(k_from, h ^ 1, n + 2);
        s[h ^ 1] = E::mfma32(k_piece[n], q[n], n == 0 ? floatx16_t{} : s[h ^ 1]);
      } else {
        if (n + 2 < 2 * kColumns) read_values(v_from, h ^ 1, n + 2);
        out[n % kColumns] = E::mfma32(v_piece[n], weights[h ^ 1][n / kColumns], out[n % kColumns]);
      }
#pragma unroll
      for (int e = 16 * i / kSlots; e < 16 * (i + 1) / kSlots; ++e) {
        if (SCORES == kCapped) s[h][e] = shown(score.capped(s[h][e]), seen, 8 * (e / 4) + e % 4);
        const float w = weight(e, less);
        if (e % 2 == 1) {
          put(e - 1, last_weight, w);
          top = fmaxf(fmaxf(top, s[h][e - 1]), s[h][e]);
        }
        last_weight = w;
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (SCORES == kPlain) top *= score.by;
    if (__any(top > most + 8.0f)) {
      const float now = fmaxf(most, joined<true>(top, [](float a, float b) { return fmaxf(a, b); }));
      const float less = now == -kInfinity ? 0.0f : now - E::kRaise, by = now == -kInfinity ? 1.0f : __builtin_amdgcn_exp2f(most - now);
      most = now, sum = before * by;
#pragma unroll
      for (int c = 0; c < kColumns; ++c) out[c] *= by;
#pragma unroll
      for (int e = 0; e < 16; e += 2) put(e, weight(e, less), weight(e + 1, less));
    }
  };
  if (p.dim < DP) {   // what no copy reaches
    for (int i = threadIdx.x * 16; i < 4 * kTileBytes; i += WAVES * 64 * 16) *reinterpret_cast<u32x4_t*>(lds + i) = u32x4_t{};
    __syncthreads();
  }
  if (tile < last) {
    // the first tile's keys and values and the next one's keys, all on their way at once
    look_up(tile);
    const int first_page = page_ahead;
    look_up(tile + 1);
    const int second_page = page_ahead;
    look_up(tile + 2);
    const int third_page = page_ahead;
    page_ahead = first_page;
    find(tile);
    fetch_keys(k_lds);
    page_ahead = second_page;
    if constexpr (FP8) {
      spread(v_rows, places);
      fetch_values(v_lds);
#pragma unroll
      for (int i = 0; i < 2; ++i) weights[1][i] = eight{};
      if (has_k) {
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
          char* row = k_tiles + my_row_of_16 * kPitch + i * (WAVES * kGroup * kPitch);
          const int swap = key_swap<DP>(my_row_of_16);
          *reinterpret_cast<u32x4_t*>(row + 16 * (2 * k_chunk ^ swap)) = widen<T>(k_next[i][0], k_next[i][1]);
          *reinterpret_cast<u32x4_t*>(row + 16 * (2 * k_chunk + 1 ^ swap)) = widen<T>(k_next[i][2], k_next[i][3]);
        }
      }
      find(tile + 1);
      fetch_keys(k_lds + kTileBytes);
    } else {
      find(tile + 1);
      fetch_values(v_lds);
      fetch_keys(k_lds + kTileBytes);
#pragma unroll
      for (int i = 0; i < 2; ++i) weights[1][i] = eight{};
    }
    page_ahead = third_page;
    for (int i = threadIdx.x * 16; i < kTileBytes; i += WAVES * 64 * 16) *reinterpret_cast<u32x4_t*>(v_tiles + kTileBytes + i) = u32x4_t{};
    if constexpr (!FP8) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    s[0] = floatx16_t{};
#pragma unroll
    for (int d = 0; d < kSteps; ++d) {
      read_keys(k_tiles, 0, d);
      s[0] = E::mfma32(k_piece[d], q[d], s[0]);
    }
    int buffer = 0;
    for (; tile < last; ++tile, buffer ^= kTileBytes) {
      char *const k_here = k_tiles + buffer, *const v_here = v_tiles + buffer;
      char *const k_there = k_tiles + (buffer ^ kTileBytes), *const v_there = v_tiles + (buffer ^ kTileBytes);
      if (busy) step(tile, std::integral_constant<int, 0>{}, k_here, v_there);
      find(tile + 2);
      keep(k_there, v_here, tile * kTile < block_full_low || tile * kTile + kTile > block_full_high);
      __syncthreads();
      fetch_values(v_lds + (buffer ^ kTileBytes));
      fetch_keys(k_lds + buffer);
      look_up(tile + 3);
      if (busy) step(tile, std::integral_constant<int, 1>{}, k_there, v_here);
    }
#pragma unroll
    for (int n = 0; n < 2 * kColumns; ++n) {
      read_values(v_tiles + (buffer ^ kTileBytes), 1, n);
      out[n % kColumns] = E::mfma32(v_piece[n], weights[1][n / kColumns], out[n % kColumns]);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // (copies that nothing uses would land in LDS of another workgroup)
  }

  // ---- results
  __syncthreads();
  if (threadIdx.x == 0) flags[0] = 0;
  __syncthreads();
  if (bad) atomicOr(flags, 1);
  if (specials) atomicOr(flags, 2);
  __syncthreads();
  const int found = flags[0];
  sum = joined<true>(sum, [](float a, float b) { return a + b; });
  if (parts > 1) {
    if (row < r.rows) {
      const long at = part_at(p, r, split, kv_head, row);
      if (half == 0) p.part_ml[at] = make_float2(most, sum);
      float* to = p.part_o + at * p.dim + 4 * half;
#pragma unroll
      for (int c = 0; c < kColumns; ++c)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          if (32 * c + 2 * i < p.dim)
            *reinterpret_cast<floatx4_t*>(to + 32 * c + 2 * i) = floatx4_t{out[c][i], out[c][i + 1], out[c][i + 2], out[c][i + 3]};
    }
  } else {
    // through LDS, to leave as whole lines: a row's pieces of 16 bytes swapped by its number, as the tiles' are
    __syncthreads();
    char* const mine = lds + wave * 32 * kPitch;
    constexpr int kPieces = kPitch / 16, kSwap = kPieces < 16 ? kPieces - 1 : 15;
    const float by = row_scale(p, r, t, kv_head, sum);
#pragma unroll
    for (int c = 0; c < kColumns; ++c)
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *reinterpret_cast<Four<T>*>(mine + (lane & 31) * kPitch + ((4 * c + i / 4) ^ (lane & kSwap & 31)) * 16 + 8 * half) =
            four<T>(out[c][i] * by, out[c][i + 1] * by, out[c][i + 2] * by, out[c][i + 3] * by);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const long place = token * p.out_token + head * p.out_head;
    typedef uint32_t lines __attribute__((ext_vector_type(4), aligned(8)));
#pragma unroll
    for (int i = 0; i < 32 * kPieces / 64; ++i) {
      const int from = (i * 64 + lane) / kPieces, piece = (i * 64 + lane) % kPieces;
      const uint32_t low = __builtin_amdgcn_ds_bpermute(4 * from, (int)place), high = __builtin_amdgcn_ds_bpermute(4 * from, (int)(place >> 32));
      const lines x = *reinterpret_cast<const lines*>(mine + from * kPitch + (piece ^ (from & kSwap)) * 16);
      if (r.first + wave * 32 + from < r.rows && piece * 8 < p.dim)
        *reinterpret_cast<lines*>((T*)p.out + (long)((uint64_t)high << 32 | low) + piece * 8) = x;
    }
  }
  if (found & 2)
    add_specials<T, FP8>(p, r, kv_head, split, parts, first_tile, last, min(r.rows, r.first + kRows), block_full_low, block_full_high);
  if (found & 1) spoil_rows<T>(p, r, kv_head, split, parts, first_tile, last, min(r.rows, r.first + kRows));
}

// ---------------------------------------------------------------- few rows
// A workgroup takes 16 rows of a kv head, and its wavefronts take 32 keys in turn, each with a maximum, a sum and an output
// of its own, which are joined at the end.  Keys go from memory straight into the registers of the product, values through a piece
// of LDS that is the wavefront's own, to be turned there: no wavefront waits for another until the end.  Bound by memory where there is
// much to read (64 sequences of 800 to 4096 keys of 8-bit codes: 90 us, 3.7 TB/s; what widens them takes the rest), else by the trips to
// memory one after the other: lengths, page numbers, keys (one sequence of 700 keys: 7 us, and 4 the join; 9.7 both).  Two units'
// loads on their way at once, which cost a wavefront a SIMD, gave nothing (8000 keys 18.4 us for 17.2, heads of 64 55 for 53), nor did 8 wavefronts.
constexpr int kFew = 4;      // wavefronts of a workgroup
constexpr int kUnit = 32;    // keys that a wavefront takes at once

template <int DP>
constexpr int pitch() { return DP * 2 + 32; }   // bytes of a row there: 8 neighbouring rows start at banks of their own
template <int DP>
constexpr int few_lds() { return kFew * kUnit * pitch<DP>() + kFew * 16 * 8 + 16; }

constexpr int few_waves(int dp, bool fp8) { return dp == 64 ? 4 : dp == 128 ? 3 : fp8 ? 2 : 1; }   // a SIMD

template <typename T, int DP, bool FP8, int SCORES>
__global__ __launch_bounds__(kFew * 64, few_waves(DP, FP8)) void attention_few_kernel(const AttentionParams p) {
  typedef Element<T> E;
  typedef typename E::eight eight;
  constexpr int kSteps = DP / 32, kColumns = DP / 16, kPitch = pitch<DP>(), kLoads = FP8 ? DP / 64 : DP / 32;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int column = lane & 15, quarter = lane >> 4;
  char* const mine = lds + wave * kUnit * kPitch;
  float2* const sums = (float2*)(lds + kFew * kUnit * kPitch);   // [kFew][16]
  int* const flags = (int*)(sums + kFew * 16);

  int item, kv_head;
  item_of(p, p.blocks * p.splits, blockIdx.x, item, kv_head);
  const int split = item / p.blocks;
  const RowBlock r = row_block<16>(p, item % p.blocks);
  if (r.first < 0 || r.first >= r.rows || (r.seq == p.seqs && !p.clear_rest)) return;   // (negative where starts do not rise)
  const int block_t0 = r.first / p.group, block_t1 = min(r.first + 16 - 1, r.rows - 1) / p.group;
  int low, high;
  keys_seen(p, r, block_t0, block_t1, low, high);
  int first_tile = low / kTile, last_tile = high > low ? (high + kTile - 1) / kTile : low / kTile, parts;
  if (!split_of(p, r, split, first_tile, last_tile, parts)) return;
  const bool bounded = p.causal && p.tree == nullptr;
  const int full_low = bounded && p.window > 0 ? max(r.past + block_t1 - p.window + 1, 0) : 0;
  const int full_high = p.tree != nullptr ? min(r.len, r.past) : bounded ? min(r.len, r.past + block_t0 + 1) : r.len;

  const int my_row = min(r.first + column, r.rows - 1), t = my_row / p.group, head = kv_head * p.group + my_row % p.group;
  const long my_token = r.token + t;
  const Sight sight{r.past + t, r.len, r.past, bounded && p.window > 0 ? r.past + t - p.window + 1 : 0,
                    p.tree == nullptr ? nullptr : p.tree + my_token * p.tree_words, p.tree_words, p.causal};
  const Score score = score_of(p, kv_head, head);
  eight q[kSteps];
  {
    const T* from = (const T*)p.q + my_token * p.q_token + head * p.q_head;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {   // of an 8-bit cache a lane holds 16 neighbouring numbers of a key, for two steps
      const int d = FP8 ? 64 * (s / 2) + 16 * quarter + 8 * (s % 2) : 32 * s + 8 * quarter;
      q[s] = eight{};
      if (d < p.dim) q[s] = *reinterpret_cast<const eight*>(from + d);
    }
  }

  const char* const k_base = p.k.data + kv_head * p.k.head + 16 * quarter;
  const char* const v_base = p.v.data + kv_head * p.v.head + 16 * quarter;
  const int32_t* const pages = p.table + (long)min(r.seq, p.seqs - 1) * p.table_stride;
  bool bad = false;
  uint32_t specials = 0;
  u32x4_t k[2][kLoads], v[2][kLoads];   // keys 16 a + lane % 16
  int numbers[2];                       // of their pages, a unit ahead
  auto key_of = [&](int unit, int a) { return min(max(unit * kUnit + 16 * a + column, low), high - 1); };
  auto look_up = [&](int unit) {
#pragma unroll
    for (int a = 0; a < 2; ++a) numbers[a] = pages[page_of(p, key_of(unit, a))];
  };
  auto fetch = [&](int unit) {
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      const int key = key_of(unit, a), at = page_of(p, key);
      const char* k_from = row_at(k_base, place_of(p, p.k, key, at, numbers[a], bad));
      const char* v_from = row_at(v_base, place_of(p, p.v, key, at, numbers[a], bad));
#pragma unroll
      for (int s = 0; s < kLoads; ++s) {
        k[a][s] = v[a][s] = u32x4_t{};
        if ((FP8 ? 64 * s + 16 * quarter : 32 * s + 8 * quarter) < p.dim) {
          k[a][s] = *reinterpret_cast<const u32x4_t*>(k_from + 64 * s);
          v[a][s] = *reinterpret_cast<const u32x4_t*>(v_from + 64 * s);
        }
      }
    }
  };

  floatx4_t out[kColumns];
#pragma unroll
  for (int c = 0; c < kColumns; ++c) out[c] = floatx4_t{};
  float most = -kInfinity, sum = 0.0f;
  int unit = 2 * first_tile + wave;
  const int last = min(2 * last_tile, (high + kUnit - 1) / kUnit);
  if (unit < last) {
    look_up(unit);
    fetch(unit);
    if (unit + kFew < last) look_up(unit + kFew);
  }
  for (; unit < last; unit += kFew) {
    const int base = unit * kUnit;
    const bool masked = base < full_low || base + kUnit > full_high;
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int s = 0; s < kLoads; ++s) {
        char* to = mine + (16 * a + column) * kPitch + (FP8 ? 128 * s + 32 * quarter : 64 * s + 16 * quarter);
        u32x4_t v0 = v[a][s];
        if constexpr (FP8) {
          u32x4_t v1 = widen<T>(v0[2], v0[3]);
          v0 = widen<T>(v0[0], v0[1]);
          if (masked) v1 = finite_part<T>(v1, specials);
          *reinterpret_cast<u32x4_t*>(to + 16) = v1;
        }
        if (masked) v0 = finite_part<T>(v0, specials);
        *reinterpret_cast<u32x4_t*>(to) = v0;
      }
    // scores of 32 keys: lane l has those of query l % 16 with the keys 16 a + 4 (l / 16) + i
    floatx4_t s[2];
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      s[a] = floatx4_t{};
#pragma unroll
      for (int d = 0; d < kSteps; ++d) {
        u32x4_t piece;
        if constexpr (FP8) piece = d % 2 == 0 ? widen<T>(k[a][d / 2][0], k[a][d / 2][1]) : widen<T>(k[a][d / 2][2], k[a][d / 2][3]);
        else piece = k[a][d];
        s[a] = E::mfma16(__builtin_bit_cast(eight, piece), q[d], s[a]);
      }
    }
    if (unit + kFew < last) {
      fetch(unit + kFew);
      if (unit + 2 * kFew < last) look_up(unit + 2 * kFew);
    }
    eight weights;
    if (SCORES == kCapped) {
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i / 4][i % 4] = score.capped(s[i / 4][i % 4]);
    } else if (SCORES == kSloped && score.is_capped) {
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i / 4][i % 4] = score.any_capped(s[i / 4][i % 4]);
    } else if (SCORES == kSloped) {
#pragma unroll
      for (int a = 0; a < 2; ++a) s[a] *= score.by;
    }
    if (SCORES == kSloped) {
      const float distance = (float)(sight.position - base - 4 * quarter);
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i / 4][i % 4] = score.sloped(s[i / 4][i % 4], distance - (float)(16 * (i / 4) + i % 4));
    }
    if (masked) {
      const uint32_t seen = (uint32_t)(sight.of(base) >> 4 * quarter);
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i / 4][i % 4] = shown(s[i / 4][i % 4], seen, 16 * (i / 4) + i % 4);
    }
    float top = s[0][0];
#pragma unroll
    for (int i = 1; i < 8; ++i) top = fmaxf(top, s[i / 4][i % 4]);
    if (SCORES == kPlain) top *= score.by;
    if (__any(top > most + 8.0f)) {
      auto larger = [](float a, float b) { return fmaxf(a, b); };
      const float now = fmaxf(most, joined<true>(joined<false>(top, larger), larger));
      const float by = now == -kInfinity ? 1.0f : __builtin_amdgcn_exp2f(most - now);
      most = now, sum *= by;
#pragma unroll
      for (int c = 0; c < kColumns; ++c) out[c] *= by;
    }
    const float less = most == -kInfinity ? 0.0f : most - E::kRaise;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = s[i / 4][i % 4];
      const float w = __builtin_amdgcn_exp2f(SCORES == kPlain ? __builtin_fmaf(x, score.by, -less) : x - less);
      sum += w;
      weights[i] = (T)w;
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");   // (what other lanes wrote is read)
    __builtin_amdgcn_wave_barrier();
    // lane l reads column l % 16 of v for four keys at a time: keys 16 a + 4 (l / 16)
    const char* from = mine + (4 * quarter + column / 4) * kPitch + (column & 3) * 8;
#pragma unroll
    for (int c = 0; c < kColumns; ++c) {
      const short4_t a = turned(from + 32 * c), b = turned(from + 16 * kPitch + 32 * c);
      out[c] = E::mfma16(__builtin_bit_cast(eight, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7)), weights, out[c]);
    }
    __builtin_amdgcn_wave_barrier();
  }

  // ---- the wavefronts' results joined: a row's numbers 4 (DP + 4) bytes apart
  if (threadIdx.x == 0) flags[0] = 0;
  __syncthreads();
  if (bad) atomicOr(flags, 1);
  if (specials) atomicOr(flags, 2);
  constexpr int kOut = 4 * DP + 16;
  auto add = [](float a, float b) { return a + b; };
  sum = joined<true>(joined<false>(sum, add), add);
  if (quarter == 0) sums[wave * 16 + column] = make_float2(most, sum);
#pragma unroll
  for (int c = 0; c < kColumns; ++c) *reinterpret_cast<floatx4_t*>(mine + column * kOut + 64 * c + 16 * quarter) = out[c];
  __syncthreads();
  const int in_tile = threadIdx.x / 16, row = r.first + in_tile;
  if (row < r.rows) {
    const long token = r.token + row / p.group;
    const int head = kv_head * p.group + row % p.group;
    float all = -kInfinity, total = 0.0f, by[kFew];
#pragma unroll
    for (int w = 0; w < kFew; ++w) all = fmaxf(all, sums[w * 16 + in_tile].x);
    const float less = all == -kInfinity ? 0.0f : all;
#pragma unroll
    for (int w = 0; w < kFew; ++w) {
      by[w] = __builtin_amdgcn_exp2f(sums[w * 16 + in_tile].x - less);
      total = __builtin_fmaf(by[w], sums[w * 16 + in_tile].y, total);
    }
    const long at = ((long)split * p.tokens + token) * p.heads + head;
    if (parts > 1 && threadIdx.x % 16 == 0) p.part_ml[at] = make_float2(all, total);
    const float scale = row_scale(p, r, row / p.group, kv_head, total);
#pragma unroll
    for (int j = 0; j < DP / 64; ++j) {
      const int d = 64 * j + 4 * (threadIdx.x % 16);
      if (d >= p.dim) continue;
      floatx4_t o{};
#pragma unroll
      for (int w = 0; w < kFew; ++w) {
        const floatx4_t x = *reinterpret_cast<const floatx4_t*>(lds + w * kUnit * kPitch + in_tile * kOut + 4 * d);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(by[w], x[e], o[e]);
      }
      if (parts > 1) *reinterpret_cast<floatx4_t*>(p.part_o + at * p.dim + d) = o;
      else *reinterpret_cast<Four<T>*>((T*)p.out + token * p.out_token + head * p.out_head + d) =
          four<T>(o[0] * scale, o[1] * scale, o[2] * scale, o[3] * scale);
    }
  }
  if (flags[0] & 2)
    add_specials<T, FP8>(p, r, kv_head, split, parts, first_tile, last_tile, min(r.rows, r.first + 16), full_low, full_high);
  if (flags[0] & 1) spoil_rows<T>(p, r, kv_head, split, parts, first_tile, last_tile, min(r.rows, r.first + 16));
}

// ---------------------------------------------------------------- the parts of a split joined
// out = sum over the parts of 2^(m_i - m) o_i, divided by that of their sums, with a running maximum m for each group of lanes.  WAVES
// wavefronts a row (1: four rows a workgroup); LANES lanes hold a row's numbers, four each, so that a wavefront reads 64 / LANES
// parts at once.  The first parts are read before it is known how many there are: one trip to memory less.  Bound by those trips where
// rows are few (32 rows of 6 parts: 3 us), else by memory (24 sequences of up to 60 drafts, 32 heads in 2 parts: 48 MB, 15 us).
template <typename T, int LANES, int WAVES>
__global__ __launch_bounds__(WAVES == 1 ? 256 : WAVES * 64) void attention_join_kernel(const AttentionParams p) {
  constexpr int kAtOnce = 64 / LANES, kStep = WAVES * kAtOnce, kBatch = 4;
  __shared__ float4 numbers[WAVES][LANES];
  __shared__ float2 sums[WAVES];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), d = lane % LANES * 4;
  const long row = WAVES == 1 ? (long)blockIdx.x * 4 + wave : (long)blockIdx.x;
  const long step = p.tails > 0 ? (long)p.seqs * p.kv_heads * kTail : (long)p.tokens * p.heads;
  if (row >= step) return;
  float2 ml[kBatch];
  floatx4_t o[kBatch];
  auto load = [&](int first, int end) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int s = min(first + i * kStep, end - 1);
      ml[i] = p.part_ml[row + s * step];
      if (d < p.dim) o[i] = *reinterpret_cast<const floatx4_t*>(p.part_o + (row + s * step) * p.dim + d);
    }
  };
  int s = (WAVES == 1 ? 0 : wave * kAtOnce) + lane / LANES;
  load(s, p.splits);
  int token, head, kv_head;
  RowBlock r;
  if (p.tails > 0) {   // (most rows have no parts; the first one's place was read)
    kv_head = row / kTail % p.kv_heads, r = last_rows(p, row / kTail / p.kv_heads);
    const int in = r.first + row % kTail;
    if (!is_tail(r) || in >= r.rows) return;
    token = r.token + in / p.group, head = kv_head * p.group + in % p.group;
  } else {
    token = row / p.heads, head = row % p.heads, kv_head = head / p.group;
    r = sequence_of(p, token, [](int, int start) { return start; });
    if (r.seq == p.seqs || token < r.token) return;
    r.first = ((token - r.token) * p.group + head % p.group) / p.rows * p.rows;
  }
  int low, high;
  keys_seen(p, r, r.first / p.group, min(r.first + p.rows - 1, r.rows - 1) / p.group, low, high);
  int first = low / kTile, last = high > low ? (high + kTile - 1) / kTile : low / kTile, parts;
  split_of(p, r, 0, first, last, parts);
  if (parts <= 1) return;
  if (p.tails > 0) load(s, parts);
  float most = -kInfinity, sum = 0.0f;
  floatx4_t out{};
  // (to the powers of two of another maximum; both -infinity where there is nothing yet)
  auto shrink = [](float from, float to) { return to == -kInfinity ? 1.0f : __builtin_amdgcn_exp2f(from - to); };
  for (;;) {
    float top = most;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) top = s + i * kStep < parts ? fmaxf(top, ml[i].x) : top;
    const float by = shrink(most, top);
    most = top, sum *= by;
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] *= by;
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      if (s + i * kStep < parts) {
        const float w = shrink(ml[i].x, top);
        sum = __builtin_fmaf(w, ml[i].y, sum);
#pragma unroll
        for (int e = 0; e < 4; ++e) out[e] = __builtin_fmaf(w, o[i][e], out[e]);
      }
    s += kBatch * kStep;
    if (__all(s >= parts)) break;
    load(s, parts);
  }
  // the groups of lanes, then the wavefronts
  auto larger = [](float a, float b) { return fmaxf(a, b); };
  auto add = [](float a, float b) { return a + b; };
  float top = most;
  if (LANES <= 16) top = joined<false>(top, larger);
  if (LANES <= 32) top = joined<true>(top, larger);
  const float by = shrink(most, top);
  sum *= by;
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e] *= by;
  if (LANES <= 16) {
    sum = joined<false>(sum, add);
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = joined<false>(out[e], add);
  }
  if (LANES <= 32) {
    sum = joined<true>(sum, add);
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = joined<true>(out[e], add);
  }
  if (WAVES > 1) {
    if (lane < LANES) numbers[wave][lane] = make_float4(out[0], out[1], out[2], out[3]);
    if (lane == 0) sums[wave] = make_float2(top, sum);
    __syncthreads();
    if (wave != 0) return;
    most = -kInfinity;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) most = fmaxf(most, sums[w].x);
    out = floatx4_t{}, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float4 x = numbers[w][lane % LANES];
      const float by = shrink(sums[w].x, most);
      sum = __builtin_fmaf(by, sums[w].y, sum);
      out[0] = __builtin_fmaf(by, x.x, out[0]), out[1] = __builtin_fmaf(by, x.y, out[1]);
      out[2] = __builtin_fmaf(by, x.z, out[2]), out[3] = __builtin_fmaf(by, x.w, out[3]);
    }
  }
  if (lane >= LANES || d >= p.dim) return;
  const float scale = row_scale(p, r, token - r.token, kv_head, sum);
  *reinterpret_cast<Four<T>*>((T*)p.out + token * p.out_token + head * p.out_head + d) =
      four<T>(out[0] * scale, out[1] * scale, out[2] * scale, out[3] * scale);
}

// ---------------------------------------------------------------- the choice
// Whether there is a form of eight wavefronts and 256 rows: the widest heads have no registers for it, and the narrow ones gain nothing
// (8192 tokens of 32 heads of 64: 353 us, with 128 rows 344; of 128: 574 and 590).
constexpr bool eight_waves(int dp) { return dp == 128; }

// Bytes of scratch memory at most: a call must not fail for parts that it can do without, and a captured one holds them.  What more
// parts would be chosen for gains little by them: 64 sequences of 33 tokens with 131072 keys 10.0 ms with 7 parts and with 16; 512 of up to
// 17 tokens, one with 100000 keys, 2.11 ms with 3 and 2.03 with 4; 1024 of up to 17 in heads of 256 4.2 ms with none and 4.8 with 4.
constexpr int64_t kMostScratch = 256 << 20;

struct Plan {
  int rows;   // of a block: 16 in the form for few rows, 128 and 256 in that for many
  long blocks, splits, split_tiles, tails;
  int longest, queries;
  float few_share;
  PartsCost cost;
  size_t ml_bytes, o_bytes;
};

Plan plan_of(int64_t tokens, int64_t seqs, int64_t heads, int64_t kv_heads, int64_t head_dim, bool fp8, int64_t max_seq_len, int64_t window) {
  Plan plan{};
  const int64_t group = heads / kv_heads, queries = (tokens + seqs - 1) / std::max<int64_t>(seqs, 1);
  const int64_t keys = std::max<int64_t>(window > 0 ? std::min(max_seq_len, window + queries) : max_seq_len, 1), longest = (keys + kTile - 1) / kTile;
  const int dp = head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256;
  plan.longest = (int)keys;
  const int64_t row_bytes = head_dim * (int64_t)sizeof(float) + (int64_t)sizeof(float2);
  auto parts_of = [&](int64_t rows) { return std::max<int64_t>((kMostScratch - 16) / (rows * row_bytes), 1); };   // at most
  auto groups_of = [&](int rows) {
    return std::max<int64_t>((tokens * group + rows - 1) / rows, std::min(seqs, tokens)) * kv_heads;
  };
  // Few rows a sequence: the form for many, whose copies are further ahead, once there is much to read, and of 16-bit numbers in
  // heads of more than 64 (64 sequences of 800 to 4096 keys, 4 rows each: 142 us, the form for few 154; of 8-bit codes 104 and 89, in
  // heads of 64 50 and 52; one sequence of 700 keys 10.4 and 9.3, of 8000 18.5 and 17.1).  From two rounds of workgroups on blocks of
  // 256 rows: two pieces of 2048 tokens behind 6144 others 488 us, with 128 rows 510; 33 sequences of up to 500 tokens, one round, 212
  // and 177.
  const bool few = queries * group <= 16 && (fp8 || dp == 64 || groups_of(16) * longest < 2048);
  plan.rows = few ? 16 : eight_waves(dp) && tokens * heads / 256 >= 512 ? 256 : 128;
  plan.blocks = tokens * group / plan.rows + seqs + 1;
  const int64_t groups = groups_of(plan.rows);
  if (few) {
    // Workgroups that find no part for them cost a trip to memory each, and the lengths may be far below what they might be: no more
    // than 256 parts, and of more than 4 no more than make 4096 workgroups.
    plan.few_share = (float)groups / 4096.0f;
    plan.split_tiles = 2;
    plan.splits = std::min<int64_t>(std::max<int64_t>(4096 / groups, 4), 256);
    plan.splits = std::min<int64_t>(plan.splits, (longest + few_tiles((int)longest, plan.few_share) - 1) / few_tiles((int)longest, plan.few_share));
    plan.splits = std::min(plan.splits, parts_of(tokens * heads));
  } else {
    // (for a tile: alone, and as many workgroups as a compute unit holds together)
    plan.cost = dp == 256 || plan.rows == 256 ? PartsCost{0, 1, dp == 256 ? 2.6f : 2.2f, 0.0f, 0.0f, 0.0f}
                : dp == 64                    ? PartsCost{0, 3, 1.3f, 0.9f, 1.1f, 0.0f}
                                              : PartsCost{0, 2, 2.1f, queries * group > 64 ? 1.9f : 1.35f, 0.0f, 0.0f};
    plan.cost.groups = (int)std::min<int64_t>(groups, 1 << 24);
    plan.cost.part = 0.3f + (float)(8.0 * (double)(tokens * heads * head_dim) / 4e6);
    plan.queries = (int)queries;
    const int tiles = mean_tiles((int)keys, plan.queries), most = (int)std::min<int64_t>({parts_of(tokens * heads), 64, tiles});
    float best = plan.cost.of(tiles, 1);
    plan.splits = 1;
    for (int n = 2; n <= most; ++n)
      if (plan.cost.of(tiles, n) < kWorth * best) best = plan.cost.of(tiles, n), plan.splits = n;
    plan.split_tiles = std::min<int64_t>((longest + plan.splits - 1) / plan.splits, 4);
  }
  if (tokens * heads >= 1LL << 24 || plan.blocks * kv_heads * plan.splits >= 1LL << 24) plan.splits = 1;   // (2^32 threads are a launch's most)
  // Many rows, but not of each sequence: single tokens beside prompts.  Their keys are split, though the rest has workgroups enough, as
  // a workgroup for all of them would end long after the others (one token with 100000 keys beside 16 prompts of 1000: 1816 us, so
  // 392; parts of 4 tiles at least: 9 sequences with a window of 1024 92 us, 2 tiles 95, 8 101, unsplit 108).
  // Not in batches of single tokens alone: 63 sequences of up to 4096 keys and one of 100000 take 1904 us so, 668 with such parts, but 64 of up
  // to 1000 that might have had 131072 34 and 55.
  if (!few && plan.splits == 1 && seqs > 1 && queries * group > kTail && 2 * queries < max_seq_len && seqs * kv_heads <= 8192)
    plan.tails = std::min({std::max<int64_t>(2048 / (seqs * kv_heads), 4), (longest + 3) / 4, parts_of(seqs * kv_heads * kTail)});
  if (plan.tails < 2) plan.tails = 0;
  if (plan.splits > 1 || plan.tails > 0) {
    const int64_t rows = plan.tails > 0 ? plan.tails * seqs * kv_heads * kTail : plan.splits * tokens * heads;
    plan.ml_bytes = (size_t)rows * sizeof(float2);
    plan.ml_bytes = (plan.ml_bytes + 15) / 16 * 16;
    plan.o_bytes = (size_t)(rows * head_dim) * sizeof(float);
  }
  return plan;
}

template <typename T, int DP>
int launch_join(const AttentionParams& p, hipStream_t st) {
  if (p.splits == 1 && p.tails == 0) return SONAR_OK;
  const long rows = p.tails > 0 ? (long)p.seqs * p.kv_heads * kTail : (long)p.tokens * p.heads;
  // (a workgroup a row where parts are many and rows few: one sequence of 8000 keys 18 us, a wavefront a row 24)
  if (p.splits > 8 && rows <= 256) attention_join_kernel<T, DP / 4, 8><<<(uint32_t)rows, 512, 0, st>>>(p);
  else attention_join_kernel<T, DP / 4, 1><<<(uint32_t)((rows + 3) / 4), 256, 0, st>>>(p);
  return launch_status("attention_join_kernel");
}

template <typename K>
int launch_one(K kernel, const AttentionParams& p, int waves, int lds, const char* name, hipStream_t st) {
  if (lds > 65536) SONAR_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
  kernel<<<(uint32_t)(p.blocks * p.kv_heads * p.splits + std::max(p.tails - 1, 0) * p.seqs * p.kv_heads), waves * 64, lds, st>>>(p);
  return launch_status(name);
}

template <typename T, int DP, bool FP8, int SCORES>
int launch_form(const AttentionParams& p, hipStream_t st) {
  int rc;
  if (p.rows == 16) rc = launch_one(attention_few_kernel<T, DP, FP8, SCORES>, p, kFew, few_lds<DP>(), "attention_few_kernel", st);
  else if (p.rows == 128) rc = launch_one(attention_rows_kernel<T, DP, FP8, SCORES, 4>, p, 4, rows_lds<DP>(), "attention_rows_kernel", st);
  else if constexpr (eight_waves(DP)) rc = launch_one(attention_rows_kernel<T, DP, FP8, SCORES, 8>, p, 8, rows_lds<DP>(), "attention_rows_kernel", st);
  else return fail(SONAR_E_INVALID, "no form of %d rows", p.rows);
  return rc != SONAR_OK ? rc : launch_join<T, DP>(p, st);
}

template <typename T, int DP, bool FP8>
int launch_scores(const AttentionParams& p, hipStream_t st) {
  // (a cap of at most 128 is off by 2^-15 in the shorter form, much less than a weight's own rounding)
  if (p.slopes != nullptr || p.cap > 128.0f) return launch_form<T, DP, FP8, kSloped>(p, st);
  return p.cap > 0.0f ? launch_form<T, DP, FP8, kCapped>(p, st) : launch_form<T, DP, FP8, kPlain>(p, st);
}

template <typename T, int DP>
int launch_width(const AttentionParams& p, bool fp8, hipStream_t st) {
  return fp8 ? launch_scores<T, DP, true>(p, st) : launch_scores<T, DP, false>(p, st);
}

template <typename T>
int launch(const AttentionParams& p, bool fp8, hipStream_t st) {
  if (p.dim <= 64) return launch_width<T, 64>(p, fp8, st);
  if (p.dim <= 128) return launch_width<T, 128>(p, fp8, st);
  return launch_width<T, 256>(p, fp8, st);
}

int check_sizes(int64_t tokens, int64_t seqs, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t max_seq_len, int64_t window) {
  SONAR_REQUIRE(heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0, "heads = %ld is no multiple of kv_heads = %ld", (long)heads, (long)kv_heads);
  SONAR_REQUIRE(head_dim >= 16 && head_dim <= 256 && head_dim % 16 == 0, "head_dim = %ld must be a multiple of 16, at most 256", (long)head_dim);
  SONAR_REQUIRE(tokens >= 0 && heads < (1LL << 31) && tokens < (1LL << 31) && tokens * heads < (1LL << 31), "tokens = %ld of %ld heads: too many",
                (long)tokens, (long)heads);
  SONAR_REQUIRE(seqs >= 0 && seqs < (1LL << 30), "seqs = %ld", (long)seqs);
  SONAR_REQUIRE(max_seq_len >= 0 && max_seq_len < (1LL << 31), "max_seq_len = %ld", (long)max_seq_len);
  SONAR_REQUIRE(window >= 0 && window < (1LL << 31), "window = %ld", (long)window);
  return SONAR_OK;
}

}  // namespace
}  // namespace sonar

using namespace sonar;

extern "C" size_t sonar_paged_attention_scratch_bytes(int64_t tokens, int64_t seqs, int64_t heads, int64_t kv_heads,
                                                      int64_t head_dim, int cache_dtype, int64_t max_seq_len, int64_t window) {
  if (check_sizes(tokens, seqs, heads, kv_heads, head_dim, max_seq_len, window) != SONAR_OK || tokens == 0 || seqs == 0) return 0;
  const Plan plan = plan_of(tokens, seqs, heads, kv_heads, head_dim, cache_dtype == SONAR_CACHE_FP8, max_seq_len, window);
  return plan.ml_bytes + plan.o_bytes;
}

extern "C" int sonar_paged_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, const sonar_kv_cache* key_cache,
                                     const sonar_kv_cache* value_cache, int cache_dtype, int64_t pages, int64_t page_size,
                                     const int32_t* block_table, int64_t table_stride, int64_t table_pages, const int32_t* seq_lens,
                                     const int32_t* starts, void* out, int64_t out_token_stride, int64_t out_head_stride,
                                     int clear_rest, double scale, double cap, int64_t window, int causal, const float* slopes,
                                     const int64_t* tree_mask, int64_t tree_words, void* scratch, size_t scratch_bytes, int dtype,
                                     int64_t tokens, int64_t seqs, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                     int64_t max_seq_len, void* stream) {
  if (int rc = check_sizes(tokens, seqs, heads, kv_heads, head_dim, max_seq_len, window)) return rc;
  SONAR_REQUIRE(dtype == SONAR_DTYPE_F16 || dtype == SONAR_DTYPE_BF16, "dtype = %d must be float16 or bfloat16", dtype);
  SONAR_REQUIRE(cache_dtype == dtype || cache_dtype == SONAR_CACHE_FP8, "cache_dtype = %d does not go with dtype = %d", cache_dtype, dtype);
  SONAR_REQUIRE(key_cache && value_cache, "key_cache and value_cache must not be NULL");
  SONAR_REQUIRE(page_size >= 1 && pages >= 0 && pages < (1LL << 31) && table_pages >= 0 && page_size < (1LL << 31) &&
                    table_pages < (1LL << 31) && table_pages * page_size < (1LL << 31) - 1024,
                "pages = %ld of %ld slots, %ld a sequence", (long)pages, (long)page_size, (long)table_pages);
  SONAR_REQUIRE(scale >= 1e-30 && scale <= 1e30, "scale = %g must be positive, from 1e-30 to 1e30", scale);
  SONAR_REQUIRE(cap == 0.0 || (cap >= 1e-30 && cap <= 1e30), "cap = %g must be 0 (none) or positive, from 1e-30 to 1e30", cap);
  SONAR_REQUIRE(tree_mask == nullptr || (tree_words >= 1 && tree_words < (1 << 20)), "tree_words = %ld", (long)tree_words);
  SONAR_REQUIRE(tree_mask == nullptr || (window == 0 && slopes == nullptr), "a tree mask goes with neither a window nor slopes");
  SONAR_REQUIRE(window == 0 || causal, "a window goes with causal attention only");
  const int64_t cache_size = cache_dtype == SONAR_CACHE_FP8 ? 1 : 2, unit = 16 / cache_size;
  for (const sonar_kv_cache* c : {key_cache, value_cache}) {
    SONAR_REQUIRE(c->page_stride % unit == 0 && c->slot_stride % unit == 0 && c->head_stride % unit == 0 && (uintptr_t)c->data % 16 == 0,
                  "a cache must be 16-byte aligned, with strides of multiples of 16 bytes; got %ld, %ld, %ld elements", (long)c->page_stride,
                  (long)c->slot_stride, (long)c->head_stride);
    SONAR_REQUIRE(c->slot_stride >= 0 && c->page_stride >= 0 && c->slot_stride < (1LL << 36) / page_size && c->page_stride < (1LL << 37) / (pages + 1) &&
                      ((pages - 1) * c->page_stride + (page_size - 1) * c->slot_stride) * cache_size < (1LL << 36),
                  "a cache of %ld pages %ld elements apart: more than 64 GiB", (long)pages, (long)c->page_stride);
    SONAR_REQUIRE(cache_dtype != SONAR_CACHE_FP8 || (c->scale != nullptr && (c->scale_len == 1 || c->scale_len == kv_heads)),
                  "an 8-bit cache needs 1 or %ld scales; got %ld", (long)kv_heads, c->scale == nullptr ? 0L : (long)c->scale_len);
  }
  SONAR_REQUIRE(q_token_stride % 8 == 0 && q_head_stride % 8 == 0 && (uintptr_t)q % 16 == 0, "q must be 16-byte aligned, its strides multiples of 8");
  SONAR_REQUIRE(out_token_stride % 4 == 0 && out_head_stride % 4 == 0 && (uintptr_t)out % 8 == 0, "out must be 8-byte aligned, its strides multiples of 4");
  if (tokens == 0) return SONAR_OK;
  SONAR_REQUIRE(q && out && starts, "q, out and starts must not be NULL");
  SONAR_REQUIRE(seqs >= 1, "tokens without sequences: seqs = 0");
  SONAR_REQUIRE(seq_lens && (table_pages == 0 || (block_table && table_stride >= table_pages && pages >= 1 && key_cache->data && value_cache->data)),
                "seq_lens, a block_table of %ld pages a row and caches with pages are needed", (long)table_pages);
  Plan plan = plan_of(tokens, seqs, heads, kv_heads, head_dim, cache_dtype == SONAR_CACHE_FP8, max_seq_len, window);
  if (scratch_bytes < plan.ml_bytes + plan.o_bytes || scratch == nullptr) plan.splits = 1, plan.tails = 0;
  SONAR_REQUIRE((uintptr_t)scratch % 16 == 0, "scratch must be 16-byte aligned");
  SONAR_REQUIRE(plan.blocks * kv_heads * plan.splits < (1LL << 24),
                "%ld tokens of %ld sequences and %ld heads take too many workgroups", (long)tokens, (long)seqs, (long)heads);
  auto pages_of = [&](const sonar_kv_cache* c) {
    const bool fp8 = cache_dtype == SONAR_CACHE_FP8;
    return CachePages{(const char*)c->data, (uint32_t)(c->page_stride * cache_size / 16), (uint32_t)(c->slot_stride * cache_size / 16),
                      c->head_stride * cache_size, fp8 ? c->scale : nullptr, c->scale_len > 1};
  };
  AttentionParams p{};
  p.q = (const char*)q, p.q_token = q_token_stride, p.q_head = q_head_stride;
  p.k = pages_of(key_cache), p.v = pages_of(value_cache);
  p.table = block_table, p.table_stride = table_stride, p.lens = seq_lens, p.starts = starts;
  p.out = (char*)out, p.out_token = out_token_stride, p.out_head = out_head_stride;
  p.slopes = slopes, p.tree = (const uint64_t*)tree_mask, p.tree_words = (int)tree_words;
  p.part_ml = (float2*)scratch, p.part_o = (float*)((char*)scratch + plan.ml_bytes);
  p.scale = (float)scale, p.cap = (float)cap, p.window = window < table_pages * page_size ? (int)window : 0, p.causal = causal != 0, p.clear_rest = clear_rest != 0;
  int log = 0;
  while ((1LL << log) < page_size) ++log;
  p.page_shift = 31 + log, p.page_magic = (uint32_t)((1ULL << p.page_shift) / (uint64_t)page_size + 1);
  p.page_size = (int)page_size, p.pages = (int)pages, p.table_pages = (int)table_pages;
  p.tokens = (int)tokens, p.seqs = (int)seqs, p.heads = (int)heads, p.kv_heads = (int)kv_heads, p.group = (int)(heads / kv_heads);
  p.dim = (int)head_dim, p.rows = plan.rows, p.blocks = (int)plan.blocks, p.splits = (int)plan.splits, p.split_tiles = (int)plan.split_tiles, p.tails = (int)plan.tails, p.longest = plan.longest, p.few_share = plan.few_share;
  p.queries = plan.queries, p.cost = plan.cost;
  p.by_dies = plan.rows == 16;
  const bool fp8 = cache_dtype == SONAR_CACHE_FP8;
  hipStream_t st = (hipStream_t)stream;
  return dtype == SONAR_DTYPE_F16 ? launch<_Float16>(p, fp8, st) : launch<__bf16>(p, fp8, st);
}
