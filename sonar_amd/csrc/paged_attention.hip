// Attention of a ragged batch over a paged cache: out = softmax(cap(scale * q k^T) - bias, what is masked left out) v.
//
// One pass over the keys with a running maximum m and sum l: a tile's scores s give p = 2^(s log2 e - m), out = out + p v,
// l = l + sum p, and where a score is above m by more than 8 (in powers of two) m rises to it, out and l shrinking with it.
// (Rising only then leaves p up to 2^8, which p's type and the sums hold as precisely.)  Products on the matrix
// instructions, sums in fp32; p is rounded to the type of v for its product, by at most half a step of each.
//
// Both products are formed turned, k q^T and v^T p^T: a lane then holds scores of one query only, so that m, l and what
// out shrinks by are a lane's own numbers, and the scores lie where the second product takes them as its operand.  The keys of
// that product are in the order in which they fell there; v is read from LDS turned, four keys at a time, in the same order.
#include <algorithm>

#include "paged_attention.hpp"

namespace sonar {
char* last_error_buffer();
namespace {

constexpr int kTile = 64;   // keys

// What turns a score q . k into a power of two, for the forms with a cap or slopes.
struct Score {
  float by, cap, slope;   // plain: s * by; capped: cap * tanh of it
  bool capped;
  __device__ __forceinline__ float of(float s, float distance) const {
    if (capped) s = cap - 2.0f * cap * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(s * by));
    else s *= by;
    return __builtin_fmaf(-slope, fabsf(distance), s);
  }
};

__device__ __forceinline__ Score score_of(const AttentionParams& p, int kv_head, int head) {
  const float k_scale = p.k.scale == nullptr ? 1.0f : p.k.scale[p.k.scale_heads ? kv_head : 0];
  Score s;
  s.capped = p.cap > 0.0f;
  s.by = s.capped ? 2.0f * kLog2E * p.scale * k_scale / p.cap : p.scale * k_scale * kLog2E;
  s.cap = p.cap * kLog2E;
  s.slope = p.slopes == nullptr ? 0.0f : p.slopes[head] * kLog2E;
  return s;
}

__device__ __forceinline__ float value_scale(const AttentionParams& p, int kv_head) {
  return p.v.scale == nullptr ? 1.0f : p.v.scale[p.v.scale_heads ? kv_head : 0];
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
        const long page = p.table[(long)r.seq * p.table_stride + at];
        if (page < 0 || page >= p.pages) continue;
        const char* from = p.v.data + page * p.v.page + (key - at * p.page_size) * p.v.slot + kv_head * p.v.head;
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
            p.part_o[(((long)split * p.tokens + token) * p.heads + head) * p.dim + d] += v;
          } else {
            T* to = (T*)p.out + token * p.out_token + head * p.out_head + d;
            *to = (T)((float)*to + v);
          }
        }
      }
    }
}

// ---------------------------------------------------------------- many rows
// A workgroup takes 128 rows of a kv head, 32 a wavefront, and walks the keys in tiles of 64 that its wavefronts share through
// LDS, two tiles there: while one is worked on, the next one's numbers are on their way in registers.
constexpr int kWaves = 4, kRows = 32 * kWaves;

template <int DP>
constexpr int pitch() { return DP * 2 + 32; }   // bytes of a row of a tile in LDS: 8 neighbouring rows start at banks of their own
template <int DP>
constexpr int tile_bytes() { return kTile * pitch<DP>(); }
template <int DP>
constexpr int rows_lds() { return 4 * tile_bytes<DP>() + 16; }

template <typename T, int DP, bool FP8, bool EXTRA>
__global__ __launch_bounds__(kWaves * 64, DP <= 128 ? 2 : 1) void attention_rows_kernel(const AttentionParams p) {
  typedef Element<T> E;
  typedef typename E::eight eight;
  constexpr int kSteps = DP / 16, kColumns = DP / 32, kPitch = pitch<DP>(), kTileBytes = tile_bytes<DP>();
  constexpr int kLanes = FP8 ? DP / 16 : DP / 8;             // of a row, 16 bytes each
  constexpr int kGroup = 64 / kLanes;                        // rows that a wavefront copies at once
  constexpr int kPasses = kTile / (kWaves * kGroup);
  extern __shared__ __attribute__((aligned(16))) char lds[];
  char* const k_tiles = lds;
  char* const v_tiles = lds + 2 * kTileBytes;
  int* const flags = (int*)(lds + 4 * kTileBytes);

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kv_head = blockIdx.x % p.kv_heads, split = blockIdx.x / p.kv_heads / p.blocks;
  // the blocks of the last tokens, which see the most keys, first
  const RowBlock r = row_block<kRows>(p, p.blocks - 1 - blockIdx.x / p.kv_heads % p.blocks);
  if (r.first >= r.rows || (r.seq == p.seqs && !p.clear_rest)) return;

  const int row = r.first + wave * 32 + (lane & 31), half = lane >> 5;
  const int my_row = min(row, r.rows - 1), t = my_row / p.group, head = kv_head * p.group + my_row % p.group;
  const long token = r.token + t;
  const int wave_t0 = min(r.first + wave * 32, r.rows - 1) / p.group, wave_t1 = min(r.first + wave * 32 + 31, r.rows - 1) / p.group;
  const int block_t0 = r.first / p.group, block_t1 = min(r.first + kRows - 1, r.rows - 1) / p.group;
  int low, high, wave_low, wave_high;
  keys_seen(p, r, block_t0, block_t1, low, high);
  keys_seen(p, r, wave_t0, wave_t1, wave_low, wave_high);
  int tile = low / kTile, last = high > low ? (high + kTile - 1) / kTile : low / kTile, parts;
  if (!split_of(p, split, tile, last, parts)) return;
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

  // ---- copies of the tiles
  u32x4_t k_next[kPasses], v_next[kPasses];
  bool bad = false;
  const int chunk = lane % kLanes, of_group = lane / kLanes;
  const bool has_chunk = chunk * (FP8 ? 16 : 8) < p.dim, whole_groups = p.page_size % kGroup == 0;
  const char* const k_base = p.k.data + kv_head * p.k.head;
  const char* const v_base = p.v.data + kv_head * p.v.head;
  const int32_t* const pages = p.table + (long)min(r.seq, p.seqs - 1) * p.table_stride;
  auto fetch = [&](int of_tile) {
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int first = of_tile * kTile + (i * kWaves + wave) * kGroup;
      k_next[i] = v_next[i] = u32x4_t{};
      if (whole_groups) {   // the rows of a group lie in one page: its address is the wavefront's
        const int key = min(max(first, low & -kGroup), (high - 1) & -kGroup), at = page_of(p, key);
        const long page = page_number(p, pages[at], bad);
        const int slot = key - at * p.page_size;
        const uint32_t k_lane = of_group * (uint32_t)p.k.slot + chunk * 16, v_lane = of_group * (uint32_t)p.v.slot + chunk * 16;
        const char* k_from = k_base + page * p.k.page + slot * p.k.slot;
        const char* v_from = v_base + page * p.v.page + slot * p.v.slot;
        if (has_chunk) {
          k_next[i] = *reinterpret_cast<const u32x4_t*>(k_from + k_lane);
          v_next[i] = *reinterpret_cast<const u32x4_t*>(v_from + v_lane);
        }
      } else {
        const int key = min(max(first + of_group, low), high - 1), at = page_of(p, key);
        const long page = page_number(p, pages[at], bad), slot = key - at * p.page_size;
        if (has_chunk) {
          k_next[i] = *reinterpret_cast<const u32x4_t*>(k_base + page * p.k.page + slot * p.k.slot + chunk * 16);
          v_next[i] = *reinterpret_cast<const u32x4_t*>(v_base + page * p.v.page + slot * p.v.slot + chunk * 16);
        }
      }
    }
  };
  bool specials = false;   // infinities and NaNs of v were left out of a tile that is masked for some query
  auto keep = [&](int of_tile, int buffer) {
    const bool masked = of_tile * kTile < block_full_low || of_tile * kTile + kTile > block_full_high;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int at = buffer * kTileBytes + ((i * kWaves + wave) * kGroup + of_group) * kPitch + chunk * (FP8 ? 32 : 16);
      u32x4_t k0 = k_next[i], v0 = v_next[i];
      if constexpr (FP8) {
        const u32x4_t k1 = widen<T>(k0[2], k0[3]);
        u32x4_t v1 = widen<T>(v0[2], v0[3]);
        k0 = widen<T>(k0[0], k0[1]), v0 = widen<T>(v0[0], v0[1]);
        if (masked) v1 = finite_part<T>(v1, specials);
        *reinterpret_cast<u32x4_t*>(k_tiles + at + 16) = k1;
        *reinterpret_cast<u32x4_t*>(v_tiles + at + 16) = v1;
      }
      if (masked) v0 = finite_part<T>(v0, specials);
      *reinterpret_cast<u32x4_t*>(k_tiles + at) = k0;
      *reinterpret_cast<u32x4_t*>(v_tiles + at) = v0;
    }
  };

  floatx16_t out[kColumns];
#pragma unroll
  for (int c = 0; c < kColumns; ++c) out[c] = floatx16_t{};
  float most = -kInfinity, sum = 0.0f;

  if (tile < last) {
    fetch(tile);
    keep(tile, 0);
  }
  __syncthreads();
  for (int buffer = 0; tile < last; ++tile, buffer ^= 1) {
    if (tile + 1 < last) fetch(tile + 1);
    const int base = tile * kTile;
    if (base < wave_high && base + kTile > wave_low) {
      const bool masked = base < wave_full_low || base + kTile > wave_full_high;
      // scores of 64 keys: lane l has those of query l % 32 with the keys 32 u + 8 (i / 4) + 4 (l / 32) + i % 4
      floatx16_t s[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        s[u] = floatx16_t{};
        const char* from = k_tiles + buffer * kTileBytes + (32 * u + (lane & 31)) * kPitch + 16 * half;
#pragma unroll
        for (int d = 0; d < kSteps; ++d) s[u] = E::mfma32(*reinterpret_cast<const eight*>(from + 32 * d), q[d], s[u]);
      }
      if (EXTRA) {
        const float distance = (float)(sight.position - base - 4 * half);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 16; ++i) s[u][i] = score.of(s[u][i], distance - (float)(32 * u + 8 * (i / 4) + i % 4));
      }
      if (masked) {
        const uint64_t bits = sight.of(base) >> 4 * half;
        const uint32_t seen[2] = {(uint32_t)bits, (uint32_t)(bits >> 32)};
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 16; ++i) s[u][i] = seen[u] & (1u << (8 * (i / 4) + i % 4)) ? s[u][i] : -kInfinity;
      }
      float top = s[0][0];
#pragma unroll
      for (int i = 1; i < 32; ++i) top = fmaxf(top, s[i / 16][i % 16]);
      top = joined<true>(top, [](float a, float b) { return fmaxf(a, b); });
      if (!EXTRA) top *= score.by;
      if (__any(top > most + 8.0f)) {
        const float now = fmaxf(most, top), by = now == -kInfinity ? 1.0f : __builtin_amdgcn_exp2f(most - now);
        most = now, sum *= by;
#pragma unroll
        for (int c = 0; c < kColumns; ++c) out[c] *= by;
      }
      const float less = most == -kInfinity ? 0.0f : most;
      eight weights[4];
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const float x = s[i / 16][i % 16];
        const float w = __builtin_amdgcn_exp2f(EXTRA ? x - less : __builtin_fmaf(x, score.by, -less));
        sum += w;
        weights[i / 8][i % 8] = (T)w;
      }
      // lane l reads column l % 16 of v for four keys at a time: keys 16 t + 8 u + 4 (l / 32), columns 32 c + 16 (l / 16 % 2)
      const char* from = v_tiles + buffer * kTileBytes + (4 * half + (lane & 15) / 4) * kPitch + 32 * (lane >> 4 & 1) + (lane & 3) * 8;
      auto column = [&](int c, int t) {
        const short4_t a = turned(from + 16 * t * kPitch + 64 * c), b = turned(from + (16 * t + 8) * kPitch + 64 * c);
        return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
      };
#pragma unroll
      for (int c = 0; c < kColumns; ++c)
#pragma unroll
        for (int t = 0; t < 4; ++t) out[c] = E::mfma32(__builtin_bit_cast(eight, column(c, t)), weights[t], out[c]);
    }
    if (tile + 1 < last) keep(tile + 1, buffer ^ 1);
    __syncthreads();
  }

  // ---- results
  if (threadIdx.x == 0) flags[0] = 0;
  __syncthreads();
  if (bad) atomicOr(flags, 1);
  if (specials) atomicOr(flags, 2);
  __syncthreads();
  const int found = flags[0];
  sum = joined<true>(sum, [](float a, float b) { return a + b; });
  if (found & 1) sum = __builtin_nanf("");
  if (parts > 1) {
    if (row < r.rows) {
      const long at = ((long)split * p.tokens + token) * p.heads + head;
      if (half == 0) p.part_ml[at] = make_float2(most, sum);
      float* to = p.part_o + at * p.dim + 4 * half;
#pragma unroll
      for (int c = 0; c < kColumns; ++c)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          if (32 * c + 2 * i < p.dim)
            *reinterpret_cast<floatx4_t*>(to + 32 * c + 2 * i) = floatx4_t{out[c][i], out[c][i + 1], out[c][i + 2], out[c][i + 3]};
    }
  } else if (row < r.rows) {
    const float by = sum == 0.0f ? 0.0f : value_scale(p, kv_head) / sum;
    T* to = (T*)p.out + token * p.out_token + head * p.out_head + 4 * half;
#pragma unroll
    for (int c = 0; c < kColumns; ++c)
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        if (32 * c + 2 * i < p.dim)
          *reinterpret_cast<Four<T>*>(to + 32 * c + 2 * i) = four<T>(out[c][i] * by, out[c][i + 1] * by, out[c][i + 2] * by, out[c][i + 3] * by);
  }
  if (found & 2)
    add_specials<T, FP8>(p, r, kv_head, split, parts, first_tile, last, min(r.rows, r.first + kRows), block_full_low, block_full_high);
}

// ---------------------------------------------------------------- the parts of a split joined
// A wavefront a row: out = sum over the parts of 2^(m_i - m) o_i, divided by that of their sums.
template <typename T, int ROWS>
__global__ __launch_bounds__(256) void attention_join_kernel(const AttentionParams p) {
  const int lane = threadIdx.x & 63;
  const int kv_head = blockIdx.x % p.kv_heads, rest = blockIdx.x / p.kv_heads;
  constexpr int kQuarters = ROWS >= 16 ? ROWS / 16 : 1;   // workgroups of a block of rows, 16 rows each
  const RowBlock r = row_block<ROWS>(p, rest / kQuarters);
  if (r.first >= r.rows || r.seq == p.seqs) return;
  int low, high, first, last, parts;
  keys_seen(p, r, r.first / p.group, min(r.first + ROWS - 1, r.rows - 1) / p.group, low, high);
  first = low / kTile, last = high > low ? (high + kTile - 1) / kTile : low / kTile;
  split_of(p, 0, first, last, parts);
  if (parts <= 1) return;
  const float v_scale = value_scale(p, kv_head);
  for (int i = threadIdx.x >> 6; i < min(ROWS, 16); i += 4) {
    const int row = r.first + rest % kQuarters * 16 + i;
    if (row >= r.rows) return;
    const long token = r.token + row / p.group, head = kv_head * p.group + row % p.group;
    const long at = token * p.heads + head, step = (long)p.tokens * p.heads;
    float most = -kInfinity;
    for (int s = 0; s < parts; ++s) most = fmaxf(most, p.part_ml[at + s * step].x);
    const float less = most == -kInfinity ? 0.0f : most;
    float sum = 0.0f, out[4] = {};
    for (int s = 0; s < parts; ++s) {
      const float2 ml = p.part_ml[at + s * step];
      const float by = __builtin_amdgcn_exp2f(ml.x - less);
      sum = __builtin_fmaf(by, ml.y, sum);
      if (4 * lane < p.dim) {
        const floatx4_t o = *reinterpret_cast<const floatx4_t*>(p.part_o + (at + s * step) * p.dim + 4 * lane);
#pragma unroll
        for (int e = 0; e < 4; ++e) out[e] = __builtin_fmaf(by, o[e], out[e]);
      }
    }
    const float by = sum == 0.0f ? 0.0f : v_scale / sum;
    if (4 * lane < p.dim) {
      *reinterpret_cast<Four<T>*>((T*)p.out + token * p.out_token + head * p.out_head + 4 * lane) =
          four<T>(out[0] * by, out[1] * by, out[2] * by, out[3] * by);
    }
  }
}

// ---------------------------------------------------------------- the choice
struct Plan {
  long blocks, splits, split_tiles;
  size_t ml_bytes, o_bytes;
};

Plan plan_of(int64_t tokens, int64_t seqs, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t max_seq_len, int64_t window) {
  Plan plan{};
  const int64_t group = heads / kv_heads;
  plan.blocks = tokens * group / kRows + seqs + 1;
  // parts of the keys so that there are some 512 workgroups, of 256 keys at least
  const int64_t rows = std::max<int64_t>((tokens * group + kRows - 1) / kRows, std::min(seqs, tokens));
  const int64_t keys = window > 0 ? std::min(max_seq_len, window + (tokens + seqs - 1) / std::max<int64_t>(seqs, 1)) : max_seq_len;
  const int64_t tiles = std::max<int64_t>((keys + kTile - 1) / kTile, 1);
  const int64_t wanted = std::max<int64_t>(512 / std::max<int64_t>(rows * kv_heads, 1), 1);
  plan.split_tiles = std::max<int64_t>((tiles + wanted - 1) / wanted, 4);
  plan.splits = (tiles + plan.split_tiles - 1) / plan.split_tiles;
  if (plan.splits > 1) {
    plan.ml_bytes = (size_t)(plan.splits * tokens * heads) * sizeof(float2);
    plan.ml_bytes = (plan.ml_bytes + 15) / 16 * 16;
    plan.o_bytes = (size_t)(plan.splits * tokens * heads * head_dim) * sizeof(float);
  }
  return plan;
}

template <typename T, int DP, bool FP8, bool EXTRA>
int launch_rows(const AttentionParams& p, hipStream_t st) {
  const void* kernel = (const void*)attention_rows_kernel<T, DP, FP8, EXTRA>;
  if (rows_lds<DP>() > 65536) SONAR_HIP(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, rows_lds<DP>()));
  attention_rows_kernel<T, DP, FP8, EXTRA><<<(uint32_t)(p.blocks * p.kv_heads * p.splits), kWaves * 64, rows_lds<DP>(), st>>>(p);
  if (int rc = launch_status("attention_rows_kernel")) return rc;
  if (p.splits > 1) {
    attention_join_kernel<T, kRows><<<(uint32_t)(p.blocks * (kRows / 16) * p.kv_heads), 256, 0, st>>>(p);
    return launch_status("attention_join_kernel");
  }
  return SONAR_OK;
}

template <typename T, int DP>
int launch_width(const AttentionParams& p, bool fp8, hipStream_t st) {
  const bool extra = p.cap > 0.0f || p.slopes != nullptr;
  if (fp8) return extra ? launch_rows<T, DP, true, true>(p, st) : launch_rows<T, DP, true, false>(p, st);
  return extra ? launch_rows<T, DP, false, true>(p, st) : launch_rows<T, DP, false, false>(p, st);
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
                                                      int64_t head_dim, int64_t max_seq_len, int64_t window) {
  if (check_sizes(tokens, seqs, heads, kv_heads, head_dim, max_seq_len, window) != SONAR_OK || tokens == 0 || seqs == 0) return 0;
  const Plan plan = plan_of(tokens, seqs, heads, kv_heads, head_dim, max_seq_len, window);
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
                    table_pages < (1LL << 31) && table_pages * page_size < (1LL << 31),
                "pages = %ld of %ld slots, %ld a sequence", (long)pages, (long)page_size, (long)table_pages);
  SONAR_REQUIRE(scale > 0.0 && scale <= 3e38, "scale = %g must be positive", scale);
  SONAR_REQUIRE(cap >= 0.0 && cap <= 1e30, "cap = %g must be 0 (none) or positive", cap);
  SONAR_REQUIRE(tree_mask == nullptr || (tree_words >= 1 && tree_words < (1 << 20)), "tree_words = %ld", (long)tree_words);
  SONAR_REQUIRE(tree_mask == nullptr || (window == 0 && slopes == nullptr), "a tree mask goes with neither a window nor slopes");
  SONAR_REQUIRE(window == 0 || causal, "a window goes with causal attention only");
  const int64_t cache_size = cache_dtype == SONAR_CACHE_FP8 ? 1 : 2, unit = 16 / cache_size;
  for (const sonar_kv_cache* c : {key_cache, value_cache}) {
    SONAR_REQUIRE(c->page_stride % unit == 0 && c->slot_stride % unit == 0 && c->head_stride % unit == 0 && (uintptr_t)c->data % 16 == 0,
                  "a cache must be 16-byte aligned, with strides of multiples of 16 bytes; got %ld, %ld, %ld elements", (long)c->page_stride,
                  (long)c->slot_stride, (long)c->head_stride);
    SONAR_REQUIRE(c->slot_stride >= 0 && c->slot_stride * cache_size * 64 < (1LL << 31), "a cache's slots are %ld elements apart", (long)c->slot_stride);
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
  Plan plan = plan_of(tokens, seqs, heads, kv_heads, head_dim, max_seq_len, window);
  if (scratch_bytes < plan.ml_bytes + plan.o_bytes || scratch == nullptr) plan.splits = 1;
  SONAR_REQUIRE((uintptr_t)scratch % 16 == 0, "scratch must be 16-byte aligned");
  SONAR_REQUIRE(plan.blocks * kv_heads * plan.splits < (1LL << 24) && plan.blocks * (kRows / 16) * kv_heads < (1LL << 24),
                "%ld tokens of %ld sequences and %ld heads take too many workgroups", (long)tokens, (long)seqs, (long)heads);
  auto pages_of = [&](const sonar_kv_cache* c) {
    const bool fp8 = cache_dtype == SONAR_CACHE_FP8;
    return CachePages{(const char*)c->data, c->page_stride * cache_size, c->slot_stride * cache_size, c->head_stride * cache_size,
                      fp8 ? c->scale : nullptr, c->scale_len > 1};
  };
  AttentionParams p{};
  p.q = (const char*)q, p.q_token = q_token_stride, p.q_head = q_head_stride;
  p.k = pages_of(key_cache), p.v = pages_of(value_cache);
  p.table = block_table, p.table_stride = table_stride, p.lens = seq_lens, p.starts = starts;
  p.out = (char*)out, p.out_token = out_token_stride, p.out_head = out_head_stride;
  p.slopes = slopes, p.tree = (const uint64_t*)tree_mask, p.tree_words = (int)tree_words;
  p.part_ml = (float2*)scratch, p.part_o = (float*)((char*)scratch + plan.ml_bytes);
  p.scale = (float)scale, p.cap = (float)cap, p.window = (int)window, p.causal = causal != 0, p.clear_rest = clear_rest != 0;
  int log = 0;
  while ((1LL << log) < page_size) ++log;
  p.page_shift = 31 + log, p.page_magic = (uint32_t)((1ULL << p.page_shift) / (uint64_t)page_size + 1);
  p.page_size = (int)page_size, p.pages = (int)pages, p.table_pages = (int)table_pages;
  p.tokens = (int)tokens, p.seqs = (int)seqs, p.heads = (int)heads, p.kv_heads = (int)kv_heads, p.group = (int)(heads / kv_heads);
  p.dim = (int)head_dim, p.blocks = (int)plan.blocks, p.splits = (int)plan.splits, p.split_tiles = (int)plan.split_tiles;
  const bool fp8 = cache_dtype == SONAR_CACHE_FP8;
  hipStream_t st = (hipStream_t)stream;
  return dtype == SONAR_DTYPE_F16 ? launch<_Float16>(p, fp8, st) : launch<__bf16>(p, fp8, st);
}
