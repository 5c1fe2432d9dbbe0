// Product of 8-bit integers with a scale for each token and channel (W8A8), on the int8 matrix instructions:
//   c[m][n] = T(float(sum over k of a[m][k] b[n][k]) * (a_scales[m] * b_scales[n]) + bias[n])
// Both operands lie along K, as a checkpoint and a quantiser leave them, and both are read as they lie: nothing is laid
// out anew.  The sums are integers, so every kernel, split and order gives the same bits.
//
//   int8_stream_kernel   up to 16 (32) rows: bound by the bytes of the weight; few rows of any alignment in blocks of 32
//   int8_tile_kernel     more rows, five tile sizes: bound by the matrix pipes from a few hundred rows on
//   int8_join_kernel     sums of a K that was split over workgroups
//   int8_pad_kernel      rows that no 16-byte vector is aligned to, laid down aligned for the tiles
//   int8_general_kernel  such rows as they lie, of short K, and anything without scratch
#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "sonar_layer.h"

namespace sonar {
namespace {

typedef int intx4_t __attribute__((ext_vector_type(4)));
typedef int intx16_t __attribute__((ext_vector_type(16)));

struct Int8Params {
  const int8_t* a;
  const int8_t* b;
  void* c;
  const float* a_scales;
  const float* b_scales;
  const void* bias;
  long lda, ldb;
  int m, n, k;
  int a_many, b_many;   // a scale for each row of a / of b (else one)
};

// What a sum becomes, the same in every kernel: two roundings of float32 (the sum's own where it passes 2^24), and the type's.
template <typename T>
__device__ __forceinline__ T int8_result(int sum, float scale_a, float scale_b, float bias) {
  return (T)__builtin_fmaf((float)sum, scale_a * scale_b, bias);
}

// 16 bytes of a row of k from k0 on, zeros behind its end; any alignment.  At the end of a row its last 16 bytes are loaded and
// shifted.
__device__ __forceinline__ intx4_t load_16(const int8_t* row, int k0, int k) {
  if (k >= 16) {
    const int at = min(k0, k - 16), past = min(k0 - at, 16);
    unsigned __int128 v;
    __builtin_memcpy(&v, row + at, 16);
    return __builtin_bit_cast(intx4_t, past < 16 ? v >> (8 * past) : (unsigned __int128)0);
  }
  intx4_t v = {0, 0, 0, 0};   // rows shorter than a vector
  for (int i = 0; i < 16; ++i)
    if (k0 + i < k) v[i >> 2] |= (int)((uint32_t)(uint8_t)row[k0 + i] << (8 * (i & 3)));
  return v;
}

// A row that starts at any byte (ODD) is read by whole words: 16 bytes and the word behind them, and shifted by what is over.
// Vectors at odd bytes take the hardware three times as long: 1 x 4095 x 28672 63 us, by words 37.5, 4096 columns 25.8.  No word is read that
// holds none of the bytes asked for.
template <bool ODD>
struct Row {
  const int8_t* words;
  int over, behind;   // bytes before the row's first in its word; where the word behind a piece is (its own last one if none is needed)
  __device__ __forceinline__ Row() {}
  __device__ __forceinline__ explicit Row(const int8_t* row) {
    over = ODD ? (int)((uintptr_t)row & 3) : 0;
    words = row - over;
    behind = over ? 16 : 12;
  }
};
template <bool ODD>
struct Piece {
  intx4_t v;
  int more;
  __device__ __forceinline__ void load(const Row<ODD>& row, int k) {   // k: a multiple of 4, and k + 16 bytes in the row
    typedef int words_t __attribute__((ext_vector_type(4), aligned(4)));
    v = *reinterpret_cast<const words_t*>(row.words + k);
    if (ODD) more = *reinterpret_cast<const int*>(row.words + k + row.behind);
  }
  __device__ __forceinline__ intx4_t bytes(const Row<ODD>& row) const {
    if (!ODD) return v;
    intx4_t out;
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = (int)__builtin_amdgcn_alignbyte((uint32_t)(i < 3 ? v[i + 1] : more), (uint32_t)v[i], (uint32_t)row.over);
    return out;
  }
};

// The 32 x 32 results of a wavefront at (m0, n0).  The halves of the wavefront trade quadruples, so that a lane has 16
// neighbouring channels of its token, 32 bytes of a row.  `scale_a`: of the lane's token; `scales_b` and `bias`: of the 16 channels.
template <typename T>
__device__ __forceinline__ void store_block(const intx16_t& acc, const Int8Params& p, long m0, long n0, int lane, bool vectors,
                                            float scale_a, const floatx4_t* scales_b, const floatx4_t* bias) {
  const long m = m0 + (lane & 31), n = n0 + 16 * (lane >> 5);
  T* out = (T*)p.c + m * p.n + n;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    typedef T eight_t __attribute__((ext_vector_type(8)));
    eight_t v;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      // channels 8 q + e of the first half and 16 + 8 q + e; + 4 .. 7 are the other half's
      const auto both = __builtin_amdgcn_permlane32_swap((unsigned)acc[4 * q + e], (unsigned)acc[8 + 4 * q + e], false, false);
      v[e] = int8_result<T>((int)both[0], scale_a, scales_b[2 * q][e], bias[2 * q][e]);
      v[4 + e] = int8_result<T>((int)both[1], scale_a, scales_b[2 * q + 1][e], bias[2 * q + 1][e]);
    }
    if (m < p.m) {
      if (vectors && n + 8 * q + 8 <= p.n) {
        *reinterpret_cast<eight_t*>(out + 8 * q) = v;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (n + 8 * q + e < p.n) out[8 * q + e] = v[e];
      }
    }
  }
}

// The same with the scales and the bias from memory.
template <typename T>
__device__ __forceinline__ void scale_and_store(const intx16_t& acc, const Int8Params& p, long m0, long n0, int lane, bool vectors) {
  if (m0 >= p.m || n0 >= p.n) return;
  const long m = min(m0 + (lane & 31), (long)p.m - 1);
  floatx4_t sb[4], add[4];
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const long n = min(n0 + 16 * (lane >> 5) + e, (long)p.n - 1);
    sb[e / 4][e % 4] = p.b_scales[p.b_many ? n : 0];
    add[e / 4][e % 4] = p.bias ? (float)((const T*)p.bias)[n] : 0.0f;
  }
  store_block<T>(acc, p, m0, n0, lane, vectors, p.a_scales[p.a_many ? m : 0], sb, add);
}

// ---- rows of any alignment
// 64 x 64 results a workgroup of two sets of 2 x 2 wavefronts, which take 128 bytes of K in turn and join their sums in LDS.
// Rows go through registers into the tiles' LDS order; two rounds of loads are out while a third is multiplied.  Any strides
// and sizes, and no scratch.
template <typename T>
__global__ __launch_bounds__(512) void int8_general_kernel(const Int8Params p, int cols, bool vectors) {
  constexpr int KG = 2, kStep = 128, kSlot = 128 * kStep, kRound = KG * kStep;
  extern __shared__ __attribute__((aligned(1024))) int8_t lds[];   // [group][2][row of a, then of b][piece]
  const int tid = threadIdx.x, lane = tid & 63, all_waves = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wave = all_waves & 3, group = all_waves >> 2;
  const long m0 = (long)(blockIdx.x / cols) * 64, n0 = (long)(blockIdx.x % cols) * 64;
  int8_t* slots = lds + group * 2 * kSlot;
  const int row = tid >> 3 & 31, piece = tid & 7;   // a thread's rows row + 32 i of a, then of b
  const int8_t* rows[4];
  Row<true> words[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    rows[i] = i < 2 ? p.a + min(m0 + row + 32 * i, (long)p.m - 1) * p.lda : p.b + min(n0 + row + 32 * (i - 2), (long)p.n - 1) * p.ldb;
    words[i] = Row<true>(rows[i]);
  }
  const int put_at = row * kStep + (piece ^ (row >> 1 & 7)) * 16;
  Piece<true> held[2][4];
  auto fetch = [&](int set, int round) {
    const int k = (round * KG + group) * kStep + 16 * piece;
    if ((round + 1) * kRound <= p.k) {
#pragma unroll
      for (int i = 0; i < 4; ++i) held[set][i].load(words[i], k);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) held[set][i].v = load_16(rows[i], k, p.k);
    }
  };
  const int wm = (wave & 1) * 32, wn = 64 + (wave >> 1) * 32, r = lane & 31, h = lane >> 5;
  const int at0 = r * kStep + (h ^ (r >> 1 & 7)) * 16;
  intx16_t acc = {};
  auto put = [&](int set, int round) {
    const bool whole = (round + 1) * kRound <= p.k;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      intx4_t v = held[set][i].v;
      if (whole) v = held[set][i].bytes(words[i]);
      *reinterpret_cast<intx4_t*>(slots + set * kSlot + put_at + 32 * i * kStep) = v;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (no wait for the loads that are out)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  auto multiply = [&](int set) {
    intx4_t av[4], bv[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      av[s] = *reinterpret_cast<const intx4_t*>(slots + set * kSlot + wm * kStep + (at0 ^ (32 * s)));
      bv[s] = *reinterpret_cast<const intx4_t*>(slots + set * kSlot + wn * kStep + (at0 ^ (32 * s)));
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(bv[s], av[s], acc, 0, 0, 0);
  };
  const int rounds = (p.k + 2 * kRound - 1) / (2 * kRound) * 2;   // an even number: zeros behind the end of K
  if (rounds > 0) fetch(0, 0), fetch(1, 1);
  for (int round = 0; round < rounds; round += 2) {
#pragma unroll
    for (int set = 0; set < 2; ++set) {
      put(set, round + set);   // (the other slot's readers are through: each passed this barrier after its reads)
      if (round + 2 < rounds) fetch(set, round + 2 + set);
      multiply(set);
    }
  }
  __syncthreads();
  intx4_t* sums = reinterpret_cast<intx4_t*>(lds);   // [group][wave][quadruple][lane]
#pragma unroll
  for (int q = 0; q < 4; ++q)
    sums[((group * 4 + wave) * 4 + q) * 64 + lane] = intx4_t{acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
  __syncthreads();
  if (group != 0) return;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    intx4_t v = {0, 0, 0, 0};
#pragma unroll
    for (int g = 0; g < KG; ++g) v += sums[((g * 4 + wave) * 4 + q) * 64 + lane];
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[4 * q + e] = v[e];
  }
  scale_and_store<T>(acc, p, m0 + wm, n0 + wn - 64, lane, vectors);
}

// ---- few rows
// Up to 16 MB tokens (or blocks of as many): the weight is read once a block, past LDS, straight into the operand registers of 16 x 16 x 64 matrix
// instructions (its 16 channels the first operand), 64 bytes of a row an instruction; rows of any alignment (ODD: not of words).  A workgroup owns 16 NB
// channels; its wavefronts take steps of 128 bytes of K in turn, so that together they read a run of each row, and join their
// sums through LDS.  A wavefront has DEEP steps of loads in flight, 4 KB at DEEP = 2: with 16 wavefronts on each compute unit
// that covers the latency of memory.
template <typename T, bool ODD, int kWaves, int MB, int NB, int DEEP>
__global__ __launch_bounds__(64 * kWaves, 4) void int8_stream_kernel(const Int8Params p, bool vectors) {
  constexpr int kStepK = 128;
  __shared__ intx4_t sums[kWaves][NB * MB][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, at = 16 * (lane >> 4);   // an operand's row, and its 16 bytes of 64
  const long n0 = (long)blockIdx.x * (16 * NB), m0 = (long)blockIdx.y * (16 * MB);
  const int8_t* a_rows[MB];
  const int8_t* b_rows[NB];
#pragma unroll
  for (int i = 0; i < MB; ++i) a_rows[i] = p.a + min(m0 + 16 * i + r, (long)p.m - 1) * p.lda;   // (tokens past the end: the last one's)
#pragma unroll
  for (int j = 0; j < NB; ++j) b_rows[j] = p.b + min(n0 + 16 * j + r, (long)p.n - 1) * p.ldb;
  intx4_t acc[NB][MB] = {};
  Row<ODD> a_words[MB], b_words[NB];
#pragma unroll
  for (int i = 0; i < MB; ++i) a_words[i] = Row<ODD>(a_rows[i]);
#pragma unroll
  for (int j = 0; j < NB; ++j) b_words[j] = Row<ODD>(b_rows[j]);
  struct Step {
    Piece<ODD> a[MB][2], b[NB][2];
  } held[DEEP];
  auto fetch = [&](Step& s, int k) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
#pragma unroll
      for (int j = 0; j < NB; ++j) s.b[j][x].load(b_words[j], at + k + 64 * x);
#pragma unroll
      for (int i = 0; i < MB; ++i) s.a[i][x].load(a_words[i], at + k + 64 * x);
    }
  };
  auto multiply = [&](const Step& s) {
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int i = 0; i < MB; ++i)
          acc[j][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(s.b[j][x].bytes(b_words[j]), s.a[i][x].bytes(a_words[i]), acc[j][i], 0, 0, 0);
  };
  const int whole = p.k / kStepK, mine = (whole - wave + kWaves - 1) / kWaves;   // this wavefront's steps
  const int first = wave * kStepK, next = kWaves * kStepK;
  int done = 0;
#pragma unroll
  for (int d = 0; d < DEEP; ++d)
    if (d < mine) fetch(held[d], first + d * next);
  for (; done + 2 * DEEP <= mine; done += DEEP)
#pragma unroll
    for (int d = 0; d < DEEP; ++d) {
      multiply(held[d]);
      fetch(held[d], first + (done + d + DEEP) * next);
    }
#pragma unroll
  for (int d = 0; d < DEEP; ++d) {
    if (done + d < mine) multiply(held[d]);
    if (done + d + DEEP < mine) fetch(held[d], first + (done + d + DEEP) * next);
  }
#pragma unroll
  for (int d = 0; d < DEEP; ++d)
    if (done + d + DEEP < mine) multiply(held[d]);
  if (p.k % kStepK != 0 && wave == whole % kWaves) {   // the rest of K
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int k = whole * kStepK + 64 * x + at;
      intx4_t of_a[MB];
#pragma unroll
      for (int i = 0; i < MB; ++i) of_a[i] = load_16(a_rows[i], k, p.k);
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const intx4_t of_b = load_16(b_rows[j], k, p.k);
#pragma unroll
        for (int i = 0; i < MB; ++i) acc[j][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(of_b, of_a[i], acc[j][i], 0, 0, 0);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < NB; ++j)
#pragma unroll
    for (int i = 0; i < MB; ++i) sums[wave][j * MB + i][lane] = acc[j][i];
  __syncthreads();
  for (int x = wave; x < NB * MB; x += kWaves) {
    intx4_t v = sums[0][x][lane];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v += sums[w][x][lane];
    // a lane has token 16 i + lane % 16 and channels 4 (lane / 16) + 0 .. 3 of the sixteen
    const long m = m0 + 16 * (x % MB) + r, n = n0 + 16 * (x / MB) + 4 * (lane >> 4);
    if (m >= p.m) continue;
    const float sa = p.a_scales[p.a_many ? m : 0];
    T* out = (T*)p.c + m * p.n + n;
    typedef T four_t __attribute__((ext_vector_type(4)));
    four_t result;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const long at_n = min(n + e, (long)p.n - 1);
      result[e] = int8_result<T>(v[e], sa, p.b_scales[p.b_many ? at_n : 0], p.bias ? (float)((const T*)p.bias)[at_n] : 0.0f);
    }
    if (vectors && n + 4 <= p.n) {
      *reinterpret_cast<four_t*>(out) = result;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < p.n) out[e] = result[e];
    }
  }
}

// ---- tiles
struct TilePlan {
  int tiles_m, tiles_n, splits, per_xcd;
};

// Tile number -> row and column of tiles: panels of up to eight rows of tiles, down the rows first, so that the 32
// workgroups of a die at work together share operands.
__device__ __forceinline__ void tile_at(int tile, const TilePlan& t, int& tm, int& tn) {
  const int panel = tile / (8 * t.tiles_n), rows = min(8, t.tiles_m - 8 * panel), in = tile - panel * 8 * t.tiles_n;
  tn = __builtin_amdgcn_readfirstlane(in / rows);   // (the division leaves its quotient in a vector register)
  tm = __builtin_amdgcn_readfirstlane(8 * panel + in - tn * rows);
}

// A wavefront owns 32 MT rows x 32 NT columns in 32 x 32 x 32 instructions, WM x 2 wavefronts a tile.  The weight is the first
// operand: a lane then has one token and four neighbouring channels a register quadruple.
// K goes in stages of kStageK bytes, which LDS-DMA brings into a ring of kRing stages.  16-byte piece c of row i of a stage
// stands at c ^ (i / 2 & 7) (rows of 64: c ^ (i / 4 & 3)), so that lanes that read together find different banks: 548 bytes/ns
// a compute unit, where c ^ (i & 7) reaches half and no turn a quarter of that.  Stages of 128 bytes because a copy of whole
// 128-byte lines runs at 55 bytes a cycle and compute unit, one of half lines at 41 (2048 x 14336 x 4096: 133 -> 104 us); the
// 256 x 256 tile has no room for three of them and takes four of 64 (8192 x 4096 x 28672: two of 128 take 3 % longer).
// Operands are read one step (32 of K) ahead of their matrix instructions.
// Eight wavefronts for the tiles of 128 rows and up: while one waits at a barrier or issues its copies, the other of its
// SIMD multiplies (four wavefronts with 128 x 128 each take 10 % longer).
// KG: that many sets of wavefronts take stages in turn and join their sums through LDS, for tiles too small to keep a compute
// unit busy otherwise (100 x 4096 x 4096: 9.7 -> 9.2 us).
// What K is over whole rounds of stages is one more stage, whose pieces behind the end of a row are copied from its last
// one and cleared (those of a) once they have landed.
template <typename T, int WM, int MT, int NT, int KG, int kStageK, int kRing>
__global__ __launch_bounds__(128 * WM * KG, (32 * MT * WM + 64 * NT) * kStageK * kRing * KG <= 81920 ? WM * KG : WM * KG / 2)
void int8_tile_kernel(const Int8Params p, const TilePlan t, int* __restrict__ partial, bool vectors) {
  constexpr int BM = 32 * MT * WM, BN = 64 * NT, kWaves = 2 * WM, kThreads = 64 * kWaves, kStage = (BM + BN) * kStageK;
  constexpr int kPieces = kStageK / 16, kSteps = kStageK / 32;                                    // of a row
  constexpr int kRows = 64 / kPieces, kLoadsA = BM / kRows / kWaves, kLoads = (BM + BN) / kRows / kWaves;   // of a copy; copies of a wavefront
  static_assert(BM <= kThreads && BN <= kThreads && (kRing - 2) * kLoads < 64, "");
  extern __shared__ __attribute__((aligned(1024))) int8_t lds[];
  const int tid = threadIdx.x, lane = tid & 63, all_waves = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wave = all_waves % kWaves, group = all_waves / kWaves;
  const int unit = (blockIdx.x & 7) * t.per_xcd + (blockIdx.x >> 3);   // workgroups go to the eight dies in turn
  const int tiles = t.tiles_m * t.tiles_n;
  if (unit >= tiles * t.splits) return;
  const int split = unit / tiles, tile = unit - split * tiles;
  int tm, tn;
  tile_at(tile, t, tm, tn);
  const long m0 = (long)tm * BM, n0 = (long)tn * BN;
  // rounds of KG stages, dealt evenly; the last split has the rest of K too
  const int all = p.k / (kStageK * KG), first = split * all / t.splits, whole = (split + 1) * all / t.splits - first;
  const bool rest = split == t.splits - 1 && p.k % (kStageK * KG) != 0;
  const int count = whole + (rest ? 1 : 0);

  // the scales and the bias of the tile, a row and a column a thread, until its results are scaled
  float my_scale_a = 0, my_scale_b = 0, my_bias = 0;
  if (partial == nullptr) {
    const long m = min(m0 + tid % kThreads, (long)p.m - 1), n = min(n0 + tid % kThreads, (long)p.n - 1);
    my_scale_a = p.a_scales[p.a_many ? m : 0];
    my_scale_b = p.b_scales[p.b_many ? n : 0];
    if (p.bias != nullptr) my_bias = (float)((const T*)p.bias)[n];
  }

  // copies: of kRows rows each; lane i brings piece i % kPieces of row i / kPieces
  int8_t* ring = lds + group * (kRing * kStage);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void_t*)ring;
  const char* a_base = (const char*)p.a + m0 * p.lda;
  const char* b_base = (const char*)p.b + n0 * p.ldb;
  auto turned = [](int row) { return kStageK == 64 ? row >> 2 & 3 : row >> 1 & 7; };
  uint32_t off[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const bool b = i >= kLoadsA;
    const int row = (b ? wave * (kLoads - kLoadsA) + i - kLoadsA : wave * kLoadsA + i) * kRows + lane / kPieces;
    const long end = b ? p.n - 1 - n0 : p.m - 1 - m0;   // rows past the end repeat the last one and are not stored
    off[i] = (uint32_t)(min((long)row, end) * (b ? p.ldb : p.lda)) + (lane % kPieces ^ turned(row)) * 16;
  }
  auto to = [&](int i, int stage) {
    const bool b = i >= kLoadsA;
    return lds0 + (stage % kRing) * kStage +
           (b ? BM * kStageK + (wave * (kLoads - kLoadsA) + i - kLoadsA) * 1024 : (wave * kLoadsA + i) * 1024);
  };
  auto copy = [&](int i, int stage) {   // of this split; a whole one
    copy_to_lds<16>(to(i, stage), off[i], (i >= kLoadsA ? b_base : a_base) + ((long)(first + stage) * KG + group) * kStageK);
  };
  auto copy_rest = [&]() {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const bool b = i >= kLoadsA;
      const int row = (b ? wave * (kLoads - kLoadsA) + i - kLoadsA : wave * kLoadsA + i) * kRows + lane / kPieces;
      const uint32_t piece = (lane % kPieces ^ turned(row)) * 16, k = (all * KG + group) * kStageK + piece;
      copy_to_lds<16>(to(i, whole), off[i] - piece + min(k, (uint32_t)p.k - 16), b ? b_base : a_base);
    }
  };
  auto clear_rest = [&]() {   // the pieces of a behind the end of K
    for (int i = tid % kThreads; i < BM * kPieces; i += kThreads) {
      const int row = i / kPieces, c = i % kPieces;
      if ((all * KG + group) * kStageK + 16 * c >= p.k)
        *reinterpret_cast<intx4_t*>(ring + (whole % kRing) * kStage + row * kStageK + (c ^ turned(row)) * 16) = intx4_t{0, 0, 0, 0};
    }
    __syncthreads();
  };

  // operands: row lane % 32 of a block, piece 2 s + lane / 32 of step s
  const int wm = wave % WM, wn = wave / WM, r = lane & 31, h = lane >> 5;
  const int at0 = r * kStageK + (h ^ turned(r)) * 16;
  const int a_at = wm * MT * 32 * kStageK + at0, b_at = (BM + wn * NT * 32) * kStageK + at0;
  intx4_t fa[2][MT], fb[2][NT];
  auto read_a = [&](int s, int i, int stage) {
    fa[s & 1][i] = *reinterpret_cast<const intx4_t*>(ring + (stage % kRing) * kStage + (a_at ^ (32 * s)) + i * 32 * kStageK);
  };
  auto read_b = [&](int s, int i, int stage) {
    fb[s & 1][i] = *reinterpret_cast<const intx4_t*>(ring + (stage % kRing) * kStage + (b_at ^ (32 * s)) + i * 32 * kStageK);
  };
  intx16_t acc[MT][NT] = {};

  // Step s of a stage: its matrix instructions, between them the reads of the next step and a share of the copies.
  auto step = [&](int s, int stage, bool copies) {
    constexpr int kAll = MT * NT, kSpread = kSteps > 2 ? kSteps - 1 : 1;   // the copies are over before the last step
#pragma unroll
    for (int x = 0; x < kAll; ++x) {
      // the next step's operands, spread over the first three quarters: a's first, then b's, then a's others
#pragma unroll
      for (int y = 0; y < MT + NT; ++y)
        if (y * (kAll * 3 / 4) / (MT + NT) == x) {
          const int next = s == kSteps - 1 ? stage + 1 : stage, at = (s + 1) % kSteps;
          if (y == 0) read_a(at, 0, next);
          else if (y <= NT) read_b(at, y - 1, next);
          else read_a(at, y - NT, next);
        }
      if (copies) {
#pragma unroll
        for (int y = 0; y < kLoads; ++y)
          if (y * kSpread * kAll / kLoads == s * kAll + x) copy(y, stage + kRing - 1);
      }
      acc[x / NT][x % NT] =
          __builtin_amdgcn_mfma_i32_32x32x32_i8(fb[s & 1][x % NT], fa[s & 1][x / NT], acc[x / NT][x % NT], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  const int ahead = min(whole, kRing - 1);
  for (int i = 0; i < ahead; ++i)
#pragma unroll
    for (int y = 0; y < kLoads; ++y) copy(y, i);
  const bool rest_early = rest && whole < kRing - 1;
  if (rest_early) copy_rest();
  // stage 0: its copies have landed once those of the stages behind it are all that is out
  if (whole >= kRing - 1) asm volatile("s_waitcnt vmcnt(%0)" ::"i"((kRing - 2) * kLoads) : "memory");
  else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  if (rest && whole == 0) clear_rest();
#pragma unroll
  for (int i = 0; i < MT; ++i) read_a(0, i, 0);
#pragma unroll
  for (int i = 0; i < NT; ++i) read_b(0, i, 0);
  // The next stage has landed in every wavefront's copies, and every wavefront has read this one: behind the barrier the
  // next one may be read and this one's room filled.
  auto next_stage = [&](auto waits) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"i"(decltype(waits)::value) : "memory");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };
  int stage = 0;
  for (; stage + kRing - 1 < whole; ++stage) {
#pragma unroll
    for (int s = 0; s < kSteps - 1; ++s) step(s, stage, true);
    next_stage(std::integral_constant<int, (kRing - 2) * kLoads>());
    step(kSteps - 1, stage, false);
  }
  if (rest && !rest_early) copy_rest();
  for (; stage < count; ++stage) {   // (the last one reads operands that nothing uses)
#pragma unroll
    for (int s = 0; s < kSteps - 1; ++s) step(s, stage, false);
    next_stage(std::integral_constant<int, 0>());
    if (rest && stage + 1 == whole) clear_rest();
    step(kSteps - 1, stage, false);
  }

  // Groups: every sum to LDS, and each group's wavefront takes the blocks x with x % KG == group.
  if constexpr (KG > 1) {
    __syncthreads();
    intx4_t* sums = reinterpret_cast<intx4_t*>(lds);   // [group][wave][block][quadruple][lane]
#pragma unroll
    for (int x = 0; x < MT * NT; ++x)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const intx16_t& v = acc[x / NT][x % NT];
        sums[(((group * kWaves + wave) * MT * NT + x) * 4 + q) * 64 + lane] =
            intx4_t{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
      }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < MT * NT; ++x) {
      if (x % KG != group) continue;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        intx4_t v = {0, 0, 0, 0};
#pragma unroll
        for (int g = 0; g < KG; ++g) v += sums[(((g * kWaves + wave) * MT * NT + x) * 4 + q) * 64 + lane];
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[x / NT][x % NT][4 * q + e] = v[e];
      }
    }
  }
  const long wm0 = m0 + wm * MT * 32, wn0 = n0 + wn * NT * 32;
  if (partial != nullptr) {   // sums in the order of the registers, block after block
    int* out = partial + ((long)(split * tiles + tile) * kWaves + wave) * (MT * NT * 1024);
#pragma unroll
    for (int x = 0; x < MT * NT; ++x) {
      if (KG > 1 && x % KG != group) continue;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<intx4_t*>(out + x * 1024 + q * 256 + lane * 4) =
            intx4_t{acc[x / NT][x % NT][4 * q], acc[x / NT][x % NT][4 * q + 1], acc[x / NT][x % NT][4 * q + 2],
                    acc[x / NT][x % NT][4 * q + 3]};
    }
    return;
  }
  float* scales = reinterpret_cast<float*>(lds);   // of a's rows, of b's rows, and the bias
  __syncthreads();
  if (tid < BM) scales[tid] = my_scale_a;
  if (tid < BN) scales[BM + tid] = my_scale_b, scales[BM + BN + tid] = my_bias;
  __syncthreads();
  if constexpr (KG > 1) {
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const float scale_a = scales[(wm * MT + i) * 32 + r];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        if ((i * NT + j) % KG != group) continue;
        const float* of_b = scales + BM + (wn * NT + j) * 32 + 16 * h;
        floatx4_t sb[4], add[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sb[e] = *reinterpret_cast<const floatx4_t*>(of_b + 4 * e);
          add[e] = *reinterpret_cast<const floatx4_t*>(of_b + BN + 4 * e);
        }
        store_block<T>(acc[i][j], p, wm0 + i * 32, wn0 + j * 32, lane, vectors, scale_a, sb, add);
      }
    }
  } else {
    // 32 rows at a time turn in LDS, so that they leave as whole lines, 64 NT bytes a row (in pieces of 32 bytes from where
    // they are 8192 x 4096 x 28672 takes 3 % longer)
    constexpr int kPitch = 64 * NT + 16, kLanes = 4 * NT, kRowsOut = 64 / kLanes;
    typedef T eight_t __attribute__((ext_vector_type(8)));
    typedef T four_t __attribute__((ext_vector_type(4)));
    int8_t* turn_lds = lds + (BM + 2 * BN) * 4 + wave * 32 * kPitch;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const float scale_a = scales[(wm * MT + i) * 32 + r];
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int n = j * 32 + 8 * q + 4 * h;   // of the wavefront's columns
          const floatx4_t sb = *reinterpret_cast<const floatx4_t*>(scales + BM + wn * NT * 32 + n);
          const floatx4_t add = *reinterpret_cast<const floatx4_t*>(scales + BM + BN + wn * NT * 32 + n);
          four_t v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = int8_result<T>(acc[i][j][4 * q + e], scale_a, sb[e], add[e]);
          *reinterpret_cast<four_t*>(turn_lds + r * kPitch + n * 2) = v;
        }
      __builtin_amdgcn_sched_barrier(0);   // (one strip's registers at a time)
#pragma unroll
      for (int x = 0; x < 32 / kRowsOut; ++x) {
        const int row = x * kRowsOut + lane / kLanes, col = lane % kLanes * 8;
        const eight_t v = *reinterpret_cast<const eight_t*>(turn_lds + row * kPitch + col * 2);
        const long m = wm0 + i * 32 + row, n = wn0 + col;
        T* out = (T*)p.c + m * p.n + n;
        if (m < p.m) {
          if (vectors && n + 8 <= p.n) {
            *reinterpret_cast<eight_t*>(out) = v;
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (n + e < p.n) out[e] = v[e];
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

// The sum of the splits' partial tiles, a wavefront a block of 32 x 32.
template <typename T, int WM, int MT, int NT>
__global__ __launch_bounds__(256) void int8_join_kernel(const Int8Params p, const TilePlan t, const int* __restrict__ partial, bool vectors) {
  const int lane = threadIdx.x & 63;
  const long block = (long)blockIdx.x * 4 + (threadIdx.x >> 6);   // ((tile * 2 WM + wave) * MT + i) * NT + j
  const int tiles = t.tiles_m * t.tiles_n;
  if (block >= (long)tiles * 2 * WM * MT * NT) return;
  const int j = block % NT, i = block / NT % MT, wave = block / (MT * NT) % (2 * WM), tile = block / (MT * NT * 2 * WM);
  intx16_t acc = {};
  for (int s = 0; s < t.splits; ++s) {
    const int* from = partial + ((long)s * tiles * 2 * WM * MT * NT + block) * 1024;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const intx4_t v = *reinterpret_cast<const intx4_t*>(from + q * 256 + lane * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[4 * q + e] += v[e];
    }
  }
  int tm, tn;
  tile_at(tile, t, tm, tn);   // (a workgroup's four blocks are of one tile)
  const long m0 = (long)tm * 32 * MT * WM + (wave % WM * MT + i) * 32, n0 = (long)tn * 64 * NT + (wave / WM * NT + j) * 32;
  scale_and_store<T>(acc, p, m0, n0, lane, vectors);
}

// Rows of a and of b -> rows `pitch` bytes apart, zeros behind K; a wavefront a row, 1 KB at a time, four of them asked for at once.
__global__ __launch_bounds__(256) void int8_pad_kernel(const Int8Params p, int8_t* __restrict__ a, int8_t* __restrict__ b, int pitch) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long all = (long)p.m + p.n;
  for (long row = (long)blockIdx.x * 4 + wave; row < all; row += (long)gridDim.x * 4) {
    const bool of_a = row < p.m;
    const int8_t* from = of_a ? p.a + row * p.lda : p.b + (row - p.m) * p.ldb;
    int8_t* to = of_a ? a + row * pitch : b + (row - p.m) * pitch;
    const Row<true> words(from);
    for (int k0 = lane * 16; k0 < pitch; k0 += 4096) {
      Piece<true> pieces[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (k0 + 1024 * i + 16 <= p.k) pieces[i].load(words, k0 + 1024 * i);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = k0 + 1024 * i;
        if (k + 16 <= p.k) *reinterpret_cast<intx4_t*>(to + k) = pieces[i].bytes(words);
        else if (k < pitch) *reinterpret_cast<intx4_t*>(to + k) = load_16(from, k, p.k);
      }
    }
  }
}

// ---- host
enum Form { kGeneral, kStream32, kStream16, kStreamTwo, kTile64, kTile128Wide, kTile128, kTile256Tall, kTile256, kForms };
// Rows and columns of a form's tile, and what it takes (us): a round of 256 workgroups, and 1024 of K in it.  Fitted to 140
// shapes of 24 to 4096 rows, 256 to 28672 channels, K of 2048 to 14336; the choice they make is 0.2 % slower than the best one
// (geometric mean; at most 6 %).  Of 118 with rows of any alignment, K of 24 to 14336, 2.1 % (at most 64 %: 86 x 4148 x 1955
// takes tiles, 20.2 us, where the stream would take 12.3).
struct FormCost {
  int rows, cols;
  float round, per_k;
};
constexpr FormCost kCosts[kForms] = {{64, 64, 4.0f, 5.5f},      {16, 32, 0, 0},        {16, 16, 0, 0},        {32, 16, 0.35f, 2.5f}, {64, 64, 4.4f, 1.3f},
                                     {64, 128, 5.0f, 2.0f}, {128, 128, 5.0f, 3.1f}, {256, 128, 6.5f, 4.6f}, {256, 256, 8.1f, 8.3f}};
constexpr float kStreamUs = 3.0f;   // start and end of the streams' rounds, which overlap
constexpr float kStreamRoundUs = 2.0f;   // a further round at least, however short K is (64 x 33 x 1048576: 996 us, 512 rounds)
// A row of aligned copies at least, whatever its length.  The copies themselves take 0.22 ns a row (1048640 rows of 33 bytes
// 240 us); less is counted because the general kernel's rounds are counted a third too high where there are many of them.
constexpr float kCopyRowUs = 0.13e-3f;
constexpr float kLaunchUs = 4.5f, kBytesPerUs = 4.5e6f;   // a launch more, for partial sums or aligned copies; their bytes

struct Int8Choice {
  int form, splits;
};
constexpr int64_t kStreamRows = 32 * 65535;   // a grid's second dimension
constexpr int64_t kMostTiles = (1 << 22) - 1;   // of a launch, the parts of K counted: 512 threads each are fewer than 2^32
thread_local Int8Choice g_forced = {-1, 1};

int64_t padded_k(int64_t k) { return (k + 255) / 256 * 256; }   // of aligned copies: whole rounds of every form
int64_t tiles_of(int form, int64_t m, int64_t n) {
  return ((m + kCosts[form].rows - 1) / kCosts[form].rows) * ((n + kCosts[form].cols - 1) / kCosts[form].cols);
}

// Whether tiles can split K so: every split has 512 of it at least, so that the join costs less than it saves.
bool may_split(int splits, int64_t k) { return splits == 1 || k / splits >= 512; }

Int8Choice choose_form(int64_t m, int64_t n, int64_t k, bool aligned) {
  if (g_forced.form >= 0) return g_forced;
  // Up to 256 workgroups of 16 channels sixteen wavefronts each, else eight with 32 channels, two workgroups on a compute unit
  // (1 x 4096 x 4096 5.8 us, 7.2 with 32 channels; 16 x 4096 x 28672 29.0, 35.7 with 16).
  if (m <= 16) return {n <= 4096 ? kStream16 : kStream32, 1};
  // 17 to 32 rows: less than the tiles' 64 where the weight is small (24 x 2048 x 2048 6.1 us, tiles 6.8; 24 x 14336 x 1024 at
  // 18, split tiles 13.0).  Unaligned rows would first be laid down for the tiles.
  if (m <= 32 && ((n <= 4096 && k <= 6144) || !aligned)) return {kStreamTwo, 1};
  if (k < 16) return {kGeneral, 1};
  Int8Choice best = {kTile64, 1};
  float least = 3.4e38f, copies = 0;
  if (!aligned) {   // the tiles would have to wait for copies
    best = {kGeneral, 1};
    least = (float)((tiles_of(kGeneral, m, n) + 255) / 256) * (kCosts[kGeneral].round + kCosts[kGeneral].per_k * (float)k / 1024);
    const float rows = (float)(m + n);
    copies = kLaunchUs + std::max(rows * (float)(k + padded_k(k)) / kBytesPerUs, rows * kCopyRowUs);
    // The stream in blocks of 32 rows reads the weight once a block, but has sixteen wavefronts on 16 channels: 77 x 1003 x 1537
    // 7.9 us, the general kernel 9.8; 200 x 2047 x 513 8.3 and 12.1; 200 x 1003 x 1537 12.9 and 10.1.
    const float rounds = (float)((tiles_of(kStreamTwo, m, n) + 255) / 256);
    const float streams = kStreamUs + std::max(rounds * (kCosts[kStreamTwo].round + kCosts[kStreamTwo].per_k * (float)k / 1024),
                                               (rounds - 1) * kStreamRoundUs);
    if (m <= kStreamRows && streams < least) least = streams, best = {kStreamTwo, 1};
  }
  const float tile_k = (float)(aligned ? k : padded_k(k));
  for (int form = kTile64; form <= kTile256; ++form)
    for (int splits = 1; splits <= 8 && may_split(splits, k); splits *= 2) {
      const int64_t tiles = tiles_of(form, m, n);
      if (splits > 1 && tiles * splits > 1024) break;
      const float rounds = (float)((tiles * splits + 255) / 256);
      float us = rounds * (kCosts[form].round + kCosts[form].per_k * tile_k / splits / 1024);
      if (splits > 1) us += kLaunchUs + (float)tiles * splits * kCosts[form].rows * kCosts[form].cols * 8 / kBytesPerUs;
      us += copies;
      if (us < least) least = us, best = {form, splits};
    }
  return best;
}

bool is_tile(int form) { return form >= kTile64; }

size_t partial_bytes(const Int8Choice& s, int64_t m, int64_t n) {
  if (!is_tile(s.form) || s.splits <= 1) return 0;
  return (size_t)tiles_of(s.form, m, n) * s.splits * kCosts[s.form].rows * kCosts[s.form].cols * 4;
}
size_t padded_bytes(const Int8Choice& s, int64_t m, int64_t n, int64_t k, bool aligned) {
  return is_tile(s.form) && !aligned ? (size_t)(m + n) * padded_k(k) : 0;
}

template <typename T, int WM, int MT, int NT, int KG, int kStageK, int kRing>
int launch_tiles(const Int8Params& p, int splits, int* partial, bool vectors, hipStream_t st) {
  constexpr int BM = 32 * MT * WM, BN = 64 * NT;
  constexpr int kStages = (BM + BN) * kStageK * kRing * KG;
  constexpr int kSums = KG > 1 ? KG * BM * BN * 4 : 4 * (BM + 2 * BN) + 2 * WM * 32 * (64 * NT + 16);
  constexpr int kLds = kStages > kSums ? kStages : kSums;
  static_assert(kLds <= 163840, "");
  TilePlan t;
  t.tiles_m = (int)(((int64_t)p.m + BM - 1) / BM), t.tiles_n = (int)(((int64_t)p.n + BN - 1) / BN);
  t.splits = splits;
  const int64_t units = (int64_t)t.tiles_m * t.tiles_n * splits;   // (kMostTiles at most)
  t.per_xcd = (int)((units + 7) / 8);
  if (kLds > 65536)
    SONAR_HIP(hipFuncSetAttribute((const void*)int8_tile_kernel<T, WM, MT, NT, KG, kStageK, kRing>,
                                  hipFuncAttributeMaxDynamicSharedMemorySize, kLds));
  int8_tile_kernel<T, WM, MT, NT, KG, kStageK, kRing><<<8 * t.per_xcd, 128 * WM * KG, kLds, st>>>(p, t, partial, vectors);
  if (partial != nullptr) {
    static_assert(MT * NT * 2 * WM % 4 == 0, "");
    int8_join_kernel<T, WM, MT, NT><<<t.tiles_m * t.tiles_n * (MT * NT * WM / 2), 256, 0, st>>>(p, t, partial, vectors);
  }
  return launch_status("int8_tile_kernel");
}

template <typename T, int kWaves, int MB, int NB, int DEEP>
void launch_stream(const Int8Params& p, bool vectors, hipStream_t st) {
  const dim3 grid((p.n + 16 * NB - 1) / (16 * NB), (p.m + 16 * MB - 1) / (16 * MB));
  if (((uintptr_t)p.a | (uintptr_t)p.b | (uintptr_t)p.lda | (uintptr_t)p.ldb) % 4 != 0)
    int8_stream_kernel<T, true, kWaves, MB, NB, DEEP < 2 ? DEEP : 2><<<grid, 64 * kWaves, 0, st>>>(p, vectors);
  else
    int8_stream_kernel<T, false, kWaves, MB, NB, DEEP><<<grid, 64 * kWaves, 0, st>>>(p, vectors);
}

template <typename T>
int run_form(const Int8Params& p, const Int8Choice& s, int* partial, bool vectors, hipStream_t st) {
  switch (s.form) {
    case kTile64: return launch_tiles<T, 2, 1, 1, 2, 128, 4>(p, s.splits, partial, vectors, st);
    case kTile128Wide: return launch_tiles<T, 2, 1, 2, 2, 128, 3>(p, s.splits, partial, vectors, st);
    case kTile128: return launch_tiles<T, 4, 1, 2, 1, 128, 3>(p, s.splits, partial, vectors, st);
    case kTile256Tall: return launch_tiles<T, 4, 2, 2, 1, 128, 3>(p, s.splits, partial, vectors, st);
    case kTile256: return launch_tiles<T, 4, 2, 4, 1, 64, 4>(p, s.splits, partial, vectors, st);
    case kStream32: launch_stream<T, 8, 1, 2, 3>(p, vectors, st); break;   // (two steps in flight where a word more goes with each)
    case kStream16: launch_stream<T, 16, 1, 1, 2>(p, vectors, st); break;
    case kStreamTwo: launch_stream<T, 16, 2, 1, 2>(p, vectors, st); break;
    default: {
      const int64_t rows = ((int64_t)p.m + 63) / 64, cols = ((int64_t)p.n + 63) / 64;
      constexpr int kLds = 65536;
      int8_general_kernel<T><<<(int)(rows * cols), 512, kLds, st>>>(p, (int)cols, vectors);
    }
  }
  return launch_status("int8 product");
}

}  // namespace
}  // namespace sonar

using namespace sonar;

extern "C" int sonar_debug_int8_form(int form, int splits) {
  SONAR_REQUIRE(form >= -1 && form < kForms && splits >= 1 && splits <= 8, "form = %d, splits = %d", form, splits);
  g_forced = {form, splits};
  return SONAR_OK;
}

extern "C" int sonar_debug_int8_choice(int64_t size_m, int64_t size_n, int64_t size_k, int aligned, int* splits) {
  const Int8Choice s = choose_form(size_m, size_n, size_k, aligned && size_k % 16 == 0);
  if (splits != nullptr) *splits = s.splits;
  return s.form;
}

extern "C" size_t sonar_scaled_mm_int8_scratch_bytes(int64_t size_m, int64_t size_n, int64_t size_k, int aligned) {
  if (size_m <= 0 || size_n <= 0 || size_k <= 0) return 0;
  const bool vectors_of_k = aligned && size_k % 16 == 0;
  const Int8Choice s = choose_form(size_m, size_n, size_k, vectors_of_k);
  return padded_bytes(s, size_m, size_n, size_k, vectors_of_k) + partial_bytes(s, size_m, size_n);
}

extern "C" int sonar_scaled_mm_int8(const int8_t* a, int64_t a_row_stride, const int8_t* b, int64_t b_row_stride, void* c,
                                    const float* a_scales, int64_t a_scales_len, const float* b_scales, int64_t b_scales_len,
                                    const void* bias, void* scratch, size_t scratch_bytes, int dtype, int64_t size_m,
                                    int64_t size_n, int64_t size_k, void* stream) {
  SONAR_REQUIRE(dtype == SONAR_DTYPE_F16 || dtype == SONAR_DTYPE_BF16, "unknown dtype = %d: float16 or bfloat16 results", dtype);
  SONAR_REQUIRE(size_m >= 0 && size_m < (1LL << 25) && size_n >= 0 && size_n < (1LL << 25), "size_m = %ld, size_n = %ld",
                (long)size_m, (long)size_n);
  SONAR_REQUIRE(size_k >= 0 && size_k < 131072, "size_k = %ld: the 32-bit sums hold fewer than 131072 products", (long)size_k);
  if (size_m == 0 || size_n == 0) return SONAR_OK;
  SONAR_REQUIRE(c && a_scales && b_scales && (size_k == 0 || (a && b)), "a, b, c and the scales must not be NULL");
  SONAR_REQUIRE(a_row_stride >= size_k && b_row_stride >= size_k, "row strides %ld and %ld are smaller than size_k = %ld",
                (long)a_row_stride, (long)b_row_stride, (long)size_k);
  SONAR_REQUIRE((a_scales_len == 1 || a_scales_len == size_m) && (b_scales_len == 1 || b_scales_len == size_n),
                "a_scales holds %ld numbers (1 or size_m = %ld are needed), b_scales %ld (1 or size_n = %ld)", (long)a_scales_len,
                (long)size_m, (long)b_scales_len, (long)size_n);
  SONAR_REQUIRE(scratch == nullptr || (uintptr_t)scratch % 16 == 0, "scratch must be 16-byte aligned");
  Int8Params p{a,        b,        c, a_scales, b_scales, bias, a_row_stride, b_row_stride, (int)size_m, (int)size_n,
               (int)size_k, a_scales_len > 1, b_scales_len > 1};
  hipStream_t st = (hipStream_t)stream;
  // (a tile's rows are found with 32-bit offsets: rows further than 8 MB apart are laid down nearer first)
  const bool aligned = ((uintptr_t)a | (uintptr_t)b | (uintptr_t)a_row_stride | (uintptr_t)b_row_stride | (uintptr_t)size_k) % 16 == 0 &&
                       a_row_stride < (1 << 23) && b_row_stride < (1 << 23);
  const bool vectors = size_n % 8 == 0 && ((uintptr_t)c | (uintptr_t)bias) % 16 == 0;
  if (scratch == nullptr) scratch_bytes = 0;
  Int8Choice s = choose_form(size_m, size_n, size_k, aligned);
  if (is_tile(s.form) && size_k < 16) s = {kGeneral, 1};
  SONAR_REQUIRE(is_tile(s.form) || s.form == kGeneral || size_m <= (s.form == kStreamTwo ? kStreamRows : kCosts[s.form].rows),
                "form %d does not take %ld rows", s.form, (long)size_m);
  const size_t padded = padded_bytes(s, size_m, size_n, size_k, aligned);
  if (padded > scratch_bytes) s = {kGeneral, 1};
  if (!is_tile(s.form) || !may_split(s.splits, size_k) || padded + partial_bytes(s, size_m, size_n) > scratch_bytes) s.splits = 1;
  SONAR_REQUIRE((s.form != kGeneral && !is_tile(s.form)) || tiles_of(s.form, size_m, size_n) * s.splits <= kMostTiles,
                "size_m = %ld, size_n = %ld: more tiles than a launch takes", (long)size_m, (long)size_n);
  if (is_tile(s.form) && padded > 0) {   // (the first launch: nothing is refused behind it)
    const int pitch = (int)padded_k(size_k);
    int8_t* copies = (int8_t*)scratch;
    const int64_t groups = (size_m + size_n + 3) / 4;
    int8_pad_kernel<<<(int)(groups < 16384 ? groups : 16384), 256, 0, st>>>(p, copies, copies + size_m * pitch, pitch);
    p.a = copies, p.b = copies + size_m * pitch, p.lda = p.ldb = p.k = pitch;
  }
  int* partial = s.splits > 1 ? (int*)((char*)scratch + padded) : nullptr;
  return dtype == SONAR_DTYPE_F16 ? run_form<_Float16>(p, s, partial, vectors, st) : run_form<__bf16>(p, s, partial, vectors, st);
}
