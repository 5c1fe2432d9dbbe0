// The experts of each token and their weights, from the router's logits x:
//   s = softmax(x) or 1 / (1 + exp(-x));  c = s + bias, or x itself, which has the order of s, without a bias
//   ids: the topk largest c, of the experts in the best groups where there are groups;  weights: s of them
// Equal choices go to the lowest expert.  What decides, s + bias and the groups' sums, is taken in 64 bits: two experts whose
// float32 sums are equal, or whose scores are below float32's range, are told apart.
//
// A choice is kept as words whose unsigned order is that of the numbers: without a bias one, of the float32 logit; with a bias
// the two of the double, the lower one looked at only where upper ones are equal.  A lane holds R neighbouring experts of a
// token and knows the largest of them.  Every round finds the largest first word over the token's lanes by lane moves, asks which
// lanes have it (and looks at the second words only if several have), takes the lowest lane's lowest expert, and that lane looks
// for its next.  Word 0 is below every number's: an expert that is taken, left out or not there.
// Groups whose experts lie in 2^n whole lanes are judged from registers, others through LDS.
// Bound by the vector instructions (the 64-bit exponentials and the rounds; 4 to 8 wavefronts a SIMD take the same time), and by
// the latency of their chains where tokens are few.  16384 x 256, sigmoid, bias, 4 of 8 groups: 132 us with choices and 64-bit
// maxima in LDS; 28.6 by lane moves; 20.9 with no loop over tokens around it all (which kept constants in 80 registers), the
// scoring's branch outside the experts' loop (their chains side by side, one set of constants), which of a lane's experts it is
// as lane masks, and the groups from registers; 19.6 with the words of the double itself (before, its float32 rounding and what
// that leaves).  (Choices in float32 first, and in 64 bits only for the tokens where two come near each other: no gain.)
#include "common.hpp"
#include "lane_reduce.hpp"
#include "sonar_layer.h"

namespace sonar {
namespace {

constexpr int kMaxExperts = 1024, kMaxGroups = 64, kMaxTopk = 64, kWaves = 4;

struct RouterParams {
  const void* logits;
  long row_stride;
  const float* bias;
  float* weights;
  int32_t* ids;
  long tokens;
  int dtype, experts, topk, scoring, renormalize, groups, kept_groups;
  double factor;
};

// float -> a word with its order, above 0 (numbers and infinities; equal zeros equal)
__device__ __forceinline__ uint32_t ordered(float f) {
  const uint32_t b = __builtin_bit_cast(uint32_t, f + 0.0f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float number_of(uint32_t w) {
  return __builtin_bit_cast(float, w ^ (w & 0x80000000u ? 0x80000000u : 0xffffffffu));
}
// double -> two words, by the first of which and, where equal, the second it is ordered; the first is above 0 (numbers and
// infinities, no negative zero)
__device__ __forceinline__ uint32_t upper_ordered(double d) {
  const TwoWords w = __builtin_bit_cast(TwoWords, d);
  return (uint32_t)w.hi ^ ((uint32_t)(w.hi >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint32_t lower_ordered(double d) {
  const TwoWords w = __builtin_bit_cast(TwoWords, d);
  return (uint32_t)(w.lo ^ (w.hi >> 31));
}

// The logits of experts e0 .. e0 + R - 1 of a row; -infinity for a NaN and behind the end.  `vectors`: 16 bytes at a time lie
// aligned and whole in the row.
template <typename T, int R>
__device__ __forceinline__ void load_logits(const T* row, int e0, int E, bool vectors, float (&x)[R]) {
  constexpr int kVec = 16 / sizeof(T);
  typedef T vec_t __attribute__((ext_vector_type(kVec)));
  const float inf = __builtin_inff();
  if (R >= kVec && vectors) {
#pragma unroll
    for (int i = 0; i < R / kVec; ++i) {
      const int e = e0 + i * kVec;
      const vec_t v = *reinterpret_cast<const vec_t*>(row + (e < E ? e : 0));
#pragma unroll
      for (int j = 0; j < kVec; ++j) x[i * kVec + j] = e < E ? (float)v[j] : -inf;
    }
  } else {
#pragma unroll
    for (int r = 0; r < R; ++r) x[r] = (float)row[min(e0 + r, E - 1)];
#pragma unroll
    for (int r = 0; r < R; ++r) x[r] = e0 + r < E ? x[r] : -inf;
  }
#pragma unroll
  for (int r = 0; r < R; ++r) x[r] = x[r] == x[r] ? x[r] : -inf;
}

__device__ __forceinline__ float logit_at(const RouterParams& p, long at) {
  float f;
  if (p.dtype == SONAR_DTYPE_F32) f = ((const float*)p.logits)[at];
  else if (p.dtype == SONAR_DTYPE_BF16) f = (float)((const __bf16*)p.logits)[at];
  else f = (float)((const _Float16*)p.logits)[at];
  return f == f ? f : -__builtin_inff();
}

// e^-d for d >= 0 (also infinite): 2^n e^r with |r| <= ln(2) / 2, and the series of e^r to r^13, whose rest is below 2^-57.  The
// reduction is Cody and Waite's, with ln 2 in two parts, the first of so few bits that n times it is exact: those of fdlibm.
// The relative error grows with d, by 2^-53 for each of its units; that of a score by less, since e^-d falls faster.
__device__ __forceinline__ double exp_minus(double d) {
  const double t = -fmin(d, 800.0);
  const double n = __builtin_rint(t * 1.4426950408889634);
  const double r = __builtin_fma(-n, 1.9082149292705877e-10, __builtin_fma(-n, 0.6931471803691238, t));
  double e = 1.0 / 6227020800.0;
  e = __builtin_fma(e, r, 1.0 / 479001600.0);
  e = __builtin_fma(e, r, 1.0 / 39916800.0);
  e = __builtin_fma(e, r, 1.0 / 3628800.0);
  e = __builtin_fma(e, r, 1.0 / 362880.0);
  e = __builtin_fma(e, r, 1.0 / 40320.0);
  e = __builtin_fma(e, r, 1.0 / 5040.0);
  e = __builtin_fma(e, r, 1.0 / 720.0);
  e = __builtin_fma(e, r, 1.0 / 120.0);
  e = __builtin_fma(e, r, 1.0 / 24.0);
  e = __builtin_fma(e, r, 1.0 / 6.0);
  e = __builtin_fma(e, r, 0.5);
  e = __builtin_fma(e, r, 1.0);
  e = __builtin_fma(e, r, 1.0);
  return __builtin_ldexp(e, (int)n);
}
// 1 / x for x between 1 and 2^20: an estimate and two of Newton's steps
__device__ __forceinline__ double inverse(double x) {
  double y = __builtin_amdgcn_rcp(x);
  y = __builtin_fma(__builtin_fma(-x, y, 1.0), y, y);
  return __builtin_fma(__builtin_fma(-x, y, 1.0), y, y);
}
// e^(x - top), 0 for x = -infinity, 1 at the top (where both may be infinite)
__device__ __forceinline__ double term(float x, float top) {
  const double e = exp_minus((double)top - (double)x);
  return x == -__builtin_inff() ? 0.0 : x == top ? 1.0 : e;
}
__device__ __forceinline__ double sigmoid(float x) {
  const double e = exp_minus(fabs((double)x)), y = inverse(1.0 + e);
  return x >= 0 ? y : e * y;
}

// LANES of a wavefront a token, R experts a lane.
template <int LANES, int R, bool BIASED>
__global__ __launch_bounds__(64 * kWaves) void topk_routing_kernel(const RouterParams p, bool vectors) {
  constexpr int kTokens = 64 / LANES;
  __shared__ int chosen[kWaves][kTokens * kMaxTopk];
  extern __shared__ double all_choices[];   // [kWaves][kTokens][experts], of calls with groups
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l = lane % LANES, seg = lane / LANES, E = p.experts, e0 = l * R;
  const float inf = __builtin_inff();
  // 2^shift lanes a group, as many as there are; `in_lanes`: those hold just its experts
  const int size = E / p.groups, shift = 31 - __builtin_clz(LANES / p.groups);
  const bool in_lanes = size == R << shift;
  auto larger = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
  auto add = [](double a, double b) { return a + b; };
  const long first = ((long)blockIdx.x * kWaves + wave) * kTokens;
  if (first >= p.tokens) return;
  const long token = first + seg;
  const bool there = token < p.tokens;
  const long at = (there ? token : p.tokens - 1) * p.row_stride;
  float x[R];
  uint32_t key[R];   // of the choices
  if (p.dtype == SONAR_DTYPE_F32) load_logits((const float*)p.logits + at, e0, E, vectors, x);
  else if (p.dtype == SONAR_DTYPE_BF16) load_logits((const __bf16*)p.logits + at, e0, E, vectors, x);
  else load_logits((const _Float16*)p.logits + at, e0, E, vectors, x);
  const bool softmax = p.scoring == SONAR_SCORING_SOFTMAX;
  float top = 0;
  if (softmax) {
    uint32_t top_key = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) top_key = larger(top_key, ordered(x[r]));
    top = number_of(over_lanes<LANES>(top_key, larger));
  }
  double sum = 0;   // of a token's terms
  double choice[R];   // (with a bias; else x)
  if (BIASED) {
    if (softmax) {   // (branches outside the loops: the experts' chains of instructions side by side)
#pragma unroll
      for (int r = 0; r < R; ++r) sum += choice[r] = term(x[r], top);
      sum = over_lanes<LANES>(sum, add);
      if (sum > 0) {
        const double scale = inverse(sum);
#pragma unroll
        for (int r = 0; r < R; ++r) choice[r] *= scale;
      }
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r) choice[r] = sigmoid(x[r]);
    }
    float bias[R];
    load_logits(p.bias, e0, E, vectors, bias);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      choice[r] += (double)bias[r];   // (scores are 0 or above: no sum is a negative zero)
      if (choice[r] != choice[r]) choice[r] = -(double)inf;
      key[r] = upper_ordered(choice[r]);
    }
  } else {
#pragma unroll
    for (int r = 0; r < R; ++r) key[r] = ordered(x[r]);
    if (softmax && !p.renormalize) {   // (renormalised weights need no sum over all)
      float terms = 0;
#pragma unroll
      for (int r = 0; r < R; ++r) terms += x[r] == -inf ? 0.0f : x[r] == top ? 1.0f : __expf(x[r] - top);
      sum = over_lanes<LANES>((double)terms, add);
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) key[r] = e0 + r < E ? key[r] : 0;

  if (p.groups > 1) {
    const int g = l >> shift, share = 1 << shift;
    double best = -(double)inf, second = best;   // of the lane's share of its group
    auto count = [&](double c) {
      second = fmax(second, fmin(best, c));
      best = fmax(best, c);
    };
    if (in_lanes) {
#pragma unroll
      for (int r = 0; r < R; ++r) count(BIASED ? choice[r] : (double)x[r]);
    } else {
      double* choices = all_choices + (wave * kTokens + seg) * E;
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (e0 + r < E) choices[e0 + r] = BIASED ? choice[r] : (double)x[r];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if (g < p.groups)
        for (int j = l & (share - 1); j < size; j += share) count(choices[g * size + j]);
    }
    for (int step = 1; step < share; step <<= 1) {
      const double b = __shfl_xor(best, step, 64), s = __shfl_xor(second, step, 64);
      second = fmax(fmin(best, b), fmax(second, s));
      best = fmax(best, b);
    }
    if (BIASED && size > 1) best += second;
    if (best != best) best = -(double)inf;
    int rank = 0;   // groups before this one
#pragma unroll 4
    for (int other = 0; other < p.groups; ++other) {
      const double b = __shfl(best, seg * LANES + (other << shift), 64);
      rank += b > best || (b == best && other < g) ? 1 : 0;
    }
    const bool kept = g < p.groups && rank < p.kept_groups;
    if (in_lanes) {
#pragma unroll
      for (int r = 0; r < R; ++r) key[r] = kept ? key[r] : 0;
    } else {
      const unsigned long long open = __ballot(kept) >> (seg * LANES);
      const float per_group = 1.0f / (float)size;   // (e + 1 / 2) / size is 2^-11 from a whole number at least
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int of = (int)(((float)(e0 + r) + 0.5f) * per_group);
        if (!(open >> ((of << shift) & 63) & 1)) key[r] = 0;
      }
    }
  }

  uint32_t best;   // of this lane's experts, by the first word
  auto look = [&]() {
    best = key[0];
#pragma unroll
    for (int r = 1; r < R; ++r) best = larger(best, key[r]);
  };
  auto low = [&](int r) { return lower_ordered(choice[r]); };   // the second word
  auto low_of_best = [&]() {
    uint32_t most = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) most = larger(most, key[r] == best ? low(r) : 0);
    return most;
  };
  look();
  for (int k = 0; k < p.topk; ++k) {
    const uint32_t most = over_lanes<LANES>(best, larger);
    bool has = best == most;
    unsigned long long have = __ballot(has);
    if (BIASED && __popcll(have) != kTokens) {   // several lanes with the same first word
      const uint32_t mine_low = has ? low_of_best() : 0, rest = over_lanes<LANES>(mine_low, larger);
      has = has && mine_low == rest;
      have = __ballot(has);
    }
    bool mine;
    if (LANES == 64) mine = lane == __builtin_ctzll(have);
    else mine = l == __builtin_ctz((uint32_t)(have >> (seg * LANES)) | 0x80000000u);   // (a lane of the token has it: the lowest is the token's)
    if (mine) {
      bool seen = false, several = false;   // (lane masks: scalar instructions)
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const bool is = key[r] == best;
        several = several || (seen && is);
        seen = seen || is;
      }
      int at_r = 0;
      seen = false;
      if (BIASED && R > 1 && __ballot(several)) {   // several here with the same first word: by the second
        const uint32_t rest = low_of_best();
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const bool it = !seen && key[r] == best && low(r) == rest;
          at_r = it ? r : at_r;
          key[r] = it ? 0 : key[r];
          seen = seen || it;
        }
      } else {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const bool it = !seen && key[r] == best;
          at_r = it ? r : at_r;
          key[r] = it ? 0 : key[r];
          seen = seen || it;
        }
      }
      chosen[wave][seg * kMaxTopk + k] = e0 + at_r;
      look();
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  // the chosen scores, their sum if it divides them, then the weights; a choice a lane, and again from the first for more
  double total = 0, w = 0;
  int expert = 0;
  auto take = [&](int k) {
    expert = chosen[wave][seg * kMaxTopk + min(k, p.topk - 1)];
    const float logit = logit_at(p, at + expert);
    w = softmax ? term(logit, top) : sigmoid(logit);
    if (softmax && sum > 0) w /= sum;
  };
  const int end = (p.topk + LANES - 1) / LANES * LANES;
  if (p.renormalize)
    for (int k = l; k < end; k += LANES) {
      take(k);
      total += over_lanes<LANES>(k < p.topk ? w : 0.0, add);
    }
  const bool held = p.renormalize && end == LANES;
  for (int k = l; k < end; k += LANES) {
    if (!held) take(k);
    if (there && k < p.topk) {
      if (total > 0) w /= total;
      p.weights[token * p.topk + k] = (float)(w * p.factor);
      p.ids[token * p.topk + k] = expert;
    }
  }
}

template <int LANES, int R, bool BIASED>
void launch(const RouterParams& p, hipStream_t st) {
  const long size = p.dtype == SONAR_DTYPE_F32 ? 4 : 2;
  const bool vectors = (uintptr_t)p.logits % 16 == 0 && p.row_stride * size % 16 == 0 && p.experts * size % 16 == 0 &&
                       (uintptr_t)p.bias % 16 == 0;   // (experts: a multiple of four, whole vectors of the bias too)
  const bool in_lanes = p.experts / p.groups == R << (31 - __builtin_clz(LANES / p.groups));   // (as the kernel)
  const size_t lds = p.groups > 1 && !in_lanes ? (size_t)kWaves * (64 / LANES) * p.experts * sizeof(double) : 0;
  const long most = (1L << 20) * kWaves * (64 / LANES);   // tokens of a launch: a loop in the kernel would keep its constants in registers
  for (long from = 0; from < p.tokens; from += most) {
    RouterParams q = p;
    q.tokens = p.tokens - from < most ? p.tokens - from : most;
    q.logits = (const char*)p.logits + from * p.row_stride * size;
    q.weights += from * p.topk, q.ids += from * p.topk;
    const int grid = (int)((q.tokens + kWaves * (64 / LANES) - 1) / (kWaves * (64 / LANES)));
    topk_routing_kernel<LANES, R, BIASED><<<grid, 64 * kWaves, lds, st>>>(q, vectors);
  }
}

// Few tokens: a wavefront each, for its latency.  From 4096 on, where every SIMD has some, several share one (8192 x 128, top 8:
// 5.3 us, 9.3 with a wavefront each; 2048 x 256 4.6 and, shared, 6.6).  With a bias and more than 128 experts two instead of
// four (4096 x 256, sigmoid, 4 of 8 groups: 8.8 us, 10.6 with four; without a bias, 16384 x 256: 12.0 with two, 11.3 with four).
template <bool BIASED>
void launch_form(const RouterParams& p, hipStream_t st) {
  const bool many = p.tokens >= 4096;
  if (p.experts <= 8 && p.groups <= 8) return launch<8, 1, BIASED>(p, st);
  if (many && p.experts <= 32 && p.groups <= 8) return launch<8, 4, BIASED>(p, st);
  if (many && p.experts <= 64 && p.groups <= 16) return launch<16, 4, BIASED>(p, st);
  if (many && p.experts <= 128 && p.groups <= 16) return launch<16, 8, BIASED>(p, st);
  if constexpr (BIASED) {
    if (many && p.experts <= 256 && p.groups <= 32) return launch<32, 8, true>(p, st);
  } else {
    if (many && p.experts <= 256 && p.groups <= 16) return launch<16, 16, false>(p, st);
  }
  if (p.experts <= 64) return launch<64, 1, BIASED>(p, st);
  if (p.experts <= 256) return launch<64, 4, BIASED>(p, st);
  launch<64, 16, BIASED>(p, st);
}

}  // namespace
}  // namespace sonar

using namespace sonar;

extern "C" int sonar_topk_routing(const void* logits, int dtype, int64_t row_stride, const float* bias, float* weights,
                                  int32_t* ids, int64_t tokens, int64_t experts, int64_t topk, int scoring, int renormalize,
                                  int64_t groups, int64_t kept_groups, double factor, void* stream) {
  SONAR_REQUIRE(tokens >= 0 && tokens < (1LL << 31), "tokens = %ld", (long)tokens);
  SONAR_REQUIRE(experts >= 1 && experts <= kMaxExperts, "experts = %ld: 1 to %d are built", (long)experts, kMaxExperts);
  SONAR_REQUIRE(groups >= 1 && groups <= kMaxGroups && experts % groups == 0,
                "groups = %ld must divide experts = %ld and be at most %d", (long)groups, (long)experts, kMaxGroups);
  SONAR_REQUIRE(kept_groups >= 1 && kept_groups <= groups, "kept_groups = %ld of %ld groups", (long)kept_groups, (long)groups);
  SONAR_REQUIRE(topk >= 1 && topk <= kMaxTopk && topk <= kept_groups * (experts / groups),
                "topk = %ld: 1 to %d, and no more than the %ld experts of the kept groups, can be chosen", (long)topk, kMaxTopk,
                (long)(kept_groups * (experts / groups)));
  SONAR_REQUIRE(scoring == SONAR_SCORING_SOFTMAX || scoring == SONAR_SCORING_SIGMOID, "unknown scoring = %d", scoring);
  SONAR_REQUIRE(row_stride >= experts, "row_stride = %ld is smaller than experts = %ld", (long)row_stride, (long)experts);
  SONAR_REQUIRE(dtype == SONAR_DTYPE_F16 || dtype == SONAR_DTYPE_BF16 || dtype == SONAR_DTYPE_F32, "unknown dtype = %d", dtype);
  if (tokens == 0) return SONAR_OK;
  SONAR_REQUIRE(logits && weights && ids, "logits, weights and ids must not be NULL");
  const RouterParams p{logits, row_stride,   bias,         weights,     ids,         tokens,          dtype, (int)experts,
                       (int)topk, scoring,   renormalize,  (int)groups, (int)kept_groups, factor};
  hipStream_t st = (hipStream_t)stream;
  if (bias != nullptr) launch_form<true>(p, st);
  else launch_form<false>(p, st);
  return launch_status("topk_routing_kernel");
}
