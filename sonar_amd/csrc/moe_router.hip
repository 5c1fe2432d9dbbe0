// The experts of each token and their weights, from the router's logits x:
//   s = softmax(x) or 1 / (1 + exp(-x));  c = s + bias, or x itself, which has the order of s, without a bias
//   ids: the topk largest c, of the experts in the best groups where there are groups;  weights: s of them
// Equal choices go to the lowest expert.  What decides, s + bias and the groups' sums, is taken in 64 bits: two experts whose
// float32 sums are equal are told apart, as a 64-bit program would.
//
// A choice is kept as two words whose unsigned order is that of the numbers: its float32 rounding and what that leaves (no
// second word without a bias).  Every round finds the largest first word over a token's lanes by lane moves, asks which
// lanes have it, looks at the second words only if there are several, and takes the lowest.  Word 0 is below every number's:
// an expert that is taken, left out or not there.
// Bound by the vector instructions of the rounds and, with a bias, of the 64-bit exponentials.
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

// A number no NaN: a NaN counts as -infinity
__device__ __forceinline__ float logit_at(const RouterParams& p, long at) {
  float f;
  if (p.dtype == SONAR_DTYPE_F32) f = ((const float*)p.logits)[at];
  else if (p.dtype == SONAR_DTYPE_BF16) f = (float)((const __bf16*)p.logits)[at];
  else f = (float)((const _Float16*)p.logits)[at];
  return f == f ? f : -__builtin_inff();
}

// e^(x - top), 0 for x = -infinity, 1 at the top (where both may be infinite)
__device__ __forceinline__ double term(float x, float top) {
  return x == -__builtin_inff() ? 0.0 : x == top ? 1.0 : exp((double)x - (double)top);
}
__device__ __forceinline__ double sigmoid(float x) { return 1.0 / (1.0 + exp(-(double)x)); }

// LANES of a wavefront a token, R experts a lane: experts lane, lane + LANES, ..  R = 1 below 64 lanes.
template <int LANES, int R, bool BIASED>
__global__ __launch_bounds__(64 * kWaves) void topk_routing_kernel(const RouterParams p) {
  static_assert(R == 1 || LANES == 64, "");
  constexpr int kTokens = 64 / LANES;
  struct Chosen {
    double value;   // the logit, or with a bias the score
    int expert;
  };
  __shared__ Chosen chosen[kWaves][64];
  extern __shared__ double all_choices[];   // [kWaves][experts], of calls with groups
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l = lane % LANES, seg = lane / LANES, E = p.experts;
  const float inf = __builtin_inff();
  auto larger = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
  auto add = [](double a, double b) { return a + b; };
  for (long first = ((long)blockIdx.x * kWaves + wave) * kTokens; first < p.tokens; first += (long)gridDim.x * kWaves * kTokens) {
    const long token = first + seg;
    const bool there = token < p.tokens;
    float x[R];
    uint32_t key[R], low[R];   // of the choices
    double score[R];
    uint32_t top_key = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int e = r * LANES + l;
      x[r] = there && e < E ? logit_at(p, token * p.row_stride + e) : -inf;
      top_key = larger(top_key, ordered(x[r]));
    }
    const bool softmax = p.scoring == SONAR_SCORING_SOFTMAX;
    float top = 0;
    if (softmax) top = number_of(over_lanes<LANES>(top_key, larger));
    double sum = 0;   // of a token's terms
    if (BIASED) {
#pragma unroll
      for (int r = 0; r < R; ++r) sum += score[r] = softmax ? term(x[r], top) : sigmoid(x[r]);
      if (softmax) sum = over_lanes<LANES>(sum, add);
    } else if (softmax && !p.renormalize) {   // (renormalised weights need no sum over all)
      float terms = 0;
#pragma unroll
      for (int r = 0; r < R; ++r) terms += x[r] == -inf ? 0.0f : x[r] == top ? 1.0f : __expf(x[r] - top);
      sum = over_lanes<LANES>((double)terms, add);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int e = r * LANES + l;
      key[r] = low[r] = 0;
      double choice = (double)x[r];
      if (BIASED) {
        if (softmax && sum > 0) score[r] /= sum;
        choice = e < E ? score[r] + (double)p.bias[e] : 0.0;
        if (choice != choice) choice = -(double)inf;
        const float near = (float)choice, rest = (float)(choice - (double)near);
        if (there && e < E) key[r] = ordered(near), low[r] = rest == rest ? ordered(rest) : ordered(0.0f);
      } else if (there && e < E) {
        key[r] = ordered(x[r]);
      }
      if (LANES == 64 && p.groups > 1 && e < E) all_choices[wave * E + e] = choice;
    }

    if (LANES == 64 && p.groups > 1) {
      // 2^n lanes a group, as many as there are: the two largest choices of each, a lane's share first
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      const int size = E / p.groups, shift = 31 - __builtin_clz(64 / p.groups), g = lane >> shift, share = 1 << shift;
      double best = -(double)inf, second = best;
      if (g < p.groups)
        for (int j = lane & (share - 1); j < size; j += share) {
          const double c = all_choices[wave * E + g * size + j];
          second = fmax(second, fmin(best, c));
          best = fmax(best, c);
        }
      for (int step = 1; step < share; step <<= 1) {
        const double b = __shfl_xor(best, step, 64), s = __shfl_xor(second, step, 64);
        second = fmax(fmin(best, b), fmax(second, s));
        best = fmax(best, b);
      }
      if (BIASED && size > 1) best += second;
      if (best != best) best = -(double)inf;
      int rank = 0;   // groups before this one
      for (int other = 0; other < p.groups; ++other) {
        const double b = of_lane(best, other << shift);
        rank += b > best || (b == best && other < g) ? 1 : 0;
      }
      const unsigned long long open = __ballot(g < p.groups && rank < p.kept_groups);
      const float per_group = 1.0f / (float)size;   // (e + 1 / 2) / size is 2^-11 from a whole number at least
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int of = (int)(((float)(r * LANES + l) + 0.5f) * per_group);
        if (!(open >> ((of << shift) & 63) & 1)) key[r] = 0;
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }

    for (int k = 0; k < p.topk; ++k) {
      uint32_t best = key[0];
#pragma unroll
      for (int r = 1; r < R; ++r) best = larger(best, key[r]);
      best = over_lanes<LANES>(best, larger);
      unsigned long long have[R];
#pragma unroll
      for (int r = 0; r < R; ++r) have[r] = __ballot(key[r] == best);
      if (BIASED) {
        int count = 0;
#pragma unroll
        for (int r = 0; r < R; ++r) count += __popcll(have[r]);
        if (count != kTokens) {   // several with the same float32 number
          uint32_t rest = 0;
#pragma unroll
          for (int r = 0; r < R; ++r) rest = larger(rest, key[r] == best ? low[r] : 0);
          rest = over_lanes<LANES>(rest, larger);
#pragma unroll
          for (int r = 0; r < R; ++r) have[r] = __ballot(key[r] == best && low[r] == rest);
        }
      }
      auto take = [&](int r) {
        key[r] = 0;
        chosen[wave][seg * LANES + k] = Chosen{BIASED ? score[r] : (double)x[r], r * LANES + l};
      };
      if (LANES < 64) {
        const uint32_t mine = (uint32_t)(have[0] >> (seg * LANES));   // (a lane of the token has it, so the lowest one is of the token)
        if (l == __builtin_ctz(mine | 0x80000000u)) take(0);
      } else {
        bool found = false;
#pragma unroll
        for (int r = 0; r < R; ++r)
          if (!found && have[r] != 0) {
            found = true;
            if (lane == __builtin_ctzll(have[r])) take(r);
          }
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    double w = 0;
    int expert = 0;
    if (l < p.topk) {
      const Chosen c = chosen[wave][seg * LANES + l];
      expert = c.expert;
      w = c.value;
      if (!BIASED) {
        w = softmax ? term((float)c.value, top) : sigmoid((float)c.value);
        if (softmax && sum > 0) w /= sum;
      }
    }
    if (p.renormalize) {
      const double total = over_lanes<LANES>(w, add);
      if (total > 0) w /= total;
    }
    if (there && l < p.topk) {
      p.weights[token * p.topk + l] = (float)(w * p.factor);
      p.ids[token * p.topk + l] = expert;
    }
  }
}

template <int LANES, int R>
void launch(const RouterParams& p, hipStream_t st) {
  const long waves = (p.tokens + 64 / LANES - 1) / (64 / LANES), groups = (waves + kWaves - 1) / kWaves;
  const int grid = (int)(groups < (1 << 20) ? groups : 1 << 20);
  const size_t lds = p.groups > 1 ? (size_t)kWaves * p.experts * sizeof(double) : 0;
  if (p.bias != nullptr) topk_routing_kernel<LANES, R, true><<<grid, 64 * kWaves, lds, st>>>(p);
  else topk_routing_kernel<LANES, R, false><<<grid, 64 * kWaves, lds, st>>>(p);
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
  if (groups == 1 && experts <= 8) launch<8, 1>(p, st);
  else if (groups == 1 && experts <= 16) launch<16, 1>(p, st);
  else if (groups == 1 && experts <= 32) launch<32, 1>(p, st);
  else if (experts <= 64) launch<64, 1>(p, st);
  else if (experts <= 128) launch<64, 2>(p, st);
  else if (experts <= 256) launch<64, 4>(p, st);
  else if (experts <= 512) launch<64, 8>(p, st);
  else launch<64, 16>(p, st);
  return launch_status("topk_routing_kernel");
}
