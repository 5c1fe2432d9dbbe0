// The experts of each token and their weights from the router's logits.
#include "common.hpp"
#include "sonar_layer.h"

namespace sonar {
namespace {

constexpr int kMaxExperts = 1024, kMaxGroups = 64, kMaxTopk = 64;

struct RouterParams {
  const void* logits;
  long row_stride;
  const float* bias;
  float* weights;
  int32_t* ids;
  int tokens, experts, topk, scoring, renormalize, groups, kept_groups;
  float factor;
};

__device__ __forceinline__ bool before(double a, int ai, double b, int bi) { return a > b || (a == b && ai < bi); }

__device__ __forceinline__ void best_of_wave(double& v, int& i) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const double w = __shfl_xor(v, off, 64);
    const int j = __shfl_xor(i, off, 64);
    if (before(w, j, v, i)) v = w, i = j;
  }
}

// One wavefront a token; the choices and scores of a token stand in LDS.
template <typename T>
__global__ __launch_bounds__(64) void topk_routing_kernel(const RouterParams p) {
  __shared__ double choice[kMaxExperts], score[kMaxExperts];
  const int lane = threadIdx.x, E = p.experts;
  const long token = blockIdx.x;
  const T* x = (const T*)p.logits + token * p.row_stride;
  const double inf = __builtin_inf();
  double top = -inf;
  for (int e = lane; e < E; e += 64) {
    double v = (double)(float)x[e];
    if (v != v) v = -inf;
    choice[e] = v;
    top = fmax(top, v);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) top = fmax(top, __shfl_xor(top, off, 64));
  double sum = 0;
  for (int e = lane; e < E; e += 64) {
    const double v = choice[e];
    const double s = p.scoring == SONAR_SCORING_SIGMOID ? 1.0 / (1.0 + exp(-v)) : v == -inf ? 0.0 : v == top ? 1.0 : exp(v - top);
    score[e] = s;
    sum += s;
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
  for (int e = lane; e < E; e += 64) {
    if (p.scoring == SONAR_SCORING_SOFTMAX && sum > 0) score[e] /= sum;
    if (p.bias != nullptr) {
      const double c = score[e] + (double)p.bias[e];
      choice[e] = c != c ? -inf : c;
    }
  }
  __syncthreads();
  unsigned long long open = ~0ull;   // groups whose experts may be chosen
  const int size = E / p.groups;
  if (p.groups > 1) {
    double first = -inf, second = -inf;
    if (lane < p.groups)
      for (int j = 0; j < size; ++j) {
        const double c = choice[lane * size + j];
        if (c > first) second = first, first = c;
        else if (c > second) second = c;
      }
    double of_group = p.bias == nullptr || size == 1 ? first : first + second;
    if (of_group != of_group) of_group = -inf;
    open = 0;
    for (int k = 0; k < p.kept_groups; ++k) {
      double v = of_group;
      int i = lane < p.groups && !(open >> lane & 1) ? lane : 64 + lane;
      if (i >= 64) v = -inf;
      best_of_wave(v, i);
      open |= 1ull << (i & 63);
    }
  }
  double mine = 0, total = 0;   // lane k: the score of choice k
  int my_id = 0;
  unsigned int used = 0;        // of this lane's experts lane, lane + 64, ..
  for (int k = 0; k < p.topk; ++k) {
    double v = -inf;
    int i = 1 << 20;
    for (int e = lane, r = 0; e < E; e += 64, ++r)
      if (!(used >> r & 1) && (p.groups == 1 || (open >> (e / size) & 1)) && before(choice[e], e, v, i)) v = choice[e], i = e;
    best_of_wave(v, i);
    if ((i & 63) == lane) used |= 1u << (i >> 6);
    const double s = score[i];
    if (lane == k) mine = s, my_id = i;
    total += s;
  }
  if (lane < p.topk) {
    if (p.renormalize && total > 0) mine /= total;
    p.weights[token * p.topk + lane] = (float)(mine * (double)p.factor);
    p.ids[token * p.topk + lane] = my_id;
  }
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
  const RouterParams p{logits,   row_stride,   bias,          weights,     ids,
                       (int)tokens, (int)experts, (int)topk,     scoring,     renormalize,
                       (int)groups, (int)kept_groups, (float)factor};
  hipStream_t st = (hipStream_t)stream;
  if (dtype == SONAR_DTYPE_F16) topk_routing_kernel<_Float16><<<(int)tokens, 64, 0, st>>>(p);
  else if (dtype == SONAR_DTYPE_BF16) topk_routing_kernel<__bf16><<<(int)tokens, 64, 0, st>>>(p);
  else topk_routing_kernel<float><<<(int)tokens, 64, 0, st>>>(p);
  return launch_status("topk_routing_kernel");
}
