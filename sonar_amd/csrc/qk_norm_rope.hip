// Norms and position rotation of the query and key heads of each token, the keys and values put into the pages of a cache:
//   y = x * r * weight, r = 1 / sqrt(mean(x^2) + epsilon);  pairs (a, b) of y -> (a cos - b sin, b cos + a sin)
// in float32, rounded once at the end.  One pass over memory, bound by the bytes: a head is read once, into the lanes that
// hold both numbers of every pair, and written where it belongs.
#include "common.hpp"
#include "lane_reduce.hpp"
#include "sonar_attention.h"

namespace sonar {
namespace {
thread_local char g_attention_error[512] = "";
}  // namespace
char* last_error_buffer() { return g_attention_error; }

namespace {

constexpr int kThreads = 256;   // of a workgroup
constexpr int kAhead = 4;       // heads that a thread reads before it works on the first

struct Pages {
  char* data;
  long page, slot, head;   // strides, in elements
  const float* scale;
  int scale_heads;         // scale holds one number a head
};

struct RopeParams {
  const void *q, *k, *v;
  long q_token, q_head, k_token, k_head, v_token, v_head;
  const void* positions;
  const float* table;
  long max_position;
  const void *q_weight, *k_weight;
  void *q_out, *k_out;
  Pages keys, values;
  const void* slots;
  long all_slots, tokens;
  float inverse_dim, epsilon;
  int rotary, page_size, heads, kv_heads, dim;
  int lanes, of_token;     // lanes of a head, heads of a token that a workgroup takes at once
  bool half, positions_64, slots_64, cached, fp8;
};

__device__ __forceinline__ long index_at(const void* p, long i, bool is_64) {
  return is_64 ? ((const int64_t*)p)[i] : (long)((const int32_t*)p)[i];
}

// A cache line of a token: the elements before its heads, or -1 where its slot is none.
__device__ __forceinline__ bool place_of(const RopeParams& p, long token, long& page, long& slot) {
  const long at = index_at(p.slots, token, p.slots_64);
  if (at < 0 || at >= p.all_slots) return false;
  if (p.all_slots <= 0x7fffffffL) {
    page = (uint32_t)at / (uint32_t)p.page_size, slot = (uint32_t)at % (uint32_t)p.page_size;
  } else {
    page = at / p.page_size, slot = at % p.page_size;
  }
  return true;
}

// The nearest float8_e4m3fn of y / scale; a NaN stays one.
__device__ __forceinline__ float fp8_number(float y, float inverse) {
  return __builtin_elementwise_minimum(__builtin_elementwise_maximum(y * inverse, -448.0f), 448.0f);
}
__device__ __forceinline__ float inverse_scale(const Pages& c, int head) { return 1.0f / c.scale[c.scale_heads ? head : 0]; }

// (a launch has fewer than 2^32 threads a dimension)
__device__ __forceinline__ long block_number() { return (long)blockIdx.y * gridDim.x + blockIdx.x; }
dim3 grid_of(long blocks) {
  const long rows = (blocks + (1 << 23) - 1) >> 23;
  return dim3((uint32_t)((blocks + rows - 1) / rows), (uint32_t)rows);
}

// Sum over `lanes` neighbouring lanes (a power of two, 4 at least), in every lane.
__device__ __forceinline__ float sum_over(float v, int lanes) {
  auto moved_by = [](float x, auto ctrl) {
    return __builtin_bit_cast(float, exchanged<decltype(ctrl)::value>(__builtin_bit_cast(uint32_t, x)));
  };
  v += moved_by(v, std::integral_constant<int, 0xB1>{});
  v += moved_by(v, std::integral_constant<int, 0x4E>{});
  if (lanes >= 8) v += moved_by(v, std::integral_constant<int, 0x141>{});
  if (lanes >= 16) v += moved_by(v, std::integral_constant<int, 0x140>{});
  uint32_t one, other;
  if (lanes >= 32) {
    sides<false>(__builtin_bit_cast(uint32_t, v), one, other);
    v = __builtin_bit_cast(float, one) + __builtin_bit_cast(float, other);
  }
  if (lanes >= 64) {
    sides<true>(__builtin_bit_cast(uint32_t, v), one, other);
    v = __builtin_bit_cast(float, one) + __builtin_bit_cast(float, other);
  }
  return v;
}

// VEC neighbouring numbers.
template <typename T, int VEC>
struct Vec {
  typedef T vec __attribute__((ext_vector_type(VEC), aligned(VEC * sizeof(T) < 16 ? VEC * sizeof(T) : 16)));
  vec v;
  __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const vec*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<vec*>(p) = v; }
};

template <int VEC>
__device__ __forceinline__ void store_fp8(char* to, const float (&y)[VEC], float inverse) {
  uint32_t words[(VEC + 3) / 4];
#pragma unroll
  for (int w = 0; w < (VEC + 3) / 4; ++w) {
    const int low = __builtin_amdgcn_cvt_pk_fp8_f32(fp8_number(y[4 * w], inverse), fp8_number(y[4 * w + 1], inverse), 0, false);
    if constexpr (VEC >= 4)
      words[w] = __builtin_amdgcn_cvt_pk_fp8_f32(fp8_number(y[4 * w + 2], inverse), fp8_number(y[4 * w + 3], inverse), low, true);
    else
      words[w] = low;
  }
  if constexpr (VEC == 8) *reinterpret_cast<uint2*>(to) = make_uint2(words[0], words[1]);
  else if constexpr (VEC == 4) *reinterpret_cast<uint32_t*>(to) = words[0];
  else *reinterpret_cast<uint16_t*>(to) = (uint16_t)words[0];
}

// `lanes` lanes a head, two runs of VEC numbers a lane: of the rotated numbers those of VEC whole pairs (run i of either half,
// or runs 2i and 2i + 1), behind them two neighbouring runs.  A thread keeps its part of the cosines, sines and weights for all
// heads of its token that it takes.
// 16384 tokens of 40 heads of 128 in bf16 with norms take 72 us, 4.7 TB/s, what a large copy reaches; the append of 5000 tokens to an 8-bit cache
// 27 us, 4.2 TB/s.  (128 registers for four wavefronts a SIMD: 73 us for the 77 with 132; eight numbers of 32 bits would spill there)
template <typename T, int VEC>
__global__ __launch_bounds__(kThreads, VEC * sizeof(T) > 16 ? 3 : 4) void qk_norm_rope_kernel(const RopeParams p) {
#pragma clang fp contract(off)
  const int slot = threadIdx.x / p.lanes, j = threadIdx.x % p.lanes;
  const int tokens_here = kThreads / p.lanes / p.of_token;
  const long token = block_number() * tokens_here + slot / p.of_token;
  if (token >= p.tokens) return;
  const int turned = p.rotary / (2 * VEC);
  const bool turns = j < turned;
  const int a = turns ? (p.half ? VEC * j : 2 * VEC * j) : p.rotary + 2 * VEC * (j - turned);
  const int b = turns && p.half ? p.rotary / 2 + VEC * j : a + VEC;
  const bool has_a = a < p.dim, has_b = b < p.dim;
  const int all = p.heads + (p.cached ? 2 : 1) * p.kv_heads;

  long page = 0, place = 0;
  const bool kept = p.cached && place_of(p, token, page, place);
  Vec<float, VEC> cos, sin;
  if (turns && p.table != nullptr) {
    const long position = index_at(p.positions, token, p.positions_64);
    if (position >= 0 && position < p.max_position) {
      const float* row = p.table + position * p.rotary + VEC * j;
      cos.load(row), sin.load(row + p.rotary / 2);
    } else {
      cos.v = __builtin_nanf(""), sin.v = __builtin_nanf("");
    }
  }
  Vec<T, VEC> q_weight[2], k_weight[2];
  if (p.q_weight != nullptr) {
    if (has_a) q_weight[0].load((const T*)p.q_weight + a);
    if (has_b) q_weight[1].load((const T*)p.q_weight + b);
  }
  if (p.k_weight != nullptr) {
    if (has_a) k_weight[0].load((const T*)p.k_weight + a);
    if (has_b) k_weight[1].load((const T*)p.k_weight + b);
  }

  for (int first = slot % p.of_token; first < all; first += kAhead * p.of_token) {
    Vec<T, VEC> x[kAhead][2];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int h = first + u * p.of_token;
      if (h >= all) break;
      const T* from = h < p.heads ? (const T*)p.q + token * p.q_token + h * p.q_head
                      : h < p.heads + p.kv_heads ? (const T*)p.k + token * p.k_token + (h - p.heads) * p.k_head
                                                 : (const T*)p.v + token * p.v_token + (h - p.heads - p.kv_heads) * p.v_head;
      if (has_a) x[u][0].load(from + a);
      if (has_b) x[u][1].load(from + b);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int h = first + u * p.of_token;
      if (h >= all) break;
      const bool query = h < p.heads, value = h >= p.heads + p.kv_heads;
      float y[2][VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) y[0][e] = has_a ? (float)x[u][0].v[e] : 0.0f, y[1][e] = has_b ? (float)x[u][1].v[e] : 0.0f;
      if (!value) {
        if ((query ? p.q_weight : p.k_weight) != nullptr) {
          float sum = 0.0f;
#pragma unroll
          for (int e = 0; e < VEC; ++e) sum = __builtin_fmaf(y[0][e], y[0][e], __builtin_fmaf(y[1][e], y[1][e], sum));
          const float r = 1.0f / __builtin_sqrtf(__builtin_fmaf(sum_over(sum, p.lanes), p.inverse_dim, p.epsilon));
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            y[0][e] = y[0][e] * r * (float)(query ? q_weight[0].v[e] : k_weight[0].v[e]);
            y[1][e] = y[1][e] * r * (float)(query ? q_weight[1].v[e] : k_weight[1].v[e]);
          }
        }
        if (turns && p.table != nullptr) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            // pair e: number e of either run, or numbers 2e and 2e + 1 of both runs in a row
            if (p.half) {
              const float s = y[0][e], t = y[1][e];
              y[0][e] = __builtin_fmaf(s, cos.v[e], -(t * sin.v[e])), y[1][e] = __builtin_fmaf(t, cos.v[e], s * sin.v[e]);
            } else {
              float &s = y[2 * e / VEC][2 * e % VEC], &t = y[2 * e / VEC][2 * e % VEC + 1];
              const float old = s;
              s = __builtin_fmaf(old, cos.v[e], -(t * sin.v[e])), t = __builtin_fmaf(t, cos.v[e], old * sin.v[e]);
            }
          }
        }
      }
      if (query || !p.cached) {
        T* to = query ? (T*)p.q_out + (token * p.heads + h) * p.dim : (T*)p.k_out + (token * p.kv_heads + h - p.heads) * p.dim;
        Vec<T, VEC> out;
#pragma unroll
        for (int run = 0; run < 2; ++run)
          if (run == 0 ? has_a : has_b) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) out.v[e] = (T)y[run][e];
            out.store(to + (run == 0 ? a : b));
          }
      } else if (kept) {
        const Pages& c = value ? p.values : p.keys;
        const int head = h - p.heads - (value ? p.kv_heads : 0);
        const long at = page * c.page + place * c.slot + head * c.head;
        const float inverse = p.fp8 ? inverse_scale(c, head) : 1.0f;
#pragma unroll
        for (int run = 0; run < 2; ++run)
          if (run == 0 ? has_a : has_b) {
            const long d = at + (run == 0 ? a : b);
            if (p.fp8) {
              store_fp8<VEC>(c.data + d, y[run], inverse);
            } else {
              Vec<T, VEC> out;
#pragma unroll
              for (int e = 0; e < VEC; ++e) out.v[e] = (T)y[run][e];
              out.store((T*)c.data + d);
            }
          }
      }
    }
  }
}

// Any head_dim, rotary_dim, stride and alignment: a wavefront a head, number by number, the head read again after its norm.  Bound by
// the instructions a number and half-empty lines, not by memory: 16384 tokens of 40 heads of 127 360 us, of 128 in the form above 71.
template <typename T>
__global__ __launch_bounds__(kThreads) void qk_norm_rope_any_kernel(const RopeParams p) {
#pragma clang fp contract(off)
  const int lane = threadIdx.x & 63, all = p.heads + (p.cached ? 2 : 1) * p.kv_heads;
  const long item = block_number() * (kThreads / 64) + threadIdx.x / 64;
  if (item >= p.tokens * all) return;
  const long token = item / all;
  const int h = item % all;
  const bool query = h < p.heads, value = h >= p.heads + p.kv_heads;
  const int head = query ? h : h - p.heads - (value ? p.kv_heads : 0);
  const T* x = query ? (const T*)p.q + token * p.q_token + head * p.q_head
               : value ? (const T*)p.v + token * p.v_token + head * p.v_head : (const T*)p.k + token * p.k_token + head * p.k_head;
  const T* weight = value ? nullptr : (const T*)(query ? p.q_weight : p.k_weight);
  float r = 1.0f;
  if (weight != nullptr) {
    float sum = 0.0f;
    for (int d = lane; d < p.dim; d += 64) sum = __builtin_fmaf((float)x[d], (float)x[d], sum);
    r = 1.0f / __builtin_sqrtf(__builtin_fmaf(wave_sum(sum), p.inverse_dim, p.epsilon));
  }
  long page = 0, place = 0;
  if (!query && p.cached && !place_of(p, token, page, place)) return;
  const Pages& c = value ? p.values : p.keys;
  const long at = !query && p.cached ? page * c.page + place * c.slot + head * c.head : 0;
  const float inverse = !query && p.cached && p.fp8 ? inverse_scale(c, head) : 1.0f;
  auto number = [&](int d) { return weight != nullptr ? (float)x[d] * r * (float)weight[d] : (float)x[d]; };
  auto put = [&](int d, float y) {
    if (query) ((T*)p.q_out)[(token * p.heads + head) * p.dim + d] = (T)y;
    else if (!p.cached) ((T*)p.k_out)[(token * p.kv_heads + head) * p.dim + d] = (T)y;
    else if (p.fp8) c.data[at + d] = (char)(__builtin_amdgcn_cvt_pk_fp8_f32(fp8_number(y, inverse), 0.0f, 0, false) & 0xff);
    else ((T*)c.data)[at + d] = (T)y;
  };
  const int turned = value || p.table == nullptr ? 0 : p.rotary;
  if (turned > 0) {
    const long position = index_at(p.positions, token, p.positions_64);
    const bool known = position >= 0 && position < p.max_position;
    const float* row = p.table + (known ? position : 0) * p.rotary;
    for (int i = lane; i < turned / 2; i += 64) {
      const int first = p.half ? i : 2 * i, second = p.half ? turned / 2 + i : 2 * i + 1;
      const float s = number(first), t = number(second);
      const float cos = known ? row[i] : __builtin_nanf(""), sin = known ? row[turned / 2 + i] : __builtin_nanf("");
      put(first, __builtin_fmaf(s, cos, -(t * sin)));
      put(second, __builtin_fmaf(t, cos, s * sin));
    }
  }
  for (int d = turned + lane; d < p.dim; d += 64) put(d, number(d));
}

// Whether runs of `vec` numbers fit everything: the rows' widths, strides and addresses.
bool runs_fit(const RopeParams& p, int vec, int size) {
  long strides = p.dim | p.q_token | p.q_head | p.k_token | p.k_head | p.v_token | p.v_head;
  const long bytes = vec * size < 16 ? vec * size : 16;
  auto at = [](const void* q) { return (long)(uintptr_t)q; };
  long places = at(p.q) | at(p.k) | at(p.v) | at(p.q_out) | at(p.k_out) | at(p.q_weight) | at(p.k_weight);
  if (p.cached) {
    strides |= p.keys.page | p.keys.slot | p.keys.head | p.values.page | p.values.slot | p.values.head;
    const long caches = at(p.keys.data) | at(p.values.data);
    if (caches % (p.fp8 ? vec : bytes) != 0) return false;
  }
  return strides % vec == 0 && places % bytes == 0 && (p.table == nullptr || (p.rotary % (2 * vec) == 0 && at(p.table) % (vec < 4 ? 8 : 16) == 0));
}

template <typename T, int VEC>
int launch_runs(RopeParams p, hipStream_t st) {
  const int runs = (p.rotary / (2 * VEC)) + (p.dim - p.rotary + 2 * VEC - 1) / (2 * VEC);
  p.lanes = 4;
  while (p.lanes < runs) p.lanes *= 2;
  const int slots = kThreads / p.lanes, all = p.heads + (p.cached ? 2 : 1) * p.kv_heads;
  p.of_token = slots;
  while (p.of_token > 1 && p.of_token / 2 >= all) p.of_token /= 2;
  // Four heads or more a thread, which then reads that many at once and its cosines, sines and weights once for them, while there are
  // threads enough: 16384 tokens of 40 heads of 128 with norms 77 us, a head or two a thread 111; 4096 20.4 and 24.3.
  while (p.of_token > 1 && all / p.of_token < kAhead && p.tokens * (p.of_token / 2) * p.lanes >= 262144) p.of_token /= 2;
  const int tokens_here = slots / p.of_token;
  qk_norm_rope_kernel<T, VEC><<<grid_of((p.tokens + tokens_here - 1) / tokens_here), kThreads, 0, st>>>(p);
  return launch_status("qk_norm_rope_kernel");
}

template <typename T>
int launch(RopeParams p, hipStream_t st) {
  if (p.table == nullptr) p.rotary = 0;
  if (runs_fit(p, 8, sizeof(T)) && p.dim <= 1024) return launch_runs<T, 8>(p, st);
  if (runs_fit(p, 4, sizeof(T)) && p.dim <= 512) return launch_runs<T, 4>(p, st);
  if (runs_fit(p, 2, sizeof(T)) && p.dim <= 256) return launch_runs<T, 2>(p, st);
  const long items = p.tokens * (p.heads + (p.cached ? 2 : 1) * p.kv_heads);
  qk_norm_rope_any_kernel<T><<<grid_of((items + kThreads / 64 - 1) / (kThreads / 64)), kThreads, 0, st>>>(p);
  return launch_status("qk_norm_rope_any_kernel");
}

}  // namespace
}  // namespace sonar

using namespace sonar;

extern "C" const char* sonar_attention_last_error(void) { return last_error_buffer(); }

extern "C" int sonar_qk_norm_rope(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k, int64_t k_token_stride,
                                  int64_t k_head_stride, const void* v, int64_t v_token_stride, int64_t v_head_stride,
                                  const void* positions, int positions_64, const float* cos_sin, int64_t max_position,
                                  int64_t rotary_dim, int half, const void* q_weight, const void* k_weight, double epsilon,
                                  void* q_out, void* k_out, const sonar_kv_cache* key_cache, const sonar_kv_cache* value_cache,
                                  int cache_dtype, const void* slots, int slots_64, int64_t pages, int64_t page_size, int dtype,
                                  int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, void* stream) {
  SONAR_REQUIRE(dtype == SONAR_DTYPE_F16 || dtype == SONAR_DTYPE_BF16 || dtype == SONAR_DTYPE_F32, "unknown dtype = %d", dtype);
  SONAR_REQUIRE(heads >= 1 && kv_heads >= 1 && heads < (1 << 20) && kv_heads < (1 << 20) && head_dim >= 1 && head_dim <= 1024,
                "heads = %ld, kv_heads = %ld, head_dim = %ld (at most 1024)", (long)heads, (long)kv_heads, (long)head_dim);
  SONAR_REQUIRE(tokens >= 0 && tokens < (1LL << 31) && tokens * (heads + 2 * kv_heads) < (1LL << 31), "tokens = %ld of %ld heads: too many",
                (long)tokens, (long)(heads + 2 * kv_heads));
  SONAR_REQUIRE(cos_sin == nullptr || (rotary_dim >= 2 && rotary_dim % 2 == 0 && rotary_dim <= head_dim && max_position >= 0),
                "rotary_dim = %ld must be even and at most head_dim = %ld", (long)rotary_dim, (long)head_dim);
  SONAR_REQUIRE((q_weight == nullptr && k_weight == nullptr) || (epsilon >= 1.1754943508222875e-38 && epsilon <= 3.4e38),
                "epsilon = %g: a positive number of at least 2^-126 is needed", epsilon);
  const bool cached = key_cache != nullptr;
  SONAR_REQUIRE(cached == (value_cache != nullptr), "key_cache and value_cache go together");
  if (cached) {
    SONAR_REQUIRE(cache_dtype == dtype || (cache_dtype == SONAR_CACHE_FP8 && dtype != SONAR_DTYPE_F32),
                  "cache_dtype = %d does not go with dtype = %d", cache_dtype, dtype);
    SONAR_REQUIRE(pages >= 0 && page_size >= 1 && page_size < (1LL << 31) && pages < (1LL << 40) / page_size, "pages = %ld of %ld slots",
                  (long)pages, (long)page_size);
    for (const sonar_kv_cache* c : {key_cache, value_cache})
      SONAR_REQUIRE(cache_dtype != SONAR_CACHE_FP8 || (c->scale != nullptr && (c->scale_len == 1 || c->scale_len == kv_heads)),
                    "an 8-bit cache needs 1 or %ld scales; got %ld", (long)kv_heads, c->scale == nullptr ? 0L : (long)c->scale_len);
  }
  if (tokens == 0) return SONAR_OK;
  SONAR_REQUIRE((positions == nullptr) == (cos_sin == nullptr), "positions and cos_sin go together");
  SONAR_REQUIRE(q && k && q_out, "q, k and q_out must not be NULL");
  SONAR_REQUIRE(cached ? v && slots && key_cache->data && value_cache->data : k_out != nullptr,
                "a cache goes with v and slots, and k_out is needed without one");
  auto pages_of = [&](const sonar_kv_cache* c) {
    return c == nullptr ? Pages{} : Pages{(char*)c->data, c->page_stride, c->slot_stride, c->head_stride, c->scale, c->scale_len > 1};
  };
  RopeParams p{};
  p.q = q, p.k = k, p.v = cached ? v : nullptr;
  p.q_token = q_token_stride, p.q_head = q_head_stride, p.k_token = k_token_stride, p.k_head = k_head_stride;
  if (cached) p.v_token = v_token_stride, p.v_head = v_head_stride;
  p.positions = positions, p.table = cos_sin, p.max_position = max_position;
  p.q_weight = q_weight, p.k_weight = k_weight, p.q_out = q_out, p.k_out = cached ? nullptr : k_out;
  p.keys = pages_of(key_cache), p.values = pages_of(value_cache);
  p.slots = slots, p.all_slots = cached ? pages * page_size : 0, p.tokens = tokens;
  p.inverse_dim = (float)(1.0 / (double)head_dim), p.epsilon = (float)epsilon;
  p.rotary = cos_sin != nullptr ? (int)rotary_dim : 0, p.page_size = (int)page_size, p.heads = (int)heads, p.kv_heads = (int)kv_heads;
  p.dim = (int)head_dim;
  p.half = half != 0, p.positions_64 = positions_64 != 0, p.slots_64 = slots_64 != 0, p.cached = cached;
  p.fp8 = cached && cache_dtype == SONAR_CACHE_FP8;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == SONAR_DTYPE_F16) return launch<_Float16>(p, st);
  if (dtype == SONAR_DTYPE_BF16) return launch<__bf16>(p, st);
  return launch<float>(p, st);
}
