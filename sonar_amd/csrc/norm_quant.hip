// Root-mean-square norm with the residual's addition before it and 8-bit codes with one scale a token behind it:
//   z = T(x + residual);  r = 1 / sqrt(mean(z^2) + epsilon);  y = (z * r) * weight;  codes of y against its largest magnitude
// The sum of squares and r are held in 64 bits and r is rounded once, y and the codes' arithmetic are float32, so that the
// result hardly depends on the order of the sum, which the forms below take differently: one r in about 2^24 comes out a last
// bit apart, and that bit may turn a code of its row.
//
// One pass over memory: a row is read once, z stays in registers (16 bits a number where the type has 16), y is formed
// twice, for the maximum and for the codes.  Bound by the bytes.
#include "common.hpp"
#include "lane_reduce.hpp"
#include "sonar_layer.h"

namespace sonar {
namespace {
thread_local char g_layer_error[512] = "";
}  // namespace
char* last_error_buffer() { return g_layer_error; }

namespace {

constexpr int kThreads = 256;   // of a workgroup, where a row has no more

struct NormParams {
  const void* x;
  const void* residual;
  const void* weight;
  void* residual_out;
  void* norm_out;
  uint8_t* q;
  float* scales;
  long x_stride, residual_stride, rows;
  int cols;
  double inverse_cols, epsilon;
};

// Joins over a workgroup; `part` may be used again behind another call's barrier.
template <int THREADS, typename V, typename F>
__device__ __forceinline__ V over_block(V v, V none, V* part, F join) {
  v = over_wave(v, none, join);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = part[0];
#pragma unroll
  for (int w = 1; w < THREADS / 64; ++w) v = join(v, part[w]);
  return v;
}

// 1 / sqrt(x) for x >= 2^-126 (or infinite, NaN), rounded once: an estimate of 2^-24 or better, two of Newton's steps.
__device__ __forceinline__ float inverse_root(double x) {
  double y = __builtin_amdgcn_rsq(x);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const double e = __builtin_fma(-x * y, y, 1.0);
    y = __builtin_fma(y * e, 0.5, y);
  }
  return x <= 1.7976931348623157e308 ? (float)y : (float)(x - x);   // (infinities and NaN: NaN)
}

// A NaN stays one in these (the instructions of three operands; fmaxf and fminf would drop it).
__device__ __forceinline__ float larger_of(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float smaller_of(float a, float b) { return __builtin_elementwise_minimum(a, b); }

// A row's scale, and what its numbers are multiplied by; both NaN where one of its numbers is.
template <bool FP8>
__device__ __forceinline__ void scale_of(float most, float& scale, float& by) {
  if (FP8) {
    scale = larger_of(most / 448.0f, 1.0f / (448.0f * 512.0f));
    by = 1.0f / scale;
  } else {
    most = larger_of(most, 1e-10f);
    scale = most / 127.0f;
    by = 127.0f / most;
  }
}

// A code in the low byte: halves away from zero (int8), the nearest float8_e4m3fn.  A NaN's is 0 (int8), the type's NaN (fp8).
__device__ __forceinline__ int int8_code(float y, float by) {
#pragma clang fp contract(off)
  const float t = y * by;
  return (int)(t + __builtin_copysignf(0.5f, t)) & 0xff;
}
__device__ __forceinline__ float fp8_number(float y, float by) {
#pragma clang fp contract(off)
  const float t = y * by;
  return smaller_of(larger_of(t, -448.0f), 448.0f);
}

// Eight neighbouring numbers.
template <typename T>
struct Eight {
  typedef T vec __attribute__((ext_vector_type(8)));
  vec v;
  __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const vec*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<vec*>(p) = v; }
  __device__ __forceinline__ float at(int i) const { return (float)v[i]; }
};

// THREADS (64, 256 or 1024) a row, eight neighbouring columns of a row's KEPT turns a thread.  THREADS = 64: four rows a
// workgroup, sums and maxima by lane moves, no barrier.  THREADS = 1024: rows of any length; turns beyond KEPT are read
// again (as z).  A workgroup that goes on to a further row has its numbers loaded before it works on its own; the weight
// stays in registers.
// 16384 x 4096 bf16 to int8 with a residual (470 MB): 80 us, 5.8 TB/s (float32 151 us, 5.8 TB/s); 92 with
// eight workgroups a compute unit that walk the rows instead of a workgroup a row (fresh ones overlap their loads with the
// others' stores), 97 with a wavefront a row, 220 element by element with three passes.  Registers decide: row bases in scalar registers with 32-bit offsets of the
// columns, and no code of the repeated reads where no call needs them, took 107 registers to 68 and 16384 x 2880 without a
// residual from 47 to 34 us.
template <typename T, bool FP8, int THREADS, int KEPT>
__global__ __launch_bounds__(THREADS > kThreads ? THREADS : kThreads) void rms_norm_quant_kernel(const NormParams p) {
#pragma clang fp contract(off)
  constexpr int kRows = THREADS < kThreads ? kThreads / THREADS : 1, kStep = THREADS * 8;
  __shared__ double sums[THREADS / 64];
  __shared__ float mosts[THREADS / 64];
  const uint32_t first = threadIdx.x % THREADS * 8, cols = p.cols;
  Eight<T> weight[KEPT], z[KEPT];
#pragma unroll
  for (int i = 0; i < KEPT; ++i)
    if (first + i * kStep < cols) weight[i].load((const T*)p.weight + first + i * kStep);
  const long step = (long)gridDim.x * kRows;
  long row = (long)blockIdx.x * kRows + __builtin_amdgcn_readfirstlane(threadIdx.x / THREADS);
  Eight<T> more[KEPT];
  auto fetch = [&](long at, Eight<T> (&to)[KEPT]) {
    const T* x = (const T*)p.x + at * p.x_stride;
#pragma unroll
    for (int i = 0; i < KEPT; ++i)
      if (first + i * kStep < cols) to[i].load(x + first + i * kStep);
    if (p.residual != nullptr) {
      const T* residual = (const T*)p.residual + at * p.residual_stride;
#pragma unroll
      for (int i = 0; i < KEPT; ++i)
        if (first + i * kStep < cols) more[i].load(residual + first + i * kStep);
    }
  };
  Eight<T> next[KEPT];
  if (row < p.rows) fetch(row, next);
  for (; row < p.rows; row += step) {
    const T* x = (const T*)p.x + row * p.x_stride;
    const T* residual = (const T*)p.residual + row * p.residual_stride;
    T* out = (T*)p.residual_out + row * cols;
    double sum = 0;
    auto add = [&](const Eight<T>& v) {
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = __builtin_fma((double)v.at(e), (double)v.at(e), sum);
    };
    auto join = [&](Eight<T>& v, const Eight<T>& r, uint32_t c) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v.v[e] = (T)(v.at(e) + r.at(e));
      v.store(out + c);
    };
#pragma unroll
    for (int i = 0; i < KEPT; ++i) z[i] = next[i];
    if (p.residual != nullptr) {
#pragma unroll
      for (int i = 0; i < KEPT; ++i)
        if (first + i * kStep < cols) join(z[i], more[i], first + i * kStep);
    }
    if (row + step < p.rows) fetch(row + step, next);
#pragma unroll
    for (int i = 0; i < KEPT; ++i)
      if (first + i * kStep < cols) add(z[i]);
    const T* again = p.residual != nullptr ? out : x;   // z of the turns that no register keeps
    if (THREADS > kThreads)
      for (uint32_t c = first + KEPT * kStep; c < cols; c += kStep) {
        Eight<T> v;
        v.load(x + c);
        if (p.residual != nullptr) {
          Eight<T> more;
          more.load(residual + c);
          join(v, more, c);
        }
        add(v);
      }
    sum = THREADS == 64 ? wave_sum(sum) : over_block<THREADS>(sum, 0.0, sums, [](double a, double b) { return a + b; });
    const float r = inverse_root(__builtin_fma(sum, p.inverse_cols, p.epsilon));
    float most = 0.0f;
    auto larger = [&](const Eight<T>& v, const Eight<T>& w) {
#pragma unroll
      for (int e = 0; e < 8; ++e) most = larger_of(most, fabsf(v.at(e) * r * w.at(e)));
    };
#pragma unroll
    for (int i = 0; i < KEPT; ++i)
      if (first + i * kStep < cols) larger(z[i], weight[i]);
    if (THREADS > kThreads)
      for (uint32_t c = first + KEPT * kStep; c < cols; c += kStep) {
        Eight<T> v, w;
        v.load(again + c), w.load((const T*)p.weight + c);
        larger(v, w);
      }
    auto max_of = [](float a, float b) { return larger_of(a, b); };
    most = THREADS == 64 ? over_wave(most, 0.0f, max_of) : over_block<THREADS>(most, 0.0f, mosts, max_of);
    float scale, by;
    scale_of<FP8>(most, scale, by);
    if (first == 0) p.scales[row] = scale;
    auto code = [&](const Eight<T>& v, const Eight<T>& w, uint32_t c) {
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = v.at(e) * r * w.at(e);
      if (p.norm_out != nullptr) {
        Eight<T> n;
#pragma unroll
        for (int e = 0; e < 8; ++e) n.v[e] = (T)y[e];
        n.store((T*)p.norm_out + row * cols + c);
      }
      uint32_t word[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (FP8) {
          const int low = __builtin_amdgcn_cvt_pk_fp8_f32(fp8_number(y[4 * h], by), fp8_number(y[4 * h + 1], by), 0, false);
          word[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(fp8_number(y[4 * h + 2], by), fp8_number(y[4 * h + 3], by), low, true);
        } else {
          word[h] = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) word[h] |= (uint32_t)int8_code(y[4 * h + e], by) << (8 * e);
        }
      }
      *reinterpret_cast<uint2*>(p.q + row * cols + c) = make_uint2(word[0], word[1]);
    };
#pragma unroll
    for (int i = 0; i < KEPT; ++i)
      if (first + i * kStep < cols) code(z[i], weight[i], first + i * kStep);
    if (THREADS > kThreads)
      for (uint32_t c = first + KEPT * kStep; c < cols; c += kStep) {
        Eight<T> v, w;
        v.load(again + c), w.load((const T*)p.weight + c);
        code(v, w, c);
      }
  }
}

// Any column count, stride and alignment: a workgroup a row, element by element; z is read again in each pass (4096 x 4099 bf16
// with a residual 55 us, 2.1 TB/s of the bytes it needs; 4096 columns 24).
template <typename T, bool FP8>
__global__ __launch_bounds__(kThreads) void rms_norm_quant_any_kernel(const NormParams p) {
#pragma clang fp contract(off)
  __shared__ double sums[kThreads / 64];
  __shared__ float mosts[kThreads / 64];
  const int cols = p.cols;
  const T* weight = (const T*)p.weight;
  for (long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* z = (const T*)p.x + row * p.x_stride;
    double sum = 0;
    if (p.residual != nullptr) {
      const T* residual = (const T*)p.residual + row * p.residual_stride;
      T* out = (T*)p.residual_out + row * cols;
      for (int c = threadIdx.x; c < cols; c += kThreads) {
        const T v = (T)((float)z[c] + (float)residual[c]);
        out[c] = v;
        sum = __builtin_fma((double)(float)v, (double)(float)v, sum);
      }
      z = out;
    } else {
      for (int c = threadIdx.x; c < cols; c += kThreads) sum = __builtin_fma((double)(float)z[c], (double)(float)z[c], sum);
    }
    sum = over_block<kThreads>(sum, 0.0, sums, [](double a, double b) { return a + b; });
    const float r = inverse_root(__builtin_fma(sum, p.inverse_cols, p.epsilon));
    float most = 0.0f;
    for (int c = threadIdx.x; c < cols; c += kThreads) most = larger_of(most, fabsf((float)z[c] * r * (float)weight[c]));
    most = over_block<kThreads>(most, 0.0f, mosts, [](float a, float b) { return larger_of(a, b); });
    float scale, by;
    scale_of<FP8>(most, scale, by);
    if (threadIdx.x == 0) p.scales[row] = scale;
    for (int c = threadIdx.x; c < cols; c += kThreads) {
      const float y = (float)z[c] * r * (float)weight[c];
      if (p.norm_out != nullptr) ((T*)p.norm_out)[row * cols + c] = (T)y;
      p.q[row * cols + c] = FP8 ? (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32(fp8_number(y, by), 0.0f, 0, false) & 0xff)
                                : (uint8_t)int8_code(y, by);
    }
  }
}

// Workgroups: `each` a compute unit at most, which go on to further rows.
int grid_of(long groups, int each) { return (int)(groups < 256L * each ? groups : 256L * each); }

template <typename T, bool FP8>
int launch(const NormParams& p, hipStream_t st) {
  auto at_16 = [](const void* q) { return (uintptr_t)q % 16 == 0; };
  const long pitch = (long)(16 / sizeof(T));
  const bool vectors = p.cols % 8 == 0 && at_16(p.x) && at_16(p.residual) && at_16(p.weight) && at_16(p.residual_out) &&
                       at_16(p.norm_out) && (uintptr_t)p.q % 8 == 0 && p.x_stride % pitch == 0 && p.residual_stride % pitch == 0;
  if (!vectors) {
    rms_norm_quant_any_kernel<T, FP8><<<grid_of(p.rows, 8), kThreads, 0, st>>>(p);
    return launch_status("rms_norm_quant_any_kernel");
  }
  // Columns that a row's threads keep: as few turns as the row needs.  Rows of up to 1024: a wavefront each (4096 x 1024 with
  // a residual 8.5 us, a workgroup each 11.2), but a workgroup each where they are few (64 x 1024 3.48 and 3.32, even at 512).
  // Over 8192: 1024 threads and two workgroups a compute unit, which load ahead (4096 x 16384 88 us, with eight 102;
  // 256 threads that read half of the row again 121).
  const long fours = (p.rows + 3) / 4;
  const int grid = grid_of(p.rows, 128);
  if (p.cols <= 512) rms_norm_quant_kernel<T, FP8, 64, 1><<<grid_of(fours, 128), kThreads, 0, st>>>(p);
  else if (p.cols <= 1024 && p.rows >= 512) rms_norm_quant_kernel<T, FP8, 64, 2><<<grid_of(fours, 128), kThreads, 0, st>>>(p);
  else if (p.cols <= 2048) rms_norm_quant_kernel<T, FP8, 256, 1><<<grid, kThreads, 0, st>>>(p);
  else if (p.cols <= 4096) rms_norm_quant_kernel<T, FP8, 256, 2><<<grid, kThreads, 0, st>>>(p);
  else if (p.cols <= 8192) rms_norm_quant_kernel<T, FP8, 256, 4><<<grid, kThreads, 0, st>>>(p);
  else rms_norm_quant_kernel<T, FP8, 1024, 2><<<grid_of(p.rows, 2), 1024, 0, st>>>(p);
  return launch_status("rms_norm_quant_kernel");
}

}  // namespace
}  // namespace sonar

using namespace sonar;

extern "C" const char* sonar_layer_last_error(void) { return last_error_buffer(); }

extern "C" int sonar_rms_norm_per_token_quant(const void* x, int64_t x_row_stride, const void* residual,
                                              int64_t residual_row_stride, const void* weight, void* residual_out,
                                              void* norm_out, void* q, int q_dtype, float* scales, int dtype,
                                              int64_t rows, int64_t cols, double epsilon, void* stream) {
  SONAR_REQUIRE(rows >= 0 && rows < (1LL << 31) && cols > 0 && cols < (1LL << 30), "rows = %ld, cols = %ld", (long)rows,
                (long)cols);
  SONAR_REQUIRE(dtype == SONAR_DTYPE_F16 || dtype == SONAR_DTYPE_BF16 || dtype == SONAR_DTYPE_F32, "unknown dtype = %d", dtype);
  SONAR_REQUIRE(q_dtype == SONAR_ADTYPE_INT8 || q_dtype == SONAR_ADTYPE_FP8, "unknown q_dtype = %d", q_dtype);
  SONAR_REQUIRE(x_row_stride >= cols, "x_row_stride = %ld is smaller than cols = %ld", (long)x_row_stride, (long)cols);
  SONAR_REQUIRE(residual == nullptr || residual_row_stride >= cols, "residual_row_stride = %ld is smaller than cols = %ld",
                (long)residual_row_stride, (long)cols);
  SONAR_REQUIRE(epsilon >= 1.1754943508222875e-38 && epsilon <= 3.4e38, "epsilon = %g: a positive number of at least 2^-126 is needed",
                epsilon);
  if (rows == 0) return SONAR_OK;
  SONAR_REQUIRE(x && weight && q && scales, "x, weight, q and scales must not be NULL");
  SONAR_REQUIRE((residual == nullptr) == (residual_out == nullptr), "residual and residual_out go together");
  const NormParams p{x, residual, weight, residual_out, norm_out, (uint8_t*)q, scales, x_row_stride, residual ? residual_row_stride : 0,
                     rows, (int)cols, 1.0 / (double)cols, epsilon};
  hipStream_t st = (hipStream_t)stream;
  const bool fp8 = q_dtype == SONAR_ADTYPE_FP8;
  if (dtype == SONAR_DTYPE_F16) return fp8 ? launch<_Float16, true>(p, st) : launch<_Float16, false>(p, st);
  if (dtype == SONAR_DTYPE_BF16) return fp8 ? launch<__bf16, true>(p, st) : launch<__bf16, false>(p, st);
  return fp8 ? launch<float, true>(p, st) : launch<float, false>(p, st);
}
