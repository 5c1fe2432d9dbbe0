// Root-mean-square norm with the residual's addition before it and 8-bit codes with one scale a token behind it.
#include "common.hpp"
#include "sonar_layer.h"

namespace sonar {
namespace {
thread_local char g_layer_error[512] = "";
}  // namespace
char* last_error_buffer() { return g_layer_error; }

namespace {

constexpr int kThreads = 256;

template <typename V, typename F>
__device__ __forceinline__ V across_block(V v, V* part, F join) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = join(v, __shfl_xor(v, off, 64));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = part[0];
#pragma unroll
  for (int w = 1; w < kThreads / 64; ++w) v = join(v, part[w]);
  return v;
}

// One workgroup a row, element by element; z is read again in each pass.
template <typename T, bool FP8>
__global__ __launch_bounds__(kThreads) void rms_norm_quant_kernel(const T* x, long x_stride, const T* residual, long residual_stride,
                                                                  const T* __restrict__ weight, T* residual_out, T* norm_out,
                                                                  uint8_t* __restrict__ q, float* __restrict__ scales, int cols,
                                                                  double epsilon) {
#pragma clang fp contract(off)
  __shared__ double sums[kThreads / 64];
  __shared__ float mosts[kThreads / 64];
  const long row = blockIdx.x;
  const T* in = x + row * x_stride;
  const T* z = in;
  double sum = 0;
  if (residual != nullptr) {
    T* out = residual_out + row * cols;
    for (int c = threadIdx.x; c < cols; c += kThreads) {
      const T v = (T)((float)in[c] + (float)residual[row * residual_stride + c]);
      out[c] = v;
      sum += (double)(float)v * (double)(float)v;
    }
    z = out;
  } else {
    for (int c = threadIdx.x; c < cols; c += kThreads) sum += (double)(float)in[c] * (double)(float)in[c];
  }
  sum = across_block(sum, sums, [](double a, double b) { return a + b; });
  const float r = (float)(1.0 / sqrt(sum / cols + epsilon));
  float most = 0.0f;
  for (int c = threadIdx.x; c < cols; c += kThreads) most = fmaxf(most, fabsf((float)z[c] * r * (float)weight[c]));
  most = across_block(most, mosts, [](float a, float b) { return fmaxf(a, b); });
  const bool finite = sum <= 1.7976931348623157e308;   // false for infinities and NaN
  float by, scale;
  if (FP8) {
    scale = fmaxf(most / 448.0f, 1.0f / (448.0f * 512.0f));
    by = 1.0f / scale;
  } else {
    most = fmaxf(most, 1e-10f);
    scale = most / 127.0f;
    by = 127.0f / most;
  }
  if (threadIdx.x == 0) scales[row] = finite ? scale : __builtin_nanf("");
  for (int c = threadIdx.x; c < cols; c += kThreads) {
    const float y = (float)z[c] * r * (float)weight[c];
    if (norm_out != nullptr) norm_out[row * cols + c] = (T)y;
    const float t = y * by;
    uint8_t code;
    if (FP8) code = (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32(fminf(fmaxf(t, -448.0f), 448.0f), 0.0f, 0, false) & 0xff);
    else code = (uint8_t)(int)(t + copysignf(0.5f, t));
    q[row * cols + c] = finite ? code : 0;
  }
}

template <bool FP8>
int launch(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride, const void* weight, void* residual_out,
           void* norm_out, void* q, float* scales, int dtype, int64_t rows, int64_t cols, double epsilon, hipStream_t st) {
#define SONAR_NORM(T)                                                                                                       \
  rms_norm_quant_kernel<T, FP8><<<(int)rows, kThreads, 0, st>>>((const T*)x, x_stride, (const T*)residual, residual_stride, \
                                                                (const T*)weight, (T*)residual_out, (T*)norm_out,           \
                                                                (uint8_t*)q, scales, (int)cols, epsilon)
  if (dtype == SONAR_DTYPE_F16) SONAR_NORM(_Float16);
  else if (dtype == SONAR_DTYPE_BF16) SONAR_NORM(__bf16);
  else SONAR_NORM(float);
#undef SONAR_NORM
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
  hipStream_t st = (hipStream_t)stream;
  return q_dtype == SONAR_ADTYPE_FP8
             ? launch<true>(x, x_row_stride, residual, residual_row_stride, weight, residual_out, norm_out, q, scales, dtype, rows,
                            cols, epsilon, st)
             : launch<false>(x, x_row_stride, residual, residual_row_stride, weight, residual_out, norm_out, q, scales, dtype, rows,
                             cols, epsilon, st);
}
