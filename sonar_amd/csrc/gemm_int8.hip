// Product of 8-bit integers with a scale for each token and channel (W8A8), on the int8 matrix instructions.
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

// 16 bytes of a row from k0 on, zeros behind its end.  Any alignment.
__device__ __forceinline__ intx4_t load_16(const int8_t* row, int k0, int k) {
  intx4_t v = {0, 0, 0, 0};
  if (k0 + 16 <= k) {
    __builtin_memcpy(&v, row + k0, 16);
  } else if (k0 < k) {
    for (int i = 0; i < 16; ++i)
      if (k0 + i < k) v[i >> 2] |= (int)((uint32_t)(uint8_t)row[k0 + i] << (8 * (i & 3)));
  }
  return v;
}

// Any strides, alignments and sizes: 64 x 64 results a workgroup, 32 x 32 a wavefront, 128 bytes of K a step through
// registers into LDS.
constexpr int kStep = 128, kPitch = kStep + 16;
template <typename T>
__global__ __launch_bounds__(256) void int8_general_kernel(const Int8Params p) {
  __shared__ __attribute__((aligned(16))) int8_t lds[2][128][kPitch];   // rows of a, then rows of b
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const long m0 = (long)blockIdx.y * 64, n0 = (long)blockIdx.x * 64;
  const int row = tid >> 3, chunk = tid & 7;   // a thread's rows row + 32 i, their 16 bytes at 16 chunk
  intx4_t held[4];
  auto fetch = [&](int k0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const long m = min(m0 + row + 32 * i, (long)p.m - 1), n = min(n0 + row + 32 * i, (long)p.n - 1);
      held[i] = load_16(p.a + m * p.lda, k0 + 16 * chunk, p.k);
      held[2 + i] = load_16(p.b + n * p.ldb, k0 + 16 * chunk, p.k);
    }
  };
  auto put = [&](int at) {
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<intx4_t*>(&lds[at][row + 32 * i][16 * chunk]) = held[i];
  };
  intx16_t acc = {};
  const int mw = (wave & 1) * 32, nw = 64 + (wave >> 1) * 32;
  fetch(0);
  for (int k0 = 0, at = 0; k0 < p.k; k0 += kStep, at ^= 1) {
    put(at);
    __syncthreads();
    if (k0 + kStep < p.k) fetch(k0 + kStep);
#pragma unroll
    for (int s = 0; s < kStep / 32; ++s) {
      const intx4_t av = *reinterpret_cast<const intx4_t*>(&lds[at][mw + (lane & 31)][32 * s + 16 * (lane >> 5)]);
      const intx4_t bv = *reinterpret_cast<const intx4_t*>(&lds[at][nw + (lane & 31)][32 * s + 16 * (lane >> 5)]);
      acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(bv, av, acc, 0, 0, 0);
    }
  }
  // a lane has row lane % 32 of a and columns 8 (r / 4) + 4 (lane / 32) + r % 4
  const long m = m0 + mw + (lane & 31);
  if (m >= p.m) return;
  const float sa = p.a_scales[p.a_many ? m : 0];
  T* out = (T*)p.c + m * p.n;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const long n = n0 + (nw - 64) + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
    if (n < p.n) {
      float v = (float)acc[r] * (sa * p.b_scales[p.b_many ? n : 0]);
      if (p.bias != nullptr) v += (float)((const T*)p.bias)[n];
      out[n] = (T)v;
    }
  }
}

}  // namespace
}  // namespace sonar

using namespace sonar;

extern "C" size_t sonar_scaled_mm_int8_scratch_bytes(int64_t size_m, int64_t size_n, int64_t size_k) {
  (void)size_m, (void)size_n, (void)size_k;
  return 0;
}

extern "C" int sonar_scaled_mm_int8(const int8_t* a, int64_t a_row_stride, const int8_t* b, int64_t b_row_stride, void* c,
                                    const float* a_scales, int64_t a_scales_len, const float* b_scales, int64_t b_scales_len,
                                    const void* bias, void* scratch, size_t scratch_bytes, int dtype, int64_t size_m,
                                    int64_t size_n, int64_t size_k, void* stream) {
  (void)scratch, (void)scratch_bytes;
  SONAR_REQUIRE(dtype == SONAR_DTYPE_F16 || dtype == SONAR_DTYPE_BF16, "unknown dtype = %d: float16 or bfloat16 results", dtype);
  SONAR_REQUIRE(size_m >= 0 && size_m < (1LL << 31) - 256 && size_n >= 0 && size_n < (1LL << 31) - 256, "size_m = %ld, size_n = %ld",
                (long)size_m, (long)size_n);
  SONAR_REQUIRE(size_k >= 0 && size_k < 131072, "size_k = %ld: the 32-bit sums hold fewer than 131072 products", (long)size_k);
  if (size_m == 0 || size_n == 0) return SONAR_OK;
  SONAR_REQUIRE(c && a_scales && b_scales && (size_k == 0 || (a && b)), "a, b, c and the scales must not be NULL");
  SONAR_REQUIRE(a_row_stride >= size_k && b_row_stride >= size_k, "row strides %ld and %ld are smaller than size_k = %ld",
                (long)a_row_stride, (long)b_row_stride, (long)size_k);
  SONAR_REQUIRE((a_scales_len == 1 || a_scales_len == size_m) && (b_scales_len == 1 || b_scales_len == size_n),
                "a_scales holds %ld numbers (1 or size_m = %ld are needed), b_scales %ld (1 or size_n = %ld)", (long)a_scales_len,
                (long)size_m, (long)b_scales_len, (long)size_n);
  const Int8Params p{a,        b,        c, a_scales, b_scales, bias, a_row_stride, b_row_stride, (int)size_m, (int)size_n,
                     (int)size_k, a_scales_len > 1, b_scales_len > 1};
  hipStream_t st = (hipStream_t)stream;
  const int64_t rows = (size_m + 63) / 64, cols = (size_n + 63) / 64;
  SONAR_REQUIRE(rows < 65536 && cols < (1 << 24), "size_m = %ld, size_n = %ld", (long)size_m, (long)size_n);
  const dim3 grid((unsigned)cols, (unsigned)rows);
  if (dtype == SONAR_DTYPE_F16) int8_general_kernel<_Float16><<<grid, 256, 0, st>>>(p);
  else int8_general_kernel<__bf16><<<grid, 256, 0, st>>>(p);
  return launch_status("int8_general_kernel");
}
