// Sums and maxima over a wavefront by data-parallel moves: no LDS, six steps, the result in every lane (a scalar register).
#pragma once

#include "common.hpp"

namespace sonar {

// `v` of the lane that CTRL names; `none` where there is none or ROWS (of 16 lanes, a bit each) leaves the lane out
template <int CTRL, int ROWS>
__device__ __forceinline__ int moved(int v, int none) {
  return __builtin_amdgcn_update_dpp(none, v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ float moved(float v, float none) {
  return __builtin_bit_cast(float, moved<CTRL, ROWS>(__builtin_bit_cast(int, v), __builtin_bit_cast(int, none)));
}
struct TwoWords {
  int lo, hi;
};
template <int CTRL, int ROWS>
__device__ __forceinline__ double moved(double v, double none) {
  const TwoWords x = __builtin_bit_cast(TwoWords, v), y = __builtin_bit_cast(TwoWords, none);
  return __builtin_bit_cast(double, TwoWords{moved<CTRL, ROWS>(x.lo, y.lo), moved<CTRL, ROWS>(x.hi, y.hi)});
}

__device__ __forceinline__ int of_lane(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ __forceinline__ float of_lane(float v, int lane) {
  return __builtin_bit_cast(float, of_lane(__builtin_bit_cast(int, v), lane));
}
__device__ __forceinline__ double of_lane(double v, int lane) {
  const TwoWords x = __builtin_bit_cast(TwoWords, v);
  return __builtin_bit_cast(double, TwoWords{of_lane(x.lo, lane), of_lane(x.hi, lane)});
}

// `join` of all 64 lanes' values, in one order; `none` is its neutral element.  Rows of 16 lanes first (shifts by 1, 2, 4, 8),
// then the last lane of a row joins the next row's, then the last of the first half the second half's.
template <typename V, typename F>
__device__ __forceinline__ V over_wave(V v, V none, F join) {
  v = join(v, moved<0x111, 0xf>(v, none));
  v = join(v, moved<0x112, 0xf>(v, none));
  v = join(v, moved<0x114, 0xf>(v, none));
  v = join(v, moved<0x118, 0xf>(v, none));
  v = join(v, moved<0x142, 0xa>(v, none));
  v = join(v, moved<0x143, 0xc>(v, none));
  return of_lane(v, 63);
}
template <typename V>
__device__ __forceinline__ V wave_sum(V v) {
  return over_wave(v, (V)0, [](V a, V b) { return a + b; });
}

}  // namespace sonar
