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

// `join` over LANES neighbouring lanes (8, 16, 32 or 64), every lane with the result: exchanges within four lanes, mirrors of
// eight and sixteen, then swaps of rows and of halves.  The order is fixed; a `join` that commutes gives all lanes the same bits.
template <int CTRL>
__device__ __forceinline__ uint32_t exchanged(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
template <int CTRL>
__device__ __forceinline__ double exchanged(double v) {
  const TwoWords x = __builtin_bit_cast(TwoWords, v);
  return __builtin_bit_cast(double, TwoWords{(int)exchanged<CTRL>((uint32_t)x.lo), (int)exchanged<CTRL>((uint32_t)x.hi)});
}
template <bool HALVES>   // the two sides of a swap of rows (of halves) of `v` with itself
__device__ __forceinline__ void sides(uint32_t v, uint32_t& one, uint32_t& other) {
  const auto both = HALVES ? __builtin_amdgcn_permlane32_swap(v, v, false, false) : __builtin_amdgcn_permlane16_swap(v, v, false, false);
  one = both[0], other = both[1];
}
template <bool HALVES>
__device__ __forceinline__ void sides(double v, double& one, double& other) {
  const TwoWords x = __builtin_bit_cast(TwoWords, v);
  uint32_t lo[2], hi[2];
  sides<HALVES>((uint32_t)x.lo, lo[0], lo[1]);
  sides<HALVES>((uint32_t)x.hi, hi[0], hi[1]);
  one = __builtin_bit_cast(double, TwoWords{(int)lo[0], (int)hi[0]});
  other = __builtin_bit_cast(double, TwoWords{(int)lo[1], (int)hi[1]});
}
template <int LANES, typename V, typename F>
__device__ __forceinline__ V over_lanes(V v, F join) {
  static_assert(LANES == 8 || LANES == 16 || LANES == 32 || LANES == 64, "");
  v = join(v, exchanged<0xB1>(v));
  v = join(v, exchanged<0x4E>(v));
  v = join(v, exchanged<0x141>(v));
  if constexpr (LANES >= 16) v = join(v, exchanged<0x140>(v));
  V one, other;
  if constexpr (LANES >= 32) {
    sides<false>(v, one, other);
    v = join(one, other);
  }
  if constexpr (LANES >= 64) {
    sides<true>(v, one, other);
    v = join(one, other);
  }
  return v;
}

}  // namespace sonar
