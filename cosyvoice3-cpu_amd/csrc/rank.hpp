// Numbers as unsigned keys of the same order, for choices by the largest.
#pragma once

#include "common.hpp"
#include "decode_common.hpp"   // DPP lane exchanges

namespace cv3 {

// Rises with f; -0 as 0, a NaN as -inf.  0 is below every number's: an absent candidate.
__device__ __forceinline__ uint32_t rank_bits(float f) {
  f += 0.f;
  if (!(f == f)) f = -INFINITY;
  const uint32_t b = __float_as_uint(f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float rank_value(uint32_t r) {
  return __uint_as_float(r & 0x80000000u ? r & 0x7fffffffu : ~r);
}
__device__ __forceinline__ uint64_t rank_bits(double f) {
  f += 0.0;
  if (!(f == f)) f = -INFINITY;
  const uint64_t b = (uint64_t)__double_as_longlong(f);
  return b >> 63 ? ~b : b | (uint64_t)1 << 63;
}
__device__ __forceinline__ double rank_value(uint64_t r) {
  return __longlong_as_double((int64_t)(r >> 63 ? r & ~((uint64_t)1 << 63) : ~r));
}

// Sum over the wave by DPP row permutations and four lane reads.
template <int CTRL>
__device__ __forceinline__ double dpp_d(double v) {
  return __longlong_as_double((int64_t)dpp64<CTRL>((uint64_t)__double_as_longlong(v)));
}
__device__ __forceinline__ double wave_sum_dpp(double v) {
  v += dpp_d<kDppXor1>(v);
  v += dpp_d<kDppXor2>(v);
  v += dpp_d<kDppHalfMirror>(v);
  v += dpp_d<kDppMirror>(v);
  return (readlane_d(v, 0) + readlane_d(v, 16)) + (readlane_d(v, 32) + readlane_d(v, 48));
}

}  // namespace cv3
