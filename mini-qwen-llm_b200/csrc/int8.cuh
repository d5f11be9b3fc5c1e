// Symmetric int8 quantisation of a row, as every int8 path of the library does it:
//   scale = max|x| / 127, rounded to fp32;  q = the whole number nearest to x / scale, halves to even.
// A row of zeros has scale 0 and q 0.  A row that holds an infinity or a NaN has scale NaN and q 0, so that everything
// computed from it is NaN: one bad token must not come back as plausible numbers.
#pragma once

#include "common.cuh"

namespace mq {
namespace int8 {

// max|x| of a row is kept as the bits of a non-negative float: they order as integers, infinities above every finite
// number and NaNs above infinities, where fmaxf would lose a NaN.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

__device__ __forceinline__ float scale_of(uint32_t max_bits) {
  if (max_bits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  return __fdiv_rn(__uint_as_float(max_bits), 127.0f);
}

// What a row's values are multiplied by on their way to q: 0 for rows without values to scale.  Scales below 2^-120 have
// a reciprocal out of range or too coarse; those rows divide (quantize() below, exact = true).
struct RowScale {
  float scale, inv;
  bool exact;
};
__device__ __forceinline__ RowScale row_scale(uint32_t max_bits) {
  RowScale r;
  r.scale = scale_of(max_bits);
  r.exact = r.scale < 0x1p-120f && r.scale > 0.0f;
  r.inv = r.scale >= 0x1p-120f ? __frcp_rn(r.scale) : 0.0f;      // false for NaN and 0
  return r;
}

// x * inv is off by less than 2e-5 (|q| <= 127.5, three roundings of 2^-24), so it names the nearest whole number unless
// it lies within 1e-4 of a half.  There, and for tiny scales, the quotient is taken in 64 bits, where it is a half only
// if it is exactly one.
__device__ __forceinline__ int quantize(float x, const RowScale& r) {
  if (r.inv == 0.0f && !r.exact) return 0;                       // nothing to scale
  const float v = __fmul_rn(x, r.inv);
  float q = rintf(v);
  if (r.exact || fabsf(v - q) > 0.4999f) q = (float)rint(__ddiv_rn((double)x, (double)r.scale));
  return (int)fminf(fmaxf(q, -127.0f), 127.0f);
}

}  // namespace int8
}  // namespace mq
