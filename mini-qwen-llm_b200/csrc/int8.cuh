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

// What a row's values are multiplied by on their way to q; 0 for rows without values to scale.  Scales below 2^-120 have a
// reciprocal out of range or too coarse; those rows divide (exact).
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

// The quotient in 64 bits, where it is a half only if it is exactly one (out of line: it is rare, and long).
static __device__ __noinline__ int exact_quotient(float x, float scale) {
  return (int)fmin(fmax(rint(__ddiv_rn((double)x, (double)scale)), -127.0), 127.0);
}

// N values to bytes.  1.5 * 2^23 + x * inv, rounded once, has the nearest whole number n in its low bits.  x * inv is off the
// quotient by |q| 2^-24 < 8e-6 at most, so n is the right one unless x * inv lies within 1.6e-5 of a half h = n +- 1/2.  There
// the sign of x - h * scale decides, which one fused multiply-add gives exactly (h * scale has 32 bits, and no difference
// from 2^-120 on vanishes); 0 is a half, which goes to the even side.  16-bit numbers meet halves often: half of the row's
// maximum is 63.5.  (With a quotient in 64 bits there, 32768 rows of 2048 bf16 numbers took 77 us.)  No clamp:
// |x| * inv <= 127 (1 + 2^-22).
template <int N>
__device__ __forceinline__ void quantize(const float (&x)[N], const RowScale& r, uint32_t (&q)[N / 4]) {
  constexpr float MAGIC = 12582912.0f;
  uint32_t y[N];
  float off = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float v = __fmaf_rn(x[i], r.inv, MAGIC);
    y[i] = __float_as_uint(v);
    off = fmaxf(off, fabsf(__fmaf_rn(x[i], r.inv, __fsub_rn(MAGIC, v))));
  }
  if (r.inv == 0.0f) {                                           // zeros, no numbers, or tiny ones
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] = r.exact ? (uint32_t)exact_quotient(x[i], r.scale) : 0u;
  } else if (off > 0.499984f) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float n = __fsub_rn(__uint_as_float(y[i]), MAGIC), d = __fmaf_rn(x[i], r.inv, -n), side = copysignf(1.0f, d);
      const float past = side * __fmaf_rn(-__fmaf_rn(0.5f, side, n), r.scale, x[i]);
      if (fabsf(d) > 0.499984f && (past > 0.0f || (past == 0.0f && (y[i] & 1u) != 0))) y[i] += d > 0.0f ? 1u : 0xffffffffu;
    }
  }
#pragma unroll
  for (int i = 0; i < N / 4; ++i)
    q[i] = __byte_perm(__byte_perm(y[4 * i], y[4 * i + 1], 0x0040), __byte_perm(y[4 * i + 2], y[4 * i + 3], 0x0040), 0x5410);
}
__device__ __forceinline__ int quantize(float x, const RowScale& r) {
  const float v[4] = {x, 0.0f, 0.0f, 0.0f};
  uint32_t q[1];
  quantize<4>(v, r, q);
  return (int)(int8_t)(q[0] & 0xffu);
}

}  // namespace int8
}  // namespace mq
