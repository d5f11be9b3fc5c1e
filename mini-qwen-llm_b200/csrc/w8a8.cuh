// What the W8A8 kernels share: a call's arguments, and the arithmetic behind the int32 sums.
#pragma once

#include "common.cuh"

namespace mq {

struct W8Args {
  const int8_t* x;             // [T, K]
  const float* x_scale;        // [T]
  const int8_t* w;             // [period, N or 2 N, K]
  const float* w_scale;        // [period, N or 2 N]
  const int32_t* offsets;      // [E + 1], or null: one group of all rows
  const int32_t* perm;         // row r of the sorted order is row perm[r] / top_k of x; null: row r
  int S, T, top_k, E, period;
  int N, K;                    // N: output columns (SwiGLU: gate rows, then as many up rows)
  void* out;                   // [S, N]
  int grid;                    // 16: rows of x and w start at multiples of 16 bytes; else 1
  uint32_t k_mul, k_shift;     // n / top_k = umulhi(n, k_mul) >> k_shift for n < 2^31; k_mul 0: n
};

// Offsets outside 0..S, and permutation entries outside x, are the caller's mistake; they must not become addresses.
__device__ __forceinline__ int w8_offset(const W8Args& A, int e) { return min(max(A.offsets[e], 0), A.S); }
__device__ __forceinline__ size_t w8_source(const W8Args& A, int row) {
  if (A.perm == nullptr) return (size_t)row;
  const uint32_t slot = (uint32_t)max(A.perm[row], 0);
  return min(A.k_mul == 0 ? slot : __umulhi(slot, A.k_mul) >> A.k_shift, (uint32_t)(A.T - 1));
}

// The sum may pass 2^24, so the conversion rounds; with the two products that is 1.5 * 2^-23 in all at most.
__device__ __forceinline__ float w8_value(int sum, float row_scale, float channel_scale) {
  return __fmul_rn(__fmul_rn(__int2float_rn(sum), row_scale), channel_scale);
}
// silu(g) * u with the hardware's exponential and reciprocal, 2^-22 and 2^-23 relative.  With the exponential of -|g| nothing
// overflows and the denominator is in 1..2.
// 16-bit results: the exponent's rounding makes 1.5 |g| 2^-24, far below the rounding of the result, and where the exponential is
// below 2^-126 (g < -87) the result is 0, off by less than 1e-36 |u|.  The library's expf and a true quotient take some 40
// instructions more for each of the 25 million outputs of 4096 tokens (132 against 125 us).
// fp32 results: what the exponent t = -|g| log2(e) lost, c, comes back to first order, 2^(t + c) = 2^t (1 + c ln 2) with
// c < 2^-16, and small exponentials keep their step: 12 * 2^-24 in all (131 us, 123 without; with expf and a true quotient 163).
template <typename OutT>
__device__ __forceinline__ float w8_swiglu(float g, float u) {
  float p, r;
  if (sizeof(OutT) == 4) {
    constexpr float L = 1.44269504f, L_REST = 1.92596299e-8f, LN2 = 0.693147181f;      // L + L_REST = log2(e)
    const float a = fminf(fabsf(g), 256.0f), t = __fmul_rn(a, -L);                     // no infinities in c
    const float c = __fmaf_rn(a, -L_REST, __fmaf_rn(a, -L, -t));
    asm("ex2.approx.f32 %0, %1;" : "=f"(p) : "f"(t));
    p = __fmaf_rn(p, __fmul_rn(c, LN2), p);
  } else {
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p) : "f"(__fmul_rn(fabsf(g), -1.44269504f)));
  }
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(__fadd_rn(1.0f, p)));
  return __fmul_rn(__fmul_rn(g < 0.0f ? __fmul_rn(p, g) : g, r), u);
}

}  // namespace mq
