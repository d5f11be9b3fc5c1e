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
  int words;                   // rows of x and w start at multiples of four bytes
  void* out;                   // [S, N]
};

// Offsets outside 0..S, and permutation entries outside x, are the caller's mistake; they must not become addresses.
__device__ __forceinline__ int w8_offset(const W8Args& A, int e) { return min(max(A.offsets[e], 0), A.S); }
__device__ __forceinline__ size_t w8_source(const W8Args& A, int row) {
  return A.perm == nullptr ? (size_t)row : (size_t)min(max(A.perm[row], 0) / A.top_k, A.T - 1);
}

// The sum may pass 2^24, so the conversion rounds; with the two products that is 1.5 * 2^-23 in all at most.
__device__ __forceinline__ float w8_value(int sum, float row_scale, float channel_scale) {
  return __fmul_rn(__fmul_rn(__int2float_rn(sum), row_scale), channel_scale);
}
// silu(g) * u, with the exponential of -|g| so that nothing overflows and the quotient's denominator is in 1..2.
__device__ __forceinline__ float w8_swiglu(float g, float u) {
  const float p = expf(-fabsf(g));
  return __fdividef(g < 0.0f ? p * g : g, 1.0f + p) * u;
}

}  // namespace mq
