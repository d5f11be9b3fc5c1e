// Int8 rows for the W8A8 products (int8.cuh has the arithmetic).  One pass: a warp, some warps or a CTA keep their row
// in registers between the maximum and the quotients; rows of over 32 KB, or off the 16-byte grid, are read a second time.
// Bound by HBM: size + 1 bytes per element (32768 x 768 bf16 18.2 us, 4.2 TB/s; each further 8192 rows 3.7 us, 5.1 TB/s; fp32 27 us,
// 4.7 TB/s, 32768 x 2048 of it 55 us, 6.1 TB/s).  Rows off the grid are bound by their loads, an element each (bf16, 32768 x 2047
// 114 us, 1.8 TB/s; 8192 x 20000, over 32 KB, 249 us).
#include <string.h>

#include "int8.cuh"

namespace mq {
namespace {

using namespace int8;

__device__ __forceinline__ uint32_t warp_max(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }

// The largest magnitude of a lane's vectors, as the bits of an fp32 number.  16-bit numbers are compared two at a time, as
// integers.
template <typename T, int NV>
__device__ __forceinline__ uint32_t largest(const uint4 (&v)[NV]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (sizeof(T) == 4) top = max(top, w[j] & 0x7fffffffu);
      else top = __vmaxu2(top, w[j] & 0x7fff7fffu);
    }
  }
  if (sizeof(T) == 4) return top;
  const uint16_t one = (uint16_t)max(top & 0xffffu, top >> 16);
  T value;
  memcpy(&value, &one, sizeof(one));
  return abs_bits(to_float<T>(value));
}

// TPR threads a row, NV of its 16-byte vectors each: a warp a row, some warps, or a CTA of 256.
template <typename T, int NV, int TPR>
__global__ void __launch_bounds__(256)
quantize_rows(const T* __restrict__ x, int64_t stride, int64_t rows, int K, int8_t* __restrict__ q, float* __restrict__ scale) {
  constexpr int V = 16 / sizeof(T);
  const int at = (int)threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
  const bool live = row < rows;
  if (TPR == 32 && !live) return;
  const int nvec = K / V;
  const uint4* src = reinterpret_cast<const uint4*>(x + row * stride);
  uint4 v[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int p = i * TPR + at;
    v[i] = live && p < nvec ? src[p] : make_uint4(0u, 0u, 0u, 0u);
  }
  uint32_t top = warp_max(largest<T, NV>(v));
  if (TPR > 32) {
    __shared__ uint32_t part[8];
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
    __syncthreads();
    if (!live) return;
#pragma unroll
    for (int i = 0; i < TPR / 32; ++i) top = max(top, part[threadIdx.x / TPR * (TPR / 32) + i]);
  }
  const RowScale r = row_scale(top);
  if (at == 0) scale[row] = r.scale;
  int8_t* dst = q + row * K;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int p = i * TPR + at;
    if (p < nvec) {
      const T* e = reinterpret_cast<const T*>(&v[i]);
      float f[V];
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] = to_float<T>(e[j]);
      uint32_t w[V / 4];
      quantize<V>(f, r, w);
      if (V == 8) *reinterpret_cast<uint2*>(dst + p * 8) = make_uint2(w[0], w[V / 4 - 1]);
      else *reinterpret_cast<uint32_t*>(dst + p * 4) = w[0];
    }
  }
}

// Any length, stride and alignment: one CTA a row, element by element.
template <typename T>
__global__ void __launch_bounds__(256)
quantize_any_rows(const T* __restrict__ x, int64_t stride, int64_t K, int8_t* __restrict__ q, float* __restrict__ scale) {
  __shared__ uint32_t part[8];
  const T* src = x + (int64_t)blockIdx.x * stride;
  int8_t* dst = q + (int64_t)blockIdx.x * K;
  uint32_t top = 0;
  for (int64_t k = threadIdx.x; k < K; k += 256) top = max(top, abs_bits(to_float<T>(src[k])));
  top = warp_max(top);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, part[i]);
  const RowScale r = row_scale(top);
  if (threadIdx.x == 0) scale[blockIdx.x] = r.scale;
  for (int64_t k = threadIdx.x; k < K; k += 256) dst[k] = (int8_t)quantize(to_float<T>(src[k]), r);
}

// Few rows finish sooner with many threads each, many rows with many loads under way in each thread (bf16, 2048 columns: 2500
// rows 6.5 us with 256 threads, 7.0 with 64; 4096 rows 9.2 : 8.9; 32768 rows 60.8 : 44.7).
constexpr int64_t MANY_ROWS = 4096;

template <typename T>
int launch_quantize(const void* x, int64_t rows, int64_t K, int64_t stride, int8_t* q, float* scale, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const T* xs = reinterpret_cast<const T*>(x);
  const int64_t nvec = K / V;
  if (K % V == 0 && stride % V == 0 && aligned16(x) && (reinterpret_cast<uintptr_t>(q) & 7u) == 0 && nvec <= 256 * 8) {
#define MQ_QUANTIZE(NV, TPR) \
  quantize_rows<T, NV, TPR><<<(unsigned)((rows + 256 / TPR - 1) / (256 / TPR)), 256, 0, st>>>(xs, stride, rows, (int)K, q, scale)
    if (nvec <= 32) MQ_QUANTIZE(1, 32);
    else if (nvec <= 32 * 2) MQ_QUANTIZE(2, 32);
    else if (nvec <= 32 * 3) MQ_QUANTIZE(3, 32);
    else if (nvec <= 32 * 4) MQ_QUANTIZE(4, 32);
    else if (nvec <= 256 && rows >= MANY_ROWS) MQ_QUANTIZE(4, 64);
    else if (nvec <= 256) MQ_QUANTIZE(1, 256);
    else if (nvec <= 256 * 2 && rows >= MANY_ROWS) MQ_QUANTIZE(4, 128);
    else if (nvec <= 256 * 2) MQ_QUANTIZE(2, 256);
    else if (nvec <= 256 * 4) MQ_QUANTIZE(4, 256);
    else MQ_QUANTIZE(8, 256);
#undef MQ_QUANTIZE
  } else {
    quantize_any_rows<T><<<(unsigned)rows, 256, 0, st>>>(xs, stride, K, q, scale);
  }
  return check_launch();
}

}  // namespace
}  // namespace mq

extern "C" int mq_quantize_rows_int8(const void* x, int dtype, int64_t rows, int64_t K, int64_t row_stride, int8_t* q,
                                     float* scale, void* stream) {
  using namespace mq;
  if (rows < 0 || K <= 0 || row_stride < 0 || !valid_dtype(dtype)) return MQ_ERR_INVALID_ARGUMENT;
  if (rows > 0x7fffffff) return MQ_ERR_UNSUPPORTED_SHAPE;
  if (rows == 0) return MQ_OK;
  if (!x || !q || !scale) return MQ_ERR_INVALID_ARGUMENT;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == MQ_F32) return launch_quantize<float>(x, rows, K, row_stride, q, scale, st);
  if (dtype == MQ_BF16) return launch_quantize<__nv_bfloat16>(x, rows, K, row_stride, q, scale, st);
  return launch_quantize<__half>(x, rows, K, row_stride, q, scale, st);
}
