// Int8 rows for the W8A8 products (int8.cuh has the arithmetic).  One pass: a warp keeps its row in registers between
// the maximum and the quotients (rows of up to 8 KB); longer rows are read a second time, from L2.
// Bound by HBM: size + 1 bytes per element.
#include "int8.cuh"

namespace mq {
namespace {

using namespace int8;

__device__ __forceinline__ uint32_t warp_max(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }

// The row's 16-byte vectors i * 32 + lane, NV a lane.
template <typename T, int NV>
__global__ void __launch_bounds__(256)
quantize_rows(const T* __restrict__ x, int64_t stride, int64_t rows, int K, int8_t* __restrict__ q, float* __restrict__ scale) {
  constexpr int V = 16 / sizeof(T);
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int nvec = K / V;
  const uint4* src = reinterpret_cast<const uint4*>(x + row * stride);
  uint4 v[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int p = i * 32 + lane;
    v[i] = p < nvec ? src[p] : make_uint4(0u, 0u, 0u, 0u);
  }
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const T* e = reinterpret_cast<const T*>(&v[i]);
#pragma unroll
    for (int j = 0; j < V; ++j) top = max(top, abs_bits(to_float<T>(e[j])));
  }
  const RowScale r = row_scale(warp_max(top));
  if (lane == 0) scale[row] = r.scale;
  int8_t* dst = q + row * K;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int p = i * 32 + lane;
    if (p < nvec) {
      const T* e = reinterpret_cast<const T*>(&v[i]);
      uint32_t w[V / 4];
#pragma unroll
      for (int j = 0; j < V / 4; ++j) {
        w[j] = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b) w[j] |= ((uint32_t)quantize(to_float<T>(e[4 * j + b]), r) & 0xffu) << (8 * b);
      }
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

template <typename T>
int launch_quantize(const void* x, int64_t rows, int64_t K, int64_t stride, int8_t* q, float* scale, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const T* xs = reinterpret_cast<const T*>(x);
  const int64_t nvec = K / V;
  if (K % V == 0 && stride % V == 0 && aligned16(x) && (reinterpret_cast<uintptr_t>(q) & 7u) == 0 && nvec <= 32 * 16) {
    const unsigned blocks = (unsigned)((rows + 7) / 8);
#define MQ_QUANTIZE(NV) quantize_rows<T, NV><<<blocks, 256, 0, st>>>(xs, stride, rows, (int)K, q, scale)
    if (nvec <= 32) MQ_QUANTIZE(1);
    else if (nvec <= 32 * 2) MQ_QUANTIZE(2);
    else if (nvec <= 32 * 3) MQ_QUANTIZE(3);
    else if (nvec <= 32 * 4) MQ_QUANTIZE(4);
    else if (nvec <= 32 * 8) MQ_QUANTIZE(8);
    else MQ_QUANTIZE(16);
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
