// W8A8 products: int8 rows times int8 weights, int32 sums, a scale for each row and each output channel.
//   out[r, n] = round((float)(sum_k q[r, k] * w[e][n, k]) * row_scale[r] * channel_scale[e][n])
// and, with SwiGLU, h = round(silu(g) * u) of the unrounded products with the gate and the up weights.
// Follows the shapes of mini_qwen/kernels/moe_grouped_gemm.py:17-37 and mini_qwen/model/layers/moe.py:24-25; the
// reference has no 8-bit path.  The int32 sums are exact (K <= 131071: 128 * 128 * K < 2^31).
//
// This file: the entry points, and the kernel for what the tensor-core kernel (w8a8_pair.cu) leaves: any size and alignment
// (dot products of four bytes, tiles of 64 rows by 64 columns through shared memory).
#include "w8a8.cuh"

namespace mq {

// Tensor cores, CTA pairs (w8a8_pair.cu).
bool w8a8_pair_covers(const W8Args& A, bool swiglu);
int w8a8_pair(const W8Args& A, bool swiglu, int out_dtype, int32_t* d_status, cudaStream_t st);

// A few rows of floating-point numbers, quantised in the same launch (w8a8_rows.cu).
bool w8a8_rows_covers(const void* x, int x_dtype, int64_t stride, const void* w, int64_t M, int64_t N, int64_t K);
int w8a8_rows(const void* x, int x_dtype, int64_t stride, const int8_t* w, const float* w_scale, int64_t M, int64_t N, int64_t K,
              int out_dtype, void* out, cudaStream_t st);

namespace {

constexpr int G_M = 64, G_N = 64, G_K = 64;        // rows, columns and bytes of k of a tile
constexpr int G_LD = G_K / 4 + 1;                  // words of a staged row, padded

// Bytes [k, k + 4) of a row, zero past K.
__device__ __forceinline__ int load_word(const int8_t* row, int k, int K, bool words) {
  if (words && k + 4 <= K) return *reinterpret_cast<const int*>(row + k);
  uint32_t w = 0;
#pragma unroll
  for (int b = 0; b < 4; ++b)
    if (k + b < K) w |= (uint32_t)(uint8_t)row[k + b] << (8 * b);
  return (int)w;
}

template <typename OutT, bool SWIGLU>
__global__ void __launch_bounds__(256) w8a8_generic_kernel(const W8Args A) {
  __shared__ int s_a[G_M * G_LD], s_b[(SWIGLU ? 2 : 1) * G_N * G_LD];
  __shared__ int s_at[2];                          // group, first row of the tile
  const int tid = threadIdx.x;
  if (A.offsets == nullptr) {
    if (tid == 0) { s_at[0] = 0; s_at[1] = (int)blockIdx.x * G_M; }
  } else if (tid < 32) {                           // the group that holds row tile blockIdx.x
    int before = 0, group = -1, first = 0;
    for (int e0 = 0; e0 < A.E && group < 0; e0 += 32) {
      const int e = e0 + tid;
      const int lo = e < A.E ? w8_offset(A, e) : 0, n = e < A.E ? max(0, w8_offset(A, e + 1) - lo) : 0;
      const int tiles = (n + G_M - 1) / G_M;
      int incl = tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (tid >= o) incl += v;
      }
      const int at = (int)blockIdx.x - before - (incl - tiles);
      const unsigned hit = __ballot_sync(0xffffffffu, at >= 0 && at < tiles);
      if (hit != 0) {
        const int src = __ffs(hit) - 1;
        group = e0 + src;
        first = __shfl_sync(0xffffffffu, lo + at * G_M, src);
      }
      before += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (tid == 0) { s_at[0] = group; s_at[1] = first; }
  }
  __syncthreads();
  const int group = s_at[0], row0 = s_at[1];
  if (group < 0) return;                           // past the last tile
  const int end = A.offsets == nullptr ? (int)A.S : w8_offset(A, group + 1);
  const int expert = group % A.period, col0 = (int)blockIdx.y * G_N;
  const int wrows = SWIGLU ? 2 * A.N : A.N;
  const int8_t* w = A.w + (size_t)expert * wrows * A.K;
  const float* ws = A.w_scale + (size_t)expert * wrows;
  const int tx = tid & 15, ty = tid >> 4;
  int acc[SWIGLU ? 2 : 1][4][4] = {};
  for (int k0 = 0; k0 < A.K; k0 += G_K) {
    for (int i = tid; i < G_M * (G_K / 4); i += 256) {
      const int r = i / (G_K / 4), c = i % (G_K / 4), row = row0 + r;
      s_a[r * G_LD + c] = row < end ? load_word(A.x + w8_source(A, row) * A.K, k0 + 4 * c, A.K, A.words) : 0;
    }
#pragma unroll
    for (int half = 0; half < (SWIGLU ? 2 : 1); ++half)
      for (int i = tid; i < G_N * (G_K / 4); i += 256) {
        const int n = i / (G_K / 4), c = i % (G_K / 4), col = col0 + n;
        s_b[(half * G_N + n) * G_LD + c] =
            col < A.N ? load_word(w + (size_t)(half * A.N + col) * A.K, k0 + 4 * c, A.K, A.words) : 0;
      }
    __syncthreads();
#pragma unroll 4
    for (int c = 0; c < G_K / 4; ++c) {
      int a[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = s_a[(ty + 16 * i) * G_LD + c];
#pragma unroll
      for (int half = 0; half < (SWIGLU ? 2 : 1); ++half)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int b = s_b[(half * G_N + tx + 16 * j) * G_LD + c];
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[half][i][j] = __dp4a(a[i], b, acc[half][i][j]);
        }
    }
    __syncthreads();
  }
  OutT* out = reinterpret_cast<OutT*>(A.out);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = row0 + ty + 16 * i;
    if (row >= end) continue;
    const float sr = A.x_scale[w8_source(A, row)];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int col = col0 + tx + 16 * j;
      if (col >= A.N) continue;
      float v = w8_value(acc[0][i][j], sr, ws[col]);
      if (SWIGLU) v = w8_swiglu(v, w8_value(acc[SWIGLU ? 1 : 0][i][j], sr, ws[A.N + col]));
      out[(size_t)row * A.N + col] = from_float<OutT>(v);
    }
  }
}

template <typename OutT>
int launch_generic(const W8Args& A, bool swiglu, cudaStream_t st) {
  const int64_t tiles = A.S / G_M + (A.offsets == nullptr ? 1 : (A.E < A.S ? A.E : A.S));
  const int64_t cols = (A.N + G_N - 1) / G_N;
  if (cols > 65535) return MQ_ERR_UNSUPPORTED_SHAPE;
  const dim3 grid((unsigned)tiles, (unsigned)cols);
  if (swiglu) w8a8_generic_kernel<OutT, true><<<grid, 256, 0, st>>>(A);
  else w8a8_generic_kernel<OutT, false><<<grid, 256, 0, st>>>(A);
  return check_launch();
}

int w8a8_dispatch(W8Args A, bool swiglu, int out_dtype, int32_t* d_status, cudaStream_t st) {
  if (A.S < 0 || A.T < 0 || A.E <= 0 || A.period <= 0 || A.period > A.E || A.N <= 0 || A.K <= 0 || A.top_k <= 0 ||
      !valid_dtype(out_dtype))
    return MQ_ERR_INVALID_ARGUMENT;
  if (A.S == 0) return MQ_OK;
  if (A.T == 0 || !A.x || !A.x_scale || !A.w || !A.w_scale || !A.out) return MQ_ERR_INVALID_ARGUMENT;
  if (A.perm == nullptr && A.T < A.S) return MQ_ERR_INVALID_ARGUMENT;
  if (A.top_k > 1) {                               // m = ceil(2^(32 + s) / k) with 2^s >= k / 2 divides every n < 2^31 exactly
    int shift = 0;
    while ((2ull << shift) < (unsigned long long)A.top_k) ++shift;
    A.k_mul = (uint32_t)(((1ull << (32 + shift)) + A.top_k - 1) / A.top_k);
    A.k_shift = (uint32_t)shift;
  }
  if (w8a8_pair_covers(A, swiglu)) return w8a8_pair(A, swiglu, out_dtype, d_status, st);
  A.words = ((A.K | (int)(reinterpret_cast<uintptr_t>(A.x) & 3u) | (int)(reinterpret_cast<uintptr_t>(A.w) & 3u)) & 3) == 0;
  if (out_dtype == MQ_F32) return launch_generic<float>(A, swiglu, st);
  if (out_dtype == MQ_BF16) return launch_generic<__nv_bfloat16>(A, swiglu, st);
  return launch_generic<__half>(A, swiglu, st);
}

// Sizes of the kernels' 32-bit arithmetic.
bool sizes_fit(int64_t S, int64_t T, int64_t E, int64_t top_k, int64_t N, int64_t K) {
  const int64_t m = (int64_t)1 << 30;
  return S < m && T < m && E < m && top_k < m && N < (m >> 1) && K <= 131071;
}

}  // namespace
}  // namespace mq

extern "C" int mq_w8a8_grouped_gemm(const int8_t* x, const float* x_scale, const int8_t* qweight, const float* w_scale,
                                    const int32_t* offsets, int64_t S, int64_t E, int64_t weight_period, int64_t N,
                                    int64_t Kd, int out_dtype, void* out, int32_t* d_status, void* stream) {
  using namespace mq;
  if (S > 0 && !offsets) return MQ_ERR_INVALID_ARGUMENT;
  if (!sizes_fit(S, S, E, 1, N, Kd)) return MQ_ERR_UNSUPPORTED_SHAPE;
  return w8a8_dispatch(W8Args{x, x_scale, qweight, w_scale, offsets, nullptr, (int)S, (int)S, 1, (int)E, (int)weight_period,
                              (int)N, (int)Kd, out, 0, 0, 0},
                       false, out_dtype, d_status, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int mq_w8a8_linear(const int8_t* x, const float* x_scale, const int8_t* qweight, const float* w_scale, int64_t M,
                              int64_t N, int64_t Kd, int out_dtype, void* out, int32_t* d_status, void* stream) {
  using namespace mq;
  if (!sizes_fit(M, M, 1, 1, N, Kd)) return MQ_ERR_UNSUPPORTED_SHAPE;
  return w8a8_dispatch(W8Args{x, x_scale, qweight, w_scale, nullptr, nullptr, (int)M, (int)M, 1, 1, 1, (int)N, (int)Kd, out, 0, 0, 0},
                       false, out_dtype, d_status, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int mq_w8a8_grouped_swiglu(const int8_t* x, const float* x_scale, const int32_t* perm, int64_t T, int64_t top_k,
                                      const int8_t* w_gate_up, const float* w_scale, const int32_t* offsets, int64_t S,
                                      int64_t E, int64_t weight_period, int64_t I, int64_t H, int out_dtype, void* h,
                                      int32_t* d_status, void* stream) {
  using namespace mq;
  if (S > 0 && !offsets) return MQ_ERR_INVALID_ARGUMENT;
  if (!sizes_fit(S, T, E, top_k, I, H)) return MQ_ERR_UNSUPPORTED_SHAPE;
  return w8a8_dispatch(W8Args{x, x_scale, w_gate_up, w_scale, offsets, perm, (int)S, (int)T, (int)top_k, (int)E,
                              (int)weight_period, (int)I, (int)H, h, 0, 0, 0},
                       true, out_dtype, d_status, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" size_t mq_w8a8_workspace_bytes(int64_t rows, int64_t Kd, int64_t groups) {
  if (rows < 0 || Kd < 0 || groups < 0) return 256;
  auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
  return up((size_t)(rows * Kd)) + up((size_t)rows * 4) + up((size_t)(groups + 1) * 4);
}

namespace {
struct W8Space {                                   // a workspace cut up
  int8_t* q;
  float* scale;
  int32_t* offsets;
  W8Space(void* p, int64_t rows, int64_t Kd) {
    auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
    uint8_t* b = reinterpret_cast<uint8_t*>(p);
    q = reinterpret_cast<int8_t*>(b);
    scale = reinterpret_cast<float*>(b + up((size_t)(rows * Kd)));
    offsets = reinterpret_cast<int32_t*>(b + up((size_t)(rows * Kd)) + up((size_t)rows * 4));
  }
};
}  // namespace

extern "C" int mq_w8a8_linear_x(const void* x, int x_dtype, int64_t row_stride, const int8_t* qweight, const float* w_scale,
                                int64_t M, int64_t N, int64_t Kd, int out_dtype, void* workspace, size_t workspace_bytes,
                                void* out, int32_t* d_status, int32_t* h_launches, void* stream) {
  using namespace mq;
  if (h_launches) *h_launches = 0;
  if (M < 0 || N <= 0 || Kd <= 0 || row_stride < 0 || !valid_dtype(x_dtype) || !valid_dtype(out_dtype))
    return MQ_ERR_INVALID_ARGUMENT;
  if (!sizes_fit(M, M, 1, 1, N, Kd)) return MQ_ERR_UNSUPPORTED_SHAPE;
  if (M == 0) return MQ_OK;
  if (!x || !qweight || !w_scale || !out) return MQ_ERR_INVALID_ARGUMENT;
  if (w8a8_rows_covers(x, x_dtype, row_stride, qweight, M, N, Kd)) {
    if (h_launches) *h_launches = 1;
    return w8a8_rows(x, x_dtype, row_stride, qweight, w_scale, M, N, Kd, out_dtype, out, reinterpret_cast<cudaStream_t>(stream));
  }
  if (!workspace || !aligned16(workspace)) return MQ_ERR_INVALID_ARGUMENT;
  if (workspace_bytes < mq_w8a8_workspace_bytes(M, Kd, 0)) return MQ_ERR_WORKSPACE_TOO_SMALL;
  const W8Space ws(workspace, M, Kd);
  const int rc = mq_quantize_rows_int8(x, x_dtype, M, Kd, row_stride, ws.q, ws.scale, stream);
  if (rc != MQ_OK) return rc;
  if (h_launches) *h_launches = 2;
  return mq_w8a8_linear(ws.q, ws.scale, qweight, w_scale, M, N, Kd, out_dtype, out, d_status, stream);
}

extern "C" int mq_w8a8_grouped_x(const void* x, int x_dtype, int64_t row_stride, const int32_t* perm, int64_t T, int64_t top_k,
                                 const int8_t* qweight, const float* w_scale, const void* offsets, int offsets_are_64, int64_t S,
                                 int64_t E, int64_t weight_period, int64_t N, int64_t Kd, int swiglu, int zero_uncovered,
                                 int out_dtype, void* workspace, size_t workspace_bytes, void* out, int32_t* d_status,
                                 int32_t* h_launches, void* stream) {
  using namespace mq;
  if (h_launches) *h_launches = 0;
  if (S < 0 || T < 0 || E <= 0 || N <= 0 || Kd <= 0 || row_stride < 0 || !valid_dtype(x_dtype) || !valid_dtype(out_dtype) ||
      weight_period <= 0 || weight_period > E || top_k <= 0 || (perm != nullptr && !swiglu))
    return MQ_ERR_INVALID_ARGUMENT;
  if (!sizes_fit(S, T, E, top_k, N, Kd)) return MQ_ERR_UNSUPPORTED_SHAPE;
  if (S == 0) return MQ_OK;
  if (T == 0 || !x || !qweight || !w_scale || !offsets || !out || !workspace || !aligned16(workspace) ||
      (perm == nullptr && T < S))
    return MQ_ERR_INVALID_ARGUMENT;
  if (workspace_bytes < mq_w8a8_workspace_bytes(T, Kd, E)) return MQ_ERR_WORKSPACE_TOO_SMALL;
  const W8Space ws(workspace, T, Kd);
  int n = 2;
  const int32_t* off = reinterpret_cast<const int32_t*>(offsets);
  if (offsets_are_64 || zero_uncovered) {
    const int rc = mq_grouped_prepare(offsets, offsets_are_64, S, E, N, out_dtype, zero_uncovered ? out : nullptr,
                                      offsets_are_64 ? ws.offsets : nullptr, nullptr, stream);
    if (rc != MQ_OK) return rc;
    if (offsets_are_64) off = ws.offsets;
    ++n;
  }
  int rc = mq_quantize_rows_int8(x, x_dtype, T, Kd, row_stride, ws.q, ws.scale, stream);
  if (rc != MQ_OK) return rc;
  if (h_launches) *h_launches = n;
  if (swiglu)
    return mq_w8a8_grouped_swiglu(ws.q, ws.scale, perm, T, top_k, qweight, w_scale, off, S, E, weight_period, N, Kd, out_dtype,
                                  out, d_status, stream);
  return mq_w8a8_grouped_gemm(ws.q, ws.scale, qweight, w_scale, off, S, E, weight_period, N, Kd, out_dtype, out, d_status, stream);
}
