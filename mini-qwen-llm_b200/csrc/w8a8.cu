// W8A8 products: int8 rows times int8 weights, int32 sums, a scale for each row and each output channel.
//   out[r, n] = round((float)(sum_k q[r, k] * w[e][n, k]) * row_scale[r] * channel_scale[e][n])
// and, with SwiGLU, h = round(silu(g) * u) of the unrounded products with the gate and the up weights.
// Follows the shapes of mini_qwen/kernels/moe_grouped_gemm.py:17-37 and mini_qwen/model/layers/moe.py:24-25; the
// reference has no 8-bit path.  The int32 sums are exact (K <= 131071: 128 * 128 * K < 2^31).
//
// This file: the entry points, and the kernel for what the CTA-pair kernel (w8a8_pair.cu) leaves: any size and alignment.
#include "w8a8.cuh"

namespace mq {

int device_sm_count();

// Tensor cores, CTA pairs (w8a8_pair.cu).
bool w8a8_pair_covers(const W8Args& A, bool swiglu);
int w8a8_pair(const W8Args& A, bool swiglu, int out_dtype, int32_t* d_status, cudaStream_t st);

// A few rows of floating-point numbers, quantised in the same launch (w8a8_rows.cu).
bool w8a8_rows_covers(const void* x, int x_dtype, int64_t stride, const void* w, int64_t M, int64_t N, int64_t K);
bool w8a8_rows_pays(int64_t M, int64_t N, int64_t K);
int w8a8_rows(const void* x, int x_dtype, int64_t stride, const int8_t* w, const float* w_scale, int64_t M, int64_t N, int64_t K,
              int out_dtype, void* out, cudaStream_t st);

namespace {

constexpr int G_N = 64;                            // columns of a tile

// 16 bytes [k, k + 16) of a row, zero past K: in one load where rows start at multiples of 16, else in words, put together
// from their aligned neighbours where rows start anywhere.  Nothing outside [first, last), the tensor, is read.
__device__ __forceinline__ int4 load_piece(const int8_t* row, int k, int K, int grid, const int8_t* first, const int8_t* last) {
  const int8_t* p = row + k;
  uint32_t w[4] = {};
  if (k + 16 <= K) {
    if (grid == 16) return *reinterpret_cast<const int4*>(p);
    const uint32_t off = (uint32_t)reinterpret_cast<uintptr_t>(p) & 3u;
    if (off == 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
      return make_int4((int)w[0], (int)w[1], (int)w[2], (int)w[3]);
    }
    const int8_t* at = p - off;
    if (at >= first && at + 20 <= last) {
      uint32_t v[5];
#pragma unroll
      for (int i = 0; i < 5; ++i) v[i] = reinterpret_cast<const uint32_t*>(at)[i];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(v[i], v[i + 1], 8 * off);
      return make_int4((int)w[0], (int)w[1], (int)w[2], (int)w[3]);
    }
  }
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (k + i < K) w[i >> 2] |= (uint32_t)(uint8_t)p[i] << (8 * (i & 3));
  return make_int4((int)w[0], (int)w[1], (int)w[2], (int)w[3]);
}

__device__ __forceinline__ void mma_s8(int (&c)[4], const int (&a)[4], int b0, int b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A tile of ROWS rows by 64 columns; blocks of KT bytes of k go through shared memory, the next one's pieces on their way in
// registers.  64 rows: a warp has 16 rows and 32 columns; 16 rows: it has 8 columns.  What bounds it is the latency of a
// block, about 2 us, so that few tiles take the larger blocks.  (Dot products of four bytes and single bytes off the grid, without
// loads ahead: 1 row of K 777, N 333 33 us, now 8; 512 rows of K 1333, N 1499 89 us, now 28.)
template <int ROWS, int KT, typename OutT, bool SWIGLU>
__global__ void __launch_bounds__(256) w8a8_generic_kernel(const W8Args A) {
  constexpr int SIDES = SWIGLU ? 2 : 1, LD = KT + 16, PIECES = KT / 16;                      // LD: no bank conflicts
  constexpr int XP = ROWS * PIECES / 256, WP = SIDES * G_N * PIECES / 256;                   // pieces of a thread
  constexpr int NT = ROWS == 64 ? 4 : 1;                                                     // 8-column tiles of a warp
  static_assert(XP >= 1 && WP >= 1, "a piece for each thread");
  __shared__ __align__(16) int8_t s_x[ROWS * LD];
  __shared__ __align__(16) int8_t s_w[SIDES * G_N * LD];
  __shared__ int s_at[2];                          // group, first row of the tile
  const int tid = threadIdx.x;
  if (A.offsets == nullptr) {
    if (tid == 0) { s_at[0] = 0; s_at[1] = (int)blockIdx.x * ROWS; }
  } else if (tid < 32) {                           // the group that holds row tile blockIdx.x
    int before = 0, group = -1, first = 0;
    for (int e0 = 0; e0 < A.E && group < 0; e0 += 32) {
      const int e = e0 + tid;
      const int lo = e < A.E ? w8_offset(A, e) : 0, n = e < A.E ? max(0, w8_offset(A, e + 1) - lo) : 0;
      const int tiles = (n + ROWS - 1) / ROWS;
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
        first = __shfl_sync(0xffffffffu, lo + at * ROWS, src);
      }
      before += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (tid == 0) { s_at[0] = group; s_at[1] = first; }
  }
  __syncthreads();
  const int group = s_at[0], row0 = s_at[1];
  if (group < 0) return;                           // past the last tile
  const int end = A.offsets == nullptr ? (int)A.S : w8_offset(A, group + 1);
  const int expert = group % A.period, col0 = (int)(blockIdx.z * gridDim.y + blockIdx.y) * G_N;
  if (col0 >= A.N) return;
  const int wrows = SIDES * A.N;
  const int8_t* const w = A.w + (size_t)expert * wrows * A.K;
  const float* ws = A.w_scale + (size_t)expert * wrows;
  const int8_t* const x_last = A.x + (size_t)A.T * A.K;
  const int8_t* const w_last = A.w + (size_t)A.period * wrows * A.K;
  // the thread's pieces: row (i * 256 + tid) / PIECES of the tile, piece tid % PIECES of the block
  const int piece = tid % PIECES;
  const int8_t *x_row[XP], *w_row[WP];
#pragma unroll
  for (int i = 0; i < XP; ++i) {
    const int row = row0 + (i * 256 + tid) / PIECES;
    x_row[i] = row < end ? A.x + w8_source(A, row) * A.K : nullptr;
  }
#pragma unroll
  for (int i = 0; i < WP; ++i) {
    const int n = (i * 256 + tid) / PIECES, col = col0 + n % G_N;
    w_row[i] = col < A.N ? w + (size_t)(n / G_N * A.N + col) * A.K : nullptr;
  }
  int4 px[XP], pw[WP];
  auto load = [&](int k0) {
    const int k = k0 + 16 * piece;
#pragma unroll
    for (int i = 0; i < XP; ++i)
      px[i] = x_row[i] != nullptr && k < A.K ? load_piece(x_row[i], k, A.K, A.grid, A.x, x_last) : make_int4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < WP; ++i)
      pw[i] = w_row[i] != nullptr && k < A.K ? load_piece(w_row[i], k, A.K, A.grid, A.w, w_last) : make_int4(0, 0, 0, 0);
  };
  const int lane = tid & 31, warp = tid >> 5, g = lane >> 2, q4 = lane & 3;
  const int wr = ROWS == 64 ? warp / 2 * 16 : 0, wc = ROWS == 64 ? warp % 2 * 32 : warp * 8;
  int acc[SIDES][NT][4] = {};
  load(0);
  for (int k0 = 0; k0 < A.K; k0 += KT) {
#pragma unroll
    for (int i = 0; i < XP; ++i) *reinterpret_cast<int4*>(s_x + (i * 256 + tid) / PIECES * LD + 16 * piece) = px[i];
#pragma unroll
    for (int i = 0; i < WP; ++i) *reinterpret_cast<int4*>(s_w + (i * 256 + tid) / PIECES * LD + 16 * piece) = pw[i];
    __syncthreads();
    if (k0 + KT < A.K) load(k0 + KT);
#pragma unroll
    for (int k = 0; k < KT; k += 32) {
      auto word = [&](const int8_t* rows, int r, int at) { return *reinterpret_cast<const int*>(rows + r * LD + k + at); };
      const int a[4] = {word(s_x, wr + g, 4 * q4), word(s_x, wr + 8 + g, 4 * q4), word(s_x, wr + g, 16 + 4 * q4),
                        word(s_x, wr + 8 + g, 16 + 4 * q4)};
#pragma unroll
      for (int side = 0; side < SIDES; ++side)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const int n = side * G_N + wc + 8 * j + g;
          mma_s8(acc[side][j], a, word(s_w, n, 4 * q4), word(s_w, n, 16 + 4 * q4));
        }
    }
    __syncthreads();
  }
  OutT* out = reinterpret_cast<OutT*>(A.out);
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int row = row0 + wr + 8 * half + g;
    if (row >= end) continue;
    const float sr = A.x_scale[w8_source(A, row)];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int col = col0 + wc + 8 * j + 2 * q4 + i;
        if (col >= A.N) continue;
        float v = w8_value(acc[0][j][2 * half + i], sr, ws[col]);
        if (SWIGLU) v = w8_swiglu<OutT>(v, w8_value(acc[SIDES - 1][j][2 * half + i], sr, ws[A.N + col]));
        out[(size_t)row * A.N + col] = from_float<OutT>(v);
      }
  }
}

template <int ROWS, int KT, typename OutT>
int launch_generic_rows(const W8Args& A, bool swiglu, cudaStream_t st) {
  const int64_t tiles = A.S / ROWS + (A.offsets == nullptr ? 1 : (A.E < A.S ? A.E : A.S));
  const int cols = (A.N + G_N - 1) / G_N, most = 65535;              // of a grid's second and third dimension
  const dim3 grid((unsigned)tiles, (unsigned)(cols < most ? cols : most), (unsigned)((cols + most - 1) / most));
  if (swiglu) w8a8_generic_kernel<ROWS, KT, OutT, true><<<grid, 256, 0, st>>>(A);
  else w8a8_generic_kernel<ROWS, KT, OutT, false><<<grid, 256, 0, st>>>(A);
  return check_launch();
}

// Tiles of 16 rows where groups have no more, or where those of 64 would leave multiprocessors without one (K 1333, N 1499:
// 100 rows 17.6 us, 24.5 in tiles of 64; 300 rows, 120 tiles 23.5 : 25.0; 512 rows, 192 tiles 39.5 : 28.2; K 777, N 999:
// 3000 rows 74.3 : 41.0).
template <typename OutT>
int launch_generic(const W8Args& A, bool swiglu, cudaStream_t st) {
  const int64_t cols = (A.N + G_N - 1) / G_N, groups = A.E < A.S ? A.E : A.S, rows = (A.S + groups - 1) / groups;
  if (rows > 16 && (rows + 63) / 64 * groups * cols >= device_sm_count()) return launch_generic_rows<64, 128, OutT>(A, swiglu, st);
  return launch_generic_rows<16, 256, OutT>(A, swiglu, st);
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
  A.grid = ((A.K | (int)(reinterpret_cast<uintptr_t>(A.x) & 15u) | (int)(reinterpret_cast<uintptr_t>(A.w) & 15u)) & 15) == 0 ? 16 : 1;
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
  // without a workspace a few rows take one launch, whatever their channels
  const bool room = workspace != nullptr && aligned16(workspace) && workspace_bytes >= mq_w8a8_workspace_bytes(M, Kd, 0);
  if (w8a8_rows_covers(x, x_dtype, row_stride, qweight, M, N, Kd) && (w8a8_rows_pays(M, N, Kd) || !room)) {
    if (h_launches) *h_launches = 1;
    return w8a8_rows(x, x_dtype, row_stride, qweight, w_scale, M, N, Kd, out_dtype, out, reinterpret_cast<cudaStream_t>(stream));
  }
  if (!workspace || !aligned16(workspace)) return MQ_ERR_INVALID_ARGUMENT;
  if (!room) return MQ_ERR_WORKSPACE_TOO_SMALL;
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
