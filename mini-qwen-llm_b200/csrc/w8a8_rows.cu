// W8A8 product of a few rows (up to 16), with the quantisation of the rows in the same launch: an attention or expert-sized
// linear while sequences are being decoded.
//
// What bounds it is reading the weights once, and at these sizes (8 MB take 1.3 us) the latencies around that.  A CTA takes 16
// weight rows, its eight warps share k in pieces of 256; a lane's 16-byte pieces of rows g and g + 8 are, with k in a suitable
// order, fragments of mma.sync (m16n8k32, tokens are the 8 columns), so the weights go from memory to the tensor cores without
// a detour, and the first pieces are on their way while the CTA quantises the rows for itself (a few KB from L2, into shared
// memory).  The warps' int32 sums meet in shared memory.
// One row, K 2048, N 4096: 6.9 us in a graph, where two launches take 12.3.
#include "int8.cuh"
#include "w8a8.cuh"

namespace mq {

int device_sm_count();

namespace {

using namespace int8;

constexpr int R_WARPS = 8, R_STEPS = 4;            // warps; steps of 64 k a warp has in flight

__device__ __forceinline__ uint4 ld_weights(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%0, %1, %2, %3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Eight values from an offset that is a multiple of eight.
__device__ __forceinline__ void load_eight(const void* p, int dt, size_t i, float (&v)[8]) {
  if (dt == MQ_F32) {
    const float4* q = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i);
    const float4 a = __ldg(q), b = __ldg(q + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    return;
  }
  const uint4 a = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p) + i));
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (dt == MQ_BF16) {
      v[2 * j] = __uint_as_float(w[j] << 16);
      v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
      v[2 * j] = f.x;
      v[2 * j + 1] = f.y;
    }
  }
}

struct RowsArgs {
  const void* x;               // [M] rows of K, `stride` elements apart
  const int8_t* w;             // [N, K]
  const float* w_scale;
  void* out;                   // [M, N]
  int64_t stride;
  int M, N, K, dtype, out_dtype;
};

template <int OCT>
__global__ void __launch_bounds__(R_WARPS * 32) w8a8_rows_kernel(const RowsArgs A) {
  extern __shared__ __align__(16) uint8_t rows_smem[];          // [M][K + 16] quantised rows, then the warps' sums
  __shared__ uint32_t s_top[16 * R_WARPS];
  __shared__ float s_scale[16];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q4 = lane & 3;
  const int M = A.M, N = A.N, K = A.K, ld = K + 16, row0 = (int)blockIdx.x * 16;
  const int8_t* w0 = A.w + (size_t)min(row0 + g, N - 1) * K;    // rows past the last are computed from it, and not stored
  const int8_t* w8 = A.w + (size_t)min(row0 + g + 8, N - 1) * K;
  uint4 a[R_STEPS][2];
  auto fetch = [&](int k0) {
#pragma unroll
    for (int s = 0; s < R_STEPS; ++s) {
      const int k = k0 + 64 * s + 16 * q4;
      a[s][0] = k < K ? ld_weights(w0 + k) : make_uint4(0u, 0u, 0u, 0u);
      a[s][1] = k < K ? ld_weights(w8 + k) : make_uint4(0u, 0u, 0u, 0u);
    }
  };
  int k0 = warp * (64 * R_STEPS);
  fetch(k0);

  // ------------------------------------------------------------------ the rows
  // `share` warps to a row; every thread keeps to the pieces it looked at, which are in the first-level cache the second time
  const int share = M == 1 ? R_WARPS : M == 2 ? 4 : M <= 4 ? 2 : 1;
  const int part = warp % share, first = warp / share, rows_at_once = R_WARPS / share;
  for (int m = first; m < M; m += rows_at_once) {
    uint32_t top = 0;
    for (int k = 8 * (part * 32 + lane); k < K; k += 256 * share) {
      float v[8];
      load_eight(A.x, A.dtype, m * A.stride + k, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, abs_bits(v[j]));
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) s_top[m * R_WARPS + part] = top;
  }
  __syncthreads();
  for (int m = first; m < M; m += rows_at_once) {
    uint32_t top = 0;
    for (int i = 0; i < share; ++i) top = max(top, s_top[m * R_WARPS + i]);
    const RowScale r = row_scale(top);
    if (part == 0 && lane == 0) s_scale[m] = r.scale;
    for (int k = 8 * (part * 32 + lane); k < K; k += 256 * share) {
      float v[8];
      uint32_t q[2];
      load_eight(A.x, A.dtype, m * A.stride + k, v);
      quantize<8>(v, r, q);
      *reinterpret_cast<uint2*>(rows_smem + (size_t)m * ld + k) = make_uint2(q[0], q[1]);
    }
  }
  __syncthreads();

  // ------------------------------------------------------------------ products
  int acc[OCT][4] = {};
  for (; k0 < K; k0 += R_WARPS * 64 * R_STEPS) {
    uint4 c[R_STEPS][2];
#pragma unroll
    for (int s = 0; s < R_STEPS; ++s) {
      c[s][0] = a[s][0];
      c[s][1] = a[s][1];
    }
    fetch(k0 + R_WARPS * 64 * R_STEPS);
    __syncwarp();
#pragma unroll
    for (int s = 0; s < R_STEPS; ++s) {
      const int k = k0 + 64 * s + 16 * q4;
#pragma unroll
      for (int o = 0; o < OCT; ++o) {
        const bool live = 8 * o + g < M && k < K;
        const uint4 b = live ? *reinterpret_cast<const uint4*>(rows_smem + (size_t)(8 * o + g) * ld + k) : make_uint4(0u, 0u, 0u, 0u);
        __syncwarp();
        mma_s8(acc[o], c[s][0].x, c[s][1].x, c[s][0].y, c[s][1].y, b.x, b.y);
        mma_s8(acc[o], c[s][0].z, c[s][1].z, c[s][0].w, c[s][1].w, b.z, b.w);
      }
    }
  }
  int4* sums = reinterpret_cast<int4*>(rows_smem + (((size_t)M * ld + 15) & ~(size_t)15));      // [warp][octet][lane]
#pragma unroll
  for (int o = 0; o < OCT; ++o) sums[(warp * OCT + o) * 32 + lane] = make_int4(acc[o][0], acc[o][1], acc[o][2], acc[o][3]);
  __syncthreads();
  for (int i = tid; i < OCT * 128; i += R_WARPS * 32) {
    // entry: (token, row), rows next to one another: where they lie in the fragments
    const int row = i % 16, tok = i / 16, o = tok / 8;
    const int at = (row & 7) * 4 + (tok & 7) / 2, reg = (row >> 3) * 2 + (tok & 1);
    int sum = 0;
#pragma unroll
    for (int w = 0; w < R_WARPS; ++w) sum += reinterpret_cast<const int*>(sums)[((w * OCT + o) * 32 + at) * 4 + reg];
    if (tok >= M || row0 + row >= N) continue;
    const float v = w8_value(sum, s_scale[tok], A.w_scale[row0 + row]);
    const size_t to = (size_t)tok * N + row0 + row;
    if (A.out_dtype == MQ_F32) reinterpret_cast<float*>(A.out)[to] = v;
    else if (A.out_dtype == MQ_BF16) reinterpret_cast<__nv_bfloat16*>(A.out)[to] = __float2bfloat16_rn(v);
    else reinterpret_cast<__half*>(A.out)[to] = __float2half_rn(v);
  }
}

size_t rows_smem_bytes(int64_t M, int64_t K) { return (size_t)M * (K + 16) + (size_t)R_WARPS * 512 * (M <= 8 ? 1 : 2) + 16; }

}  // namespace

// Every CTA quantises all the rows, so there is a size of the rows from which a launch of its own is the faster way (us, one
// launch | two: K 2048, N 4096: 6.9 | 12.3 for one row, 8.5 | 12.4 for 4, 10.5 | 12.3 for 8, 14.8 | 13.3 for 12, 15.3 | 13.2 for
// 16; K 4096, N 4096: 12.4 | 14.9 for 4, 15.7 | 15.7 for 8; 16 rows with K and N 1024: 10.0 | 10.3).
bool w8a8_rows_covers(const void* x, int x_dtype, int64_t stride, const void* w, int64_t M, int64_t N, int64_t K) {
  return M <= 16 && K % 16 == 0 && M * K <= 16384 && N < ((int64_t)1 << 30) && aligned16(x) && aligned16(w) &&
         (M == 1 || stride * (int64_t)dtype_size(x_dtype) % 16 == 0);
}

// The CTAs quantise the rows again in every round, two of them on an SM at a time, so N decides too.  Against the product on CTA
// pairs (N a multiple of 16) one launch wins in a single round, and one or two short rows in two (us, one launch | two: K 2048,
// N 8192: 10.4 | 12.7 for one row, 12.3 | 12.6 for 2, 14.4 | 12.5 for 4; 16 rows of K 64: 12.7 | 11.7; K 4096: 14.7 | 16.5 for one
// row; N 16384: 17.4 | 15.5 and 31.3 | 15.7 for 8 rows of 2048; N 151936: 111 | 60 and 210 | 61).  Against the small tiles, which
// walk K slowly, longer: K 4096, N 8195: 22.0 | 24.5 for 4 rows; K 16384, N 10243: 51 | 78; but K 256, N 6147: 10.3 | 8.7; K 2048,
// N 16387: 17.5 | 16.8, 30 | 17 for 8 rows.
bool w8a8_rows_pays(int64_t M, int64_t N, int64_t K) {
  const int64_t rounds = ((N + 15) / 16 + 2 * device_sm_count() - 1) / (2 * device_sm_count());
  if (rounds <= 1) return true;
  if (N % 16 == 0) return rounds == 2 && M <= 2 && M * K <= 4096;
  return rounds <= (M <= 2 && K >= 2048 ? 3 : M <= 4 && K >= 1024 ? 2 : 1);
}

int w8a8_rows(const void* x, int x_dtype, int64_t stride, const int8_t* w, const float* w_scale, int64_t M, int64_t N, int64_t K,
              int out_dtype, void* out, cudaStream_t st) {
  const RowsArgs A{x, w, w_scale, out, stride, (int)M, (int)N, (int)K, x_dtype, out_dtype};
  const size_t smem = rows_smem_bytes(M, K);
  const unsigned blocks = (unsigned)((N + 15) / 16);
  if (M <= 8) {
    w8a8_rows_kernel<1><<<blocks, R_WARPS * 32, smem, st>>>(A);
  } else {
    w8a8_rows_kernel<2><<<blocks, R_WARPS * 32, smem, st>>>(A);
  }
  return check_launch();
}

}  // namespace mq
