// The whole MoE layer for up to 16 tokens in two launches: router, top-k, gate/up + SwiGLU, down, weighted sum and
// residual (mini_qwen/model/layers/moe.py:49-68 and model/qwen3_moe.py:63-66 of the reference), on bf16 or fp16 experts,
// on int4 ones (W4A16) or on int8 ones (W8A8).
//
//   logits[t, e] = x[t] . router[e] (+ bias[e]);  p = softmax(logits);  the top_k largest logits, equal ones by ascending id
//   h[t, k] = silu(x[t] . gate[e]) * (x[t] . up[e])
//   out[t] = round(sum_k weight[t, k] * (h[t, k] . down[e]) + residual[t])
//
// Everything between the inputs and the one rounding at the end is held in fp32 or better: the tensor cores' fp32 sums, and
// h as the sum of two bf16 numbers (16 bits of precision; fp16 experts: two tf32 numbers).  W8A8: x and h are quantised per
// token (int8.cuh), the sums are int32.
//
// What bounds it is reading the weights of the experts that are hit; a chain of four to eight dependent launches spends more
// than that on latencies.  So:
//   * launch 1, a CTA per expert: logits.  Spare CTAs quantise the rows (W8A8) and clear the counters of launch 2;
//   * launch 2, one CTA per SM, all resident (a cooperative launch): every CTA selects the experts for itself; the gate/up
//     rows of all experts hit are dealt out evenly, to the row, so that no CTA has more than its share of bytes; one barrier
//     over the grid; then each CTA takes a few output columns of ALL experts hit, so the sum over experts stays inside the
//     CTA: no atomics, no second pass, the same bits every time;
//   * a warp reads 16-byte pieces of weight rows straight into registers, in an order of k in which they are the fragments
//     of mma.sync (tokens are its 8 columns): the tensor cores cost nothing here, and eight tokens of an expert cost one pass
//     over its weights.  The next pieces are in flight while one batch is multiplied; the first ones of the down projection
//     are issued, and the rest of its weights asked into L2, before the barrier.
// The wait at the barrier is bounded; when it runs out, MQ_DEV_WAIT_EXPIRED is set and nothing is written.
#include "int8.cuh"

namespace mq {
namespace {

using namespace int8;

constexpr int MAX_T = 16, MAX_E = 1024, MAX_K = 32;
constexpr int WARPS = 16, THREADS = WARPS * 32;
constexpr int BATCH = 4;                           // steps of k a warp has in flight
constexpr size_t SMEM_LIMIT = 229376;              // dynamic shared memory, beside the static 2 KB
constexpr uint32_t POLL_LIMIT = 1u << 22;          // looks at the barrier: about two seconds

enum Format { F_BF16, F_F16, F_INT8, F_INT4 };

struct SmallArgs {
  const void *x, *residual;
  void* out;
  const void* router;
  const float* bias;
  const void *w13, *w2;                            // bf16, fp16, int8 [E, 2I, H] and [E, H, I]
  const float *s13, *s2;                           // int8: [E, 2I], [E, H]
  const int32_t* qw[3];                            // int4: gate, up, down
  const __nv_bfloat16* sc[3];
  const int32_t* qz[3];
  int T, H, I, E, K, group, renorm, dtype, router_dtype;
  unsigned* counter;                               // workspace from here on
  uint32_t* amax;                                  // [T * K] largest |h| of a slot, as bits
  float* logits;                                   // [T, E]
  int8_t* xq;                                      // [T, H]
  float* xs;                                       // [T]
  void* h;                                         // bf16, int4: [T * K, 2, I] high and low parts; else fp32 [T * K, I]
  int32_t* d_status;
};

// ---- launch 1 -------------------------------------------------------------------------------------------

__device__ __forceinline__ void load8(const void* p, int dt, size_t i, bool vec, int64_t left, float (&v)[8]) {
  if (vec && left >= 8) {
    if (dt == MQ_F32) {
      const float4* q = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i);
      const float4 a = q[0], b = q[1];
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const uint4 a = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p) + i);
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = dt == MQ_BF16 ? __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[j]))
                                       : __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
        v[2 * j] = f.x;
        v[2 * j + 1] = f.y;
      }
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = j < left ? load_as_float(p, dt, i + j) : 0.0f;
}

template <int TN>                                  // tokens, rounded up
__global__ void __launch_bounds__(128) moe_small_router(const SmallArgs A, int router_vec) {
  __shared__ float part[4][TN];
  __shared__ uint32_t top[4];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if ((int)blockIdx.x >= A.E) {                    // spare CTAs
    const int t = (int)blockIdx.x - A.E;
    if (t == 0) {
      if (tid == 0) *A.counter = 0;
      for (int i = tid; i < A.T * A.K; i += 128) A.amax[i] = 0;
    }
    if (A.xq == nullptr) return;
    uint32_t most = 0;
    for (int k = 8 * tid; k < A.H; k += 8 * 128) {
      float v[8];
      load8(A.x, A.dtype, (size_t)t * A.H + k, true, A.H - k, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) most = max(most, abs_bits(v[j]));
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) top[warp] = most;
    __syncthreads();
    const RowScale r = row_scale(max(max(top[0], top[1]), max(top[2], top[3])));
    if (tid == 0) A.xs[t] = r.scale;
    for (int k = 8 * tid; k < A.H; k += 8 * 128) {
      float v[8];
      load8(A.x, A.dtype, (size_t)t * A.H + k, true, A.H - k, v);
      uint32_t w[2] = {0, 0};
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j >> 2] |= ((uint32_t)quantize(v[j], r) & 0xffu) << (8 * (j & 3));
      *reinterpret_cast<uint2*>(A.xq + (size_t)t * A.H + k) = make_uint2(w[0], w[1]);
    }
    return;
  }
  const int e = (int)blockIdx.x;
  float acc[TN];
#pragma unroll
  for (int t = 0; t < TN; ++t) acc[t] = 0.0f;
  for (int k = 8 * tid; k < A.H; k += 8 * 128) {
    float w[8];
    load8(A.router, A.router_dtype, (size_t)e * A.H + k, router_vec != 0, A.H - k, w);
#pragma unroll
    for (int t = 0; t < TN; ++t) {
      if (t < A.T) {
        float v[8];
        load8(A.x, A.dtype, (size_t)t * A.H + k, true, A.H - k, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[t] = fmaf(v[j], w[j], acc[t]);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < TN; ++t) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc[t] += __shfl_xor_sync(0xffffffffu, acc[t], o);
    if (lane == 0) part[warp][t] = acc[t];
  }
  __syncthreads();
  if (tid < TN && tid < A.T) {
    float v = (part[0][tid] + part[1][tid]) + (part[2][tid] + part[3][tid]);
    if (A.bias != nullptr) v += A.bias[e];
    A.logits[tid * A.E + e] = v;
  }
}

// ---- launch 2 -------------------------------------------------------------------------------------------

__device__ __forceinline__ uint4 ld_weights(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 ld_weights2(const void* p) {
  uint2 v;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%0, %1, %2, %3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// bf16 pairs (q0 - z, q4 - z), (q1 - z, q5 - z), ... of a word's eight nibbles; `minus` is the pair -(128 + z).  128 + q is
// the bit pattern 0x4300 | q, and both it and the difference are exact in bf16.
__device__ __forceinline__ void unpack_int4(uint32_t word, __nv_bfloat162 minus, uint32_t (&v)[4]) {
  const __nv_bfloat162 one = __floats2bfloat162_rn(1.0f, 1.0f);
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const uint32_t raw = ((word >> (4 * p)) & 0x000F000Fu) | 0x43004300u;
    const __nv_bfloat162 d = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&raw), one, minus);
    v[p] = *reinterpret_cast<const uint32_t*>(&d);
  }
}
// eight bf16 in their natural order -> the pairs (0, 4), (1, 5), (2, 6), (3, 7)
__device__ __forceinline__ uint4 pair_up(uint4 v) {
  return make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410),
                    __byte_perm(v.y, v.w, 0x7632));
}

// Selection for one token by a warp: the K largest logits, equal ones by ascending expert, as ids and softmax weights.
// Logits are compared as integers that order like them, so that NaNs too have a place and the ids are always K different
// experts.
template <int EPL>
__device__ __forceinline__ void select_experts(const float* logits, int E, int K, int renorm, int lane, uint16_t* ids,
                                               float* weights) {
  uint32_t key[EPL];
  float v[EPL];
  uint32_t best = 0;
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    const int e = lane + 32 * j;
    v[j] = e < E ? logits[e] + 0.0f : -INFINITY;   // + 0: minus zero is zero
    const uint32_t b = __float_as_uint(v[j]);
    key[j] = e < E ? max(b ^ ((uint32_t)((int)b >> 31) | 0x80000000u), 1u) : 0u;
    best = max(best, key[j]);
  }
  const uint32_t first = __reduce_max_sync(0xffffffffu, best);
  auto value = [](uint32_t k) { return __uint_as_float((k & 0x80000000u) != 0 ? k & 0x7fffffffu : ~k); };
  const float m = value(first);
  float sum = 0.0f;
#pragma unroll
  for (int j = 0; j < EPL; ++j)
    if (lane + 32 * j < E) sum += expf(v[j] - m);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  float mine = 0.0f, chosen = 0.0f;
  int my_id = 0;
  for (int k = 0; k < K; ++k) {
    uint32_t b = 0;
    int bj = 0;
#pragma unroll
    for (int j = 0; j < EPL; ++j)
      if (key[j] > b) { b = key[j]; bj = j; }
    const uint32_t top = __reduce_max_sync(0xffffffffu, b);
    const int id = (int)__reduce_min_sync(0xffffffffu, b == top && b != 0 ? (unsigned)(lane + 32 * bj) : 0xffffu);
#pragma unroll
    for (int j = 0; j < EPL; ++j)
      if (lane + 32 * j == id) key[j] = 0;
    const float p = expf(value(top) - m) / sum;
    if (lane == k) { mine = p; my_id = id; }
    chosen += p;
  }
  if (lane < K) {
    ids[lane] = (uint16_t)my_id;
    weights[lane] = renorm ? mine / chosen : mine;
  }
}

// Tables in shared memory behind the partial sums.
struct Tables {
  uint32_t* mask;      // [E] tokens of the expert
  uint16_t* pos;       // [E] its place among the experts hit
  uint16_t* hit;       // [hits]
  uint16_t* before;    // [hits] slots of the experts in front of it
  uint8_t* slot;       // [hits, MAX_T] which of the token's experts it is
  float* weight;       // [hits, MAX_T] its weight in the token's sum
  uint16_t* ids;       // [T, MAX_K]
  float* w;            // [T, MAX_K]
  __host__ __device__ static size_t bytes(int T, int E, int K) {
    const size_t hits = (size_t)(E < T * K ? E : T * K);
    return hits * MAX_T * 5 + hits * 4 + (size_t)E * 6 + (size_t)T * MAX_K * 6 + 64;
  }
  __device__ Tables(uint8_t* p, int T, int E, int K) {
    const int hits = min(E, T * K);
    weight = reinterpret_cast<float*>(p);
    w = weight + hits * MAX_T;
    mask = reinterpret_cast<uint32_t*>(w + T * MAX_K);
    ids = reinterpret_cast<uint16_t*>(mask + E);
    pos = ids + T * MAX_K;
    hit = pos + E;
    before = hit + hits;
    slot = reinterpret_cast<uint8_t*>(before + hits);
  }
};

// Weight bytes per k and elements of k in a step of 64 bytes (int4: 32 k, four words of a column).
template <int F> struct Fmt { static constexpr int STEP = F == F_INT8 ? 64 : 32, SIZE = F == F_INT8 ? 1 : 2; };

constexpr int PARTS = 64;                          // 16 x 8 partial sums that a meeting of the warps holds
constexpr int PART_BUFFER = PARTS * 512;           // their bytes for eight tokens
constexpr int SUM_BUFFER = WARPS * 512;            // the same of the output's sums
__host__ __device__ constexpr size_t part_bytes(int octets) { return (size_t)2 * PART_BUFFER * octets; }
// Shared memory in front of the tables: the partial sums, later the output's sums and (int8) the quantised h.
__host__ __device__ inline size_t front_bytes(bool int8, int octets, int64_t slots, int64_t I) {
  const size_t later = (size_t)2 * SUM_BUFFER * octets + (int8 ? (size_t)slots * (I + 16) : 0);
  return later > part_bytes(octets) ? (later + 15) & ~(size_t)15 : part_bytes(octets);
}

template <int F, int OCT, typename OutT>
__global__ void __launch_bounds__(THREADS, 1) moe_small_layer(const SmallArgs A) {
  using Acc = typename std::conditional<F == F_INT8, int, float>::type;
  constexpr int STEP = Fmt<F>::STEP, SIZE = Fmt<F>::SIZE;
  constexpr bool W4 = F == F_INT4;
  constexpr int TW = W4 ? 16 : 8;                  // columns of h in a tile
  constexpr int MT = W4 ? 2 : 1;                   // accumulator tiles: int4 gate and up apart, else 8 + 8 rows in one
  extern __shared__ uint8_t small_smem[];
  uint8_t* part = small_smem;
  const Tables tab(small_smem + front_bytes(F == F_INT8, OCT, A.T * A.K, A.I), A.T, A.E, A.K);
  __shared__ int s_hits, s_ok;
  __shared__ int4 s_tile[2][PARTS];                // expert's place, first column, columns
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q4 = lane & 3;
  const int T = A.T, H = A.H, I = A.I, E = A.E, K = A.K, G = (int)gridDim.x, cta = (int)blockIdx.x;

  // ------------------------------------------------------------------ who goes where
  for (int e = tid; e < E; e += THREADS) tab.mask[e] = 0;
  if (warp < T) {
    const float* row = A.logits + warp * E;
    if (E <= 128) select_experts<4>(row, E, K, A.renorm, lane, tab.ids + warp * MAX_K, tab.w + warp * MAX_K);
    else select_experts<MAX_E / 32>(row, E, K, A.renorm, lane, tab.ids + warp * MAX_K, tab.w + warp * MAX_K);
  }
  __syncthreads();
  for (int i = tid; i < T * MAX_K; i += THREADS)
    if (i % MAX_K < K) atomicOr(&tab.mask[tab.ids[i]], 1u << (i / MAX_K));
  __syncthreads();
  if (warp == 0) {
    int n = 0, slots = 0;
    for (int e0 = 0; e0 < E; e0 += 32) {
      const uint32_t m = e0 + lane < E ? tab.mask[e0 + lane] : 0u;
      const unsigned any = __ballot_sync(0xffffffffu, m != 0);
      const int at = n + __popc(any & ((1u << lane) - 1u));
      int incl = __popc(m);
      const int own = incl;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      if (m != 0) {
        tab.hit[at] = (uint16_t)(e0 + lane);
        tab.pos[e0 + lane] = (uint16_t)at;
        tab.before[at] = (uint16_t)(slots + incl - own);
      }
      n += __popc(any);
      slots += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) s_hits = n;
  }
  __syncthreads();
  for (int i = tid; i < T * MAX_K; i += THREADS)
    if (i % MAX_K < K) {
      const int at = tab.pos[tab.ids[i]] * MAX_T + i / MAX_K;
      tab.slot[at] = (uint8_t)(i % MAX_K);
      tab.weight[at] = tab.w[i];
    }
  __syncthreads();
  const int hits = s_hits;

  // ------------------------------------------------------------------ gate and up projections, SwiGLU
  // The columns of h of all experts hit, one after the other, are cut into equal ranges (int4: by 16 columns).  A CTA walks
  // its range in tiles; the warps share a tile's k (`ksplit` of them) and, where k is short, two or more tiles at a time.
  // After `together` tiles the partial sums meet in shared memory (two buffers in turn, so one barrier a meeting).
  {
    const int64_t all = (int64_t)hits * (I / (W4 ? 16 : 1));
    const int lo = (int)(all * cta / G) * (W4 ? 16 : 1), hi = (int)(all * (cta + 1) / G) * (W4 ? 16 : 1);
    const int steps = (H + STEP - 1) / STEP, batches = (steps + BATCH - 1) / BATCH;
    int ksplit = WARPS;
    while (ksplit > batches) ksplit >>= 1;
    const int at_once = WARPS / ksplit, together = PARTS / MT / ksplit, kw = warp % ksplit, tg = warp / ksplit;
    struct Walk { int pos, place, end; } cur;      // column over all experts, the expert's place, where its columns end
    cur.pos = lo;
    cur.place = lo / I;
    cur.end = (cur.place + 1) * I;
    auto width = [&](const Walk& c) { return min(TW, min(c.end, hi) - c.pos); };
    auto advance = [&](Walk& c) {
      c.pos += width(c);
      if (c.pos == c.end) { ++c.place; c.end += I; }
    };
    int tiles;                                     // of the whole range
    {
      const int p0 = lo / I, p1 = hi / I, r0 = lo - p0 * I, r1 = hi - p1 * I;
      tiles = p0 == p1 ? (hi - lo + TW - 1) / TW
                       : (I - r0 + TW - 1) / TW + (p1 - p0 - 1) * ((I + TW - 1) / TW) + (r1 + TW - 1) / TW;
    }
    uint4 a[BATCH][W4 ? 1 : 2], na[BATCH][W4 ? 1 : 2];      // row g / g + 8 pieces; int4: gate words, up words
    uint2 sz[2], nsz[2];                                    // int4: scales of two columns, word of their zero points
    auto fetch = [&](const Walk& c, int batch, uint4 (&d)[BATCH][W4 ? 1 : 2], uint2 (&dz)[2]) {
      const size_t e = tab.hit[c.place];
      const int col = c.pos - (c.end - I);
      if (W4) {
        const int k0 = batch * (BATCH * STEP), grp = k0 / A.group;
        const size_t n = (size_t)col + 2 * g;
#pragma unroll
        for (int s = 0; s < BATCH; ++s) {
          const size_t at = (e * (H / 8) + k0 / 8 + 4 * s + q4) * I + n;
          const uint2 v0 = ld_weights2(A.qw[0] + at), v1 = ld_weights2(A.qw[1] + at);
          d[s][0] = make_uint4(v0.x, v0.y, v1.x, v1.y);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const size_t row = e * (H / A.group) + grp;
          dz[j].x = *reinterpret_cast<const uint32_t*>(A.sc[j] + row * I + n);
          dz[j].y = (uint32_t)A.qz[j][row * (I / 8) + (n >> 3)] >> (4 * (n & 7));
        }
      } else {
        const bool live = g < width(c);
        const uint8_t* base = reinterpret_cast<const uint8_t*>(A.w13) + (e * 2 * I + col + g) * (size_t)H * SIZE;
        const size_t up = (size_t)I * H * SIZE;
#pragma unroll
        for (int s = 0; s < BATCH; ++s) {
          const int b = (batch * BATCH + s) * 64 + 16 * q4;
          const bool in = live && b < H * SIZE;
          d[s][0] = in ? ld_weights(base + b) : make_uint4(0u, 0u, 0u, 0u);
          d[s][W4 ? 0 : 1] = in ? ld_weights(base + up + b) : make_uint4(0u, 0u, 0u, 0u);
        }
      }
    };
    for (int i = 0; i < tg && cur.pos < hi; ++i) advance(cur);
    int index = tg;                                // of the warp's tile in the range
    if (cur.pos < hi) fetch(cur, kw, a, sz);
    const int meetings = (tiles + together - 1) / together;
    for (int meet = 0; meet < meetings; ++meet) {
      uint8_t* buf = part + (meet & 1) * PART_BUFFER * OCT;
      while (index < tiles && index / together == meet) {
        Walk nxt = cur;
        for (int i = 0; i < at_once && nxt.pos < hi; ++i) advance(nxt);
        const uint32_t mask = tab.mask[tab.hit[cur.place]];
        Acc acc[OCT][MT][4] = {};
        for (int batch = kw; batch < batches; batch += ksplit) {
          if (batch + ksplit < batches) fetch(cur, batch + ksplit, na, nsz);
          else if (nxt.pos < hi) fetch(nxt, kw, na, nsz);
#pragma unroll
          for (int o = 0; o < OCT; ++o) {
            if (((mask >> (8 * o)) & 0xffu) == 0) continue;
            const int tok = 8 * o + g;
            float grp[MT][4] = {};
#pragma unroll
            for (int s = 0; s < BATCH; ++s) {
              const int k = (batch * BATCH + s) * STEP + (16 / SIZE) * q4;
              uint4 b = make_uint4(0u, 0u, 0u, 0u);
              if (tok < T && k < H) {
                const uint8_t* rows = F == F_INT8 ? reinterpret_cast<const uint8_t*>(A.xq) : reinterpret_cast<const uint8_t*>(A.x);
                b = __ldg(reinterpret_cast<const uint4*>(rows + ((size_t)tok * H + k) * SIZE));
              }
              if constexpr (W4) {
                b = pair_up(b);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                  const uint32_t z = sz[j].y;
                  const float z0 = -(128.0f + (float)(z & 15u)), z1 = -(128.0f + (float)((z >> 4) & 15u));
                  uint32_t v0[4], v1[4];
                  unpack_int4(j == 0 ? a[s][0].x : a[s][0].z, __floats2bfloat162_rn(z0, z0), v0);
                  unpack_int4(j == 0 ? a[s][0].y : a[s][0].w, __floats2bfloat162_rn(z1, z1), v1);
                  mma_bf16(grp[j % MT], v0[0], v1[0], v0[1], v1[1], b.x, b.y);
                  mma_bf16(grp[j % MT], v0[2], v1[2], v0[3], v1[3], b.z, b.w);
                }
              } else if constexpr (F == F_INT8) {
                mma_s8(acc[o][0], a[s][0].x, a[s][1].x, a[s][0].y, a[s][1].y, b.x, b.y);
                mma_s8(acc[o][0], a[s][0].z, a[s][1].z, a[s][0].w, a[s][1].w, b.z, b.w);
              } else if constexpr (F == F_F16) {
                mma_f16(acc[o][0], a[s][0].x, a[s][1].x, a[s][0].y, a[s][1].y, b.x, b.y);
                mma_f16(acc[o][0], a[s][0].z, a[s][1].z, a[s][0].w, a[s][1].w, b.z, b.w);
              } else {
                mma_bf16(acc[o][0], a[s][0].x, a[s][1].x, a[s][0].y, a[s][1].y, b.x, b.y);
                mma_bf16(acc[o][0], a[s][0].z, a[s][1].z, a[s][0].w, a[s][1].w, b.z, b.w);
              }
            }
            if constexpr (W4) {                    // a batch lies inside a quantisation group
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                const float2 sc = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&sz[j].x));
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[o][j][i] = fmaf(grp[j][i], i < 2 ? sc.x : sc.y, acc[o][j][i]);
              }
            }
          }
#pragma unroll
          for (int s = 0; s < BATCH; ++s)
#pragma unroll
            for (int j = 0; j < (W4 ? 1 : 2); ++j) a[s][j] = na[s][j];
          sz[0] = nsz[0];
          sz[1] = nsz[1];
        }
        const int slot = index % together;
#pragma unroll
        for (int o = 0; o < OCT; ++o)
#pragma unroll
          for (int j = 0; j < MT; ++j) {
            const Acc* c = acc[o][j];
            *reinterpret_cast<int4*>(buf + ((((slot * ksplit + kw) * OCT + o) * MT + j) * 32 + lane) * 16) =
                *reinterpret_cast<const int4*>(c);
          }
        if (kw == 0 && lane == 0) s_tile[meet & 1][slot] = make_int4(cur.place, cur.pos - (cur.end - I), width(cur), 0);
        cur = nxt;
        index += at_once;
      }
      __syncthreads();
      // thread: a fragment position of a tile; its sums over the warps in order
      for (int at_part = tid; at_part < together * OCT * 32; at_part += THREADS) {
        const int slot = at_part / (OCT * 32), o = at_part / 32 % OCT;
        if (meet * together + slot < tiles) {
          const int4 tile = s_tile[meet & 1][slot];
          const uint32_t mask = tab.mask[tab.hit[tile.x]];
          if (((mask >> (8 * o)) & 0xffu) != 0) {
            Acc sum[MT][4] = {};
            for (int w = 0; w < ksplit; ++w)
#pragma unroll
              for (int j = 0; j < MT; ++j) {
                const int4 raw = *reinterpret_cast<const int4*>(buf + ((((slot * ksplit + w) * OCT + o) * MT + j) * 32 + lane) * 16);
                const Acc* c = reinterpret_cast<const Acc*>(&raw);
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[j][i] += c[i];
              }
#pragma unroll
            for (int i = 0; i < (W4 ? 4 : 2); ++i) {
              const int tok = 8 * o + 2 * q4 + (i & 1), col = W4 ? 2 * g + (i >> 1) : g;
              const bool live = ((mask >> tok) & 1u) != 0 && col < tile.z;
              float v = 0.0f;
              size_t at = 0;
              if (live) {
                at = (size_t)tok * K + tab.slot[tile.x * MAX_T + tok];
                float gv, uv;
                if constexpr (F == F_INT8) {
                  const float* s = A.s13 + (size_t)tab.hit[tile.x] * 2 * I + tile.y + col;
                  const float sx = A.xs[tok];
                  gv = __fmul_rn(__fmul_rn(__int2float_rn(sum[0][i]), sx), s[0]);
                  uv = __fmul_rn(__fmul_rn(__int2float_rn(sum[0][2 + i]), sx), s[I]);
                } else {
                  gv = (float)sum[0][i];
                  uv = W4 ? (float)sum[MT - 1][i] : (float)sum[0][(2 + i) & 3];
                }
                const float p = expf(-fabsf(gv));
                v = __fdividef(gv < 0.0f ? p * gv : gv, 1.0f + p) * uv;
                if (F == F_BF16 || W4) {
                  __nv_bfloat16* h = reinterpret_cast<__nv_bfloat16*>(A.h) + at * 2 * I + tile.y + col;
                  const __nv_bfloat16 high = __float2bfloat16_rn(v);
                  h[0] = high;
                  h[I] = __float2bfloat16_rn(__hisinf(high) ? 0.0f : v - __bfloat162float(high));
                } else {
                  reinterpret_cast<float*>(A.h)[at * I + tile.y + col] = v;
                }
              }
              if (F == F_INT8) {                   // the slot's largest |h|: first over the eight columns
                uint32_t bits = abs_bits(v);
#pragma unroll
                for (int s = 4; s < 32; s <<= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, s));
                if (g == 0 && ((mask >> tok) & 1u) != 0) atomicMax(A.amax + (size_t)tok * K + tab.slot[tile.x * MAX_T + tok], bits);
              }
            }
          }
        }
      }
    }
  }

  // ------------------------------------------------------------------ down projection: its weights on their way
  // A CTA's output columns (rows of the down weights; int4: by 16), a tile of 16 at a time; its tasks are (expert, batch of
  // k), dealt out to the warps.
  const int out_lo = W4 ? (int)((int64_t)(H / 16) * cta / G) * 16 : (int)((int64_t)H * cta / G);
  const int out_hi = W4 ? (int)((int64_t)(H / 16) * (cta + 1) / G) * 16 : (int)((int64_t)H * (cta + 1) / G);
  const int steps = (I + STEP - 1) / STEP, batches = (steps + BATCH - 1) / BATCH;
  uint4 a[BATCH], c8[BATCH];                       // rows g and g + 8; int4: the words of two columns
  uint2 sz;
  auto fetch = [&](int row0, int task, uint4 (&d)[BATCH], uint4 (&d8)[BATCH], uint2& dz) {
    const size_t e = tab.hit[task / batches];
    const int batch = task % batches;
    if (W4) {
      const int k0 = batch * (BATCH * STEP);
      const size_t n = (size_t)row0 + 2 * g, row = e * (I / A.group) + k0 / A.group;
#pragma unroll
      for (int s = 0; s < BATCH; ++s) {
        const uint2 v = ld_weights2(A.qw[2] + (e * (I / 8) + k0 / 8 + 4 * s + q4) * H + n);
        d[s].x = v.x;
        d[s].y = v.y;
      }
      dz.x = *reinterpret_cast<const uint32_t*>(A.sc[2] + row * H + n);
      dz.y = (uint32_t)A.qz[2][row * (H / 8) + (n >> 3)] >> (4 * (n & 7));
    } else {
      const uint8_t* base = reinterpret_cast<const uint8_t*>(A.w2) + (e * H + row0 + g) * (size_t)I * SIZE;
#pragma unroll
      for (int s = 0; s < BATCH; ++s) {
        const int b = (batch * BATCH + s) * 64 + 16 * q4;
        const bool in = b < I * SIZE;
        d[s] = in && row0 + g < out_hi ? ld_weights(base + b) : make_uint4(0u, 0u, 0u, 0u);
        d8[s] = in && row0 + g + 8 < out_hi ? ld_weights(base + (size_t)8 * I * SIZE + b) : make_uint4(0u, 0u, 0u, 0u);
      }
    }
  };
  const int tasks = hits * batches;
  if (out_lo < out_hi && warp < tasks) fetch(out_lo, warp, a, c8, sz);

  // ------------------------------------------------------------------ every h is there
  __syncthreads();
  if (tid == 0) {
    __threadfence();
    atomicAdd(A.counter, 1u);
    uint32_t seen = 0, looks = 0;
    do {
      asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(seen) : "l"(A.counter) : "memory");
    } while (seen < (unsigned)G && ++looks < POLL_LIMIT);
    s_ok = seen >= (unsigned)G;
    if (!s_ok && A.d_status != nullptr) atomicOr(A.d_status, (int)MQ_DEV_WAIT_EXPIRED);
    __threadfence();
  }
  __syncthreads();
  if (!s_ok) return;

  // ------------------------------------------------------------------ down projection and weighted sum
  // int8: h is quantised here, by every CTA for itself.
  int8_t* hq = reinterpret_cast<int8_t*>(part + 2 * SUM_BUFFER * OCT);
  auto hq_row = [&](int place, uint32_t mask, int tok) {
    return hq + (size_t)(tab.before[place] + __popc(mask & ((1u << tok) - 1u))) * (I + 16);
  };
  if (F == F_INT8) {
    for (int i = warp; i < hits * MAX_T; i += WARPS) {
      const int place = i / MAX_T, tok = i % MAX_T;
      const uint32_t mask = tab.mask[tab.hit[place]];
      if (((mask >> tok) & 1u) == 0) continue;
      const size_t slot = (size_t)tok * K + tab.slot[i];
      const RowScale r = row_scale(__ldcg(A.amax + slot));
      const float* src = reinterpret_cast<const float*>(A.h) + slot * I;
      int8_t* dst = hq_row(place, mask, tok);
      for (int k = 4 * lane; k < I; k += 128) {
        const float4 v = __ldcg(reinterpret_cast<const float4*>(src + k));
        *reinterpret_cast<uint32_t*>(dst + k) =
            ((uint32_t)quantize(v.x, r) & 0xffu) | ((uint32_t)quantize(v.y, r) & 0xffu) << 8 |
            ((uint32_t)quantize(v.z, r) & 0xffu) << 16 | ((uint32_t)quantize(v.w, r) & 0xffu) << 24;
      }
    }
    __syncthreads();
  }
  int meet = 0;
  for (int row0 = out_lo; row0 < out_hi; row0 += 16) {
    float sum[OCT][4] = {};
    for (int task = warp; task < tasks; task += WARPS) {
      uint4 na[BATCH], nc8[BATCH];
      uint2 nsz;
      const bool more = task + WARPS < tasks, next_tile = !more && row0 + 16 < out_hi;
      if (more) fetch(row0, task + WARPS, na, nc8, nsz);
      else if (next_tile) fetch(row0 + 16, warp, na, nc8, nsz);
      const int place = task / batches, batch = task % batches;
      const uint32_t mask = tab.mask[tab.hit[place]];
#pragma unroll
      for (int o = 0; o < OCT; ++o) {
        if (((mask >> (8 * o)) & 0xffu) == 0) continue;
        const int tok = 8 * o + g;
        const bool live = ((mask >> tok) & 1u) != 0;
        const size_t slot = live ? (size_t)tok * K + tab.slot[place * MAX_T + tok] : 0;
        Acc acc[4] = {};
#pragma unroll
        for (int s = 0; s < BATCH; ++s) {
          const int k = (batch * BATCH + s) * STEP + (16 / SIZE) * q4;
          const bool in = live && k < I;
          if constexpr (F == F_INT8) {
            uint4 b = make_uint4(0u, 0u, 0u, 0u);
            if (in) b = *reinterpret_cast<const uint4*>(hq_row(place, mask, tok) + k);
            mma_s8(acc, a[s].x, c8[s].x, a[s].y, c8[s].y, b.x, b.y);
            mma_s8(acc, a[s].z, c8[s].z, a[s].w, c8[s].w, b.z, b.w);
          } else if constexpr (F == F_F16) {
            float4 f[2] = {};
            if (in) {
              const float4* src = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(A.h) + slot * I + k);
              f[0] = __ldcg(src);
              f[1] = __ldcg(src + 1);
            }
            const float* v = reinterpret_cast<const float*>(f);
            const uint32_t* w = reinterpret_cast<const uint32_t*>(&a[s]);
            const uint32_t* w8 = reinterpret_cast<const uint32_t*>(&c8[s]);
#pragma unroll
            for (int p = 0; p < 4; ++p) {
              // a tf32 number is the upper 19 bits of an fp32 one; fp16 fits, h is a sum of two
              const float2 lo = __half22float2(*reinterpret_cast<const __half2*>(&w[p]));
              const float2 hi = __half22float2(*reinterpret_cast<const __half2*>(&w8[p]));
              const uint32_t h0 = __float_as_uint(v[2 * p]) & 0xffffe000u, h1 = __float_as_uint(v[2 * p + 1]) & 0xffffe000u;
              const uint32_t l0 = isinf(v[2 * p]) ? 0u : __float_as_uint(v[2 * p] - __uint_as_float(h0)) & 0xffffe000u;
              const uint32_t l1 = isinf(v[2 * p + 1]) ? 0u : __float_as_uint(v[2 * p + 1] - __uint_as_float(h1)) & 0xffffe000u;
              const uint32_t a0 = __float_as_uint(lo.x), a1 = __float_as_uint(hi.x), a2 = __float_as_uint(lo.y), a3 = __float_as_uint(hi.y);
              mma_tf32(acc, a0, a1, a2, a3, l0, l1);
              mma_tf32(acc, a0, a1, a2, a3, h0, h1);
            }
          } else {
            uint4 hi = make_uint4(0u, 0u, 0u, 0u), lo = hi;
            if (in) {
              const __nv_bfloat16* src = reinterpret_cast<const __nv_bfloat16*>(A.h) + slot * 2 * I + k;
              hi = __ldcg(reinterpret_cast<const uint4*>(src));
              lo = __ldcg(reinterpret_cast<const uint4*>(src + I));
            }
            if constexpr (W4) {
              hi = pair_up(hi);
              lo = pair_up(lo);
              const float z0 = -(128.0f + (float)(sz.y & 15u)), z1 = -(128.0f + (float)((sz.y >> 4) & 15u));
              uint32_t v0[4], v1[4];
              unpack_int4(a[s].x, __floats2bfloat162_rn(z0, z0), v0);
              unpack_int4(a[s].y, __floats2bfloat162_rn(z1, z1), v1);
              mma_bf16(acc, v0[0], v1[0], v0[1], v1[1], lo.x, lo.y);
              mma_bf16(acc, v0[2], v1[2], v0[3], v1[3], lo.z, lo.w);
              mma_bf16(acc, v0[0], v1[0], v0[1], v1[1], hi.x, hi.y);
              mma_bf16(acc, v0[2], v1[2], v0[3], v1[3], hi.z, hi.w);
            } else {
              mma_bf16(acc, a[s].x, c8[s].x, a[s].y, c8[s].y, lo.x, lo.y);
              mma_bf16(acc, a[s].z, c8[s].z, a[s].w, c8[s].w, lo.z, lo.w);
              mma_bf16(acc, a[s].x, c8[s].x, a[s].y, c8[s].y, hi.x, hi.y);
              mma_bf16(acc, a[s].z, c8[s].z, a[s].w, c8[s].w, hi.z, hi.w);
            }
          }
        }
        // into the tokens' sums; a token that did not choose the expert takes nothing from it, whatever its weights hold
        float s0 = 1.0f, s1 = 1.0f;
        if constexpr (W4) {
          const float2 sc = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&sz.x));
          s0 = sc.x;
          s1 = sc.y;
        } else if constexpr (F == F_INT8) {
          const float* s = A.s2 + (size_t)tab.hit[place] * H + row0 + g;
          s0 = row0 + g < out_hi ? s[0] : 0.0f;
          s1 = row0 + g + 8 < out_hi ? s[8] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int tk = 8 * o + 2 * q4 + (i & 1);
          if (((mask >> tk) & 1u) == 0) continue;
          float v = (float)acc[i];
          if (F == F_INT8) v *= scale_of(__ldcg(A.amax + (size_t)tk * K + tab.slot[place * MAX_T + tk]));
          if (F == F_INT8 || W4) v *= i < 2 ? s0 : s1;
          sum[o][i] = fmaf(v, tab.weight[place * MAX_T + tk], sum[o][i]);
        }
      }
      if (more || next_tile) {
#pragma unroll
        for (int s = 0; s < BATCH; ++s) {
          a[s] = na[s];
          c8[s] = nc8[s];
        }
        sz = nsz;
      }
    }
    // the warps' sums, in order, then the one rounding
    float4* buf = reinterpret_cast<float4*>(part + (meet & 1) * SUM_BUFFER * OCT);
    meet ^= 1;
#pragma unroll
    for (int o = 0; o < OCT; ++o)
      buf[(warp * OCT + o) * 32 + lane] = make_float4(sum[o][0], sum[o][1], sum[o][2], sum[o][3]);
    __syncthreads();
    if (tid < OCT * 128) {                         // tid: (octet, register, lane of the fragment)
      const int o = tid / 128, i = tid / 32 % 4;
      float v = 0.0f;
      for (int w = 0; w < WARPS; ++w) v += reinterpret_cast<const float*>(&buf[(w * OCT + o) * 32 + lane])[i];
      const int tok = 8 * o + 2 * q4 + (i & 1);
      const int row = row0 + (W4 ? 2 * g + (i >> 1) : g + 8 * (i >> 1));
      if (tok < T && row < out_hi) {
        const size_t at = (size_t)tok * H + row;
        if (A.residual != nullptr) v += to_float<OutT>(reinterpret_cast<const OutT*>(A.residual)[at]);
        reinterpret_cast<OutT*>(A.out)[at] = from_float<OutT>(v);
      }
    }
  }
}

// ---- host -----------------------------------------------------------------------------------------------

int format_of(const mq_moe_layer& L) {
  if (L.group_size > 0) return F_INT4;
  if (L.int8_experts) return F_INT8;
  return L.dtype == MQ_BF16 ? F_BF16 : F_F16;
}

bool shape_ok(const mq_moe_layer& L, int64_t T) {
  const int64_t H = L.hidden, I = L.inter, E = L.experts, K = L.top_k, big = (int64_t)1 << 20;
  if (T > MAX_T || E > MAX_E || K > MAX_K || K > E || H >= big || I >= big) return false;
  if (E * 2 * I >= ((int64_t)1 << 31)) return false;
  switch (format_of(L)) {
    case F_INT4: return L.group_size % 128 == 0 && H % L.group_size == 0 && I % L.group_size == 0 && L.dtype == MQ_BF16;
    case F_INT8:                                   // the quantised h of all slots lies in shared memory
      return H % 16 == 0 && I % 16 == 0 && H <= 131071 &&
             front_bytes(true, T <= 8 ? 1 : 2, T * K, I) + Tables::bytes((int)T, (int)E, (int)K) <= SMEM_LIMIT;
    default: return L.dtype != MQ_F32 && H % 8 == 0 && I % 8 == 0;
  }
}

size_t carve_small(const mq_moe_layer& L, int64_t T, uint8_t* base, SmallArgs& A) {
  size_t used = 0;
  auto take = [&](size_t bytes) {
    void* p = base + used;
    used += (bytes + 255) & ~(size_t)255;
    return p;
  };
  const size_t S = (size_t)(T * L.top_k);
  A.counter = (unsigned*)take(4);
  A.amax = (uint32_t*)take(S * 4);
  A.logits = (float*)take((size_t)(T * L.experts) * 4);
  A.xs = (float*)take((size_t)T * 4);
  A.h = take(S * (size_t)L.inter * 4);
  A.xq = format_of(L) == F_INT8 ? (int8_t*)take((size_t)(T * L.hidden)) : nullptr;
  return used;
}

bool small_layer_ok(const mq_moe_layer* L) {
  return L != nullptr && L->hidden > 0 && L->inter > 0 && L->experts > 0 && L->top_k > 0 && L->group_size >= 0 &&
         valid_dtype(L->dtype) && valid_dtype(L->router_dtype) && !(L->int8_experts && L->group_size > 0);
}

template <int F, int OCT, typename OutT>
int launch_layer(const SmallArgs& A, cudaStream_t st) {
  const size_t smem = front_bytes(F == F_INT8, OCT, A.T * A.K, A.I) + Tables::bytes(A.T, A.E, A.K);
  cudaError_t e = cudaFuncSetAttribute(moe_small_layer<F, OCT, OutT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  int dev = 0, sms = 0;
  if (e == cudaSuccess) e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e == cudaSuccess) {
    SmallArgs args = A;
    void* argv[] = {&args};
    e = cudaLaunchCooperativeKernel((const void*)moe_small_layer<F, OCT, OutT>, dim3(sms), dim3(THREADS), argv, smem, st);
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    set_last_cuda_error(e);
    return MQ_ERR_LAUNCH_FAILED;
  }
  return check_launch();
}

template <int OCT>
int launch_format(const SmallArgs& A, int format, cudaStream_t st) {
  switch (format) {
    case F_BF16: return launch_layer<F_BF16, OCT, __nv_bfloat16>(A, st);
    case F_F16: return launch_layer<F_F16, OCT, __half>(A, st);
    case F_INT4: return launch_layer<F_INT4, OCT, __nv_bfloat16>(A, st);
    default:
      if (A.dtype == MQ_F32) return launch_layer<F_INT8, OCT, float>(A, st);
      if (A.dtype == MQ_BF16) return launch_layer<F_INT8, OCT, __nv_bfloat16>(A, st);
      return launch_layer<F_INT8, OCT, __half>(A, st);
  }
}

}  // namespace
}  // namespace mq

extern "C" int mq_moe_small_covers(const mq_moe_layer* h_layer, int64_t T) {
  return mq::small_layer_ok(h_layer) && T >= 0 && mq::shape_ok(*h_layer, T) ? 1 : 0;
}

extern "C" size_t mq_moe_small_workspace_bytes(const mq_moe_layer* h_layer, int64_t T) {
  mq::SmallArgs A;
  if (!mq_moe_small_covers(h_layer, T) || T == 0) return 256;
  return mq::carve_small(*h_layer, T, nullptr, A);
}

extern "C" int mq_moe_small(const mq_moe_layer* h_layer, const void* x, const void* residual, int64_t T, void* workspace,
                            size_t workspace_bytes, void* out, int32_t* d_status, void* stream) {
  using namespace mq;
  if (!small_layer_ok(h_layer) || T < 0) return MQ_ERR_INVALID_ARGUMENT;
  const mq_moe_layer& L = *h_layer;
  if (!shape_ok(L, T)) return MQ_ERR_UNSUPPORTED_SHAPE;
  if (T == 0) return MQ_OK;
  const int format = format_of(L);
  SmallArgs A = {};
  A.x = x;
  A.residual = residual;
  A.out = out;
  A.router = L.router;
  A.bias = L.router_bias;
  bool ok = x && out && workspace && L.router && aligned16(x) && aligned16(workspace);
  auto weights = [&](const void* p) { ok = ok && p != nullptr && aligned16(p); };
  if (format == F_INT4) {
    const void* const* of[3] = {L.gate, L.up, L.down};
    for (int i = 0; i < 3; ++i) {
      weights(of[i][0]);
      ok = ok && of[i][1] && of[i][2] && ((reinterpret_cast<uintptr_t>(of[i][1]) | reinterpret_cast<uintptr_t>(of[i][2])) & 3u) == 0;
      A.qw[i] = reinterpret_cast<const int32_t*>(of[i][0]);
      A.sc[i] = reinterpret_cast<const __nv_bfloat16*>(of[i][1]);
      A.qz[i] = reinterpret_cast<const int32_t*>(of[i][2]);
    }
  } else {
    weights(L.gate[0]);
    weights(L.down[0]);
    A.w13 = L.gate[0];
    A.w2 = L.down[0];
    if (format == F_INT8) {
      ok = ok && L.gate[1] && L.down[1];
      A.s13 = reinterpret_cast<const float*>(L.gate[1]);
      A.s2 = reinterpret_cast<const float*>(L.down[1]);
    }
  }
  if (!ok) return MQ_ERR_INVALID_ARGUMENT;
  A.T = (int)T;
  A.H = (int)L.hidden;
  A.I = (int)L.inter;
  A.E = (int)L.experts;
  A.K = (int)L.top_k;
  A.group = (int)L.group_size;
  A.renorm = L.renormalize;
  A.dtype = L.dtype;
  A.router_dtype = L.router_dtype;
  A.d_status = d_status;
  if (carve_small(L, T, reinterpret_cast<uint8_t*>(workspace), A) > workspace_bytes) return MQ_ERR_WORKSPACE_TOO_SMALL;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int router_vec = aligned16(L.router);
  const unsigned grid = (unsigned)(A.E + (format == F_INT8 ? A.T : 1));
  if (T == 1) moe_small_router<1><<<grid, 128, 0, st>>>(A, router_vec);
  else if (T <= 4) moe_small_router<4><<<grid, 128, 0, st>>>(A, router_vec);
  else if (T <= 8) moe_small_router<8><<<grid, 128, 0, st>>>(A, router_vec);
  else moe_small_router<16><<<grid, 128, 0, st>>>(A, router_vec);
  const int rc = check_launch();
  if (rc != MQ_OK) return rc;
  return T <= 8 ? launch_format<1>(A, format, st) : launch_format<2>(A, format, st);
}
