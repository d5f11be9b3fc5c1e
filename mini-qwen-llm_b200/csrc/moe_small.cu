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
//   * the weights come by tensor-map copies, issued by one warp, through a ring of 128 to 160 KB that runs on through the
//     barrier, so that the first weights of the down projection arrive under it.  Sixteen warps multiply: a lane's 16-byte
//     pieces are, in a suitable order of k, the fragments of mma.sync (tokens are its 8 columns), so the tensor cores cost
//     nothing here, and all tokens of an expert cost one pass over its weights.  Three warps finish the tiles of h.
//     (A warp copying for itself, through registers or a ring of its own, spent its time on addresses: 3.7 TB/s.)
// Every wait is bounded; when one runs out, MQ_DEV_WAIT_EXPIRED is set and the output is invalid.
#include "int8.cuh"
#include "tc5.cuh"

namespace mq {
namespace {

using namespace int8;

constexpr int MAX_T = 16, MAX_E = 1024, MAX_K = 32;
constexpr int WARPS = 16;                          // that multiply
constexpr int FINISH = 3;                          // that finish the tiles of h; one more issues the copies
constexpr int THREADS = (WARPS + FINISH + 1) * 32;
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
  int tile, box_rows;                              // columns of h in a tile; rows of a down box, or word rows of an int4 gate box
  unsigned* counter;                               // workspace from here on
  uint32_t* amax;                                  // [T * K] largest |h| of a slot, as bits
  float* logits;                                   // [T, E]
  int8_t* xq;                                      // [T, H]
  int8_t* hq;                                      // [T * K, I]
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

// Tables in shared memory behind the rings and the sums.
struct Tables {
  uint32_t* mask;      // [E] tokens of the expert
  uint16_t* pos;       // [E] its place among the experts hit
  uint16_t* hit;       // [hits] the expert
  uint8_t* count;      // [hits] its tokens; they are columns 0, 1, ... of its products:
  uint16_t* slot;      // [hits, MAX_T] token * MAX_K + which of its experts it is
  uint16_t* ids;       // [T, MAX_K] the tokens' experts
  float* w;            // [T, MAX_K] and their weights
  __host__ __device__ static size_t bytes(int T, int E, int K) {
    const size_t hits = (size_t)(E < T * K ? E : T * K);
    return hits * (MAX_T * 2 + 3) + (size_t)E * 6 + (size_t)T * MAX_K * 6 + 16;
  }
  __device__ Tables(uint8_t* p, int T, int E, int K) {
    const int hits = min(E, T * K);
    w = reinterpret_cast<float*>(p);
    mask = reinterpret_cast<uint32_t*>(w + T * MAX_K);
    slot = reinterpret_cast<uint16_t*>(mask + E);
    ids = slot + hits * MAX_T;
    pos = ids + T * MAX_K;
    hit = pos + E;
    count = reinterpret_cast<uint8_t*>(hit + hits);
  }
};

// A unit is what a warp multiplies at a time: 128 bytes of k of 16 weight rows (gate and up: 8 of either), or int4 words:
// 128 k of 16 columns of gate and up, 256 k of 16 columns of down.  A stage of the ring holds a unit for each warp.
template <int F> struct Fmt {
  static constexpr bool W4 = F == F_INT4;
  static constexpr int SIZE = F == F_INT8 ? 1 : 2;
  static constexpr int UNIT_K = W4 ? 128 : 128 / SIZE, UNIT2_K = W4 ? 256 : 128 / SIZE;
  static constexpr int MT = W4 ? 2 : 1;            // accumulator tiles: int4 gate and up apart, else 8 + 8 rows in one
};
constexpr int UNIT = 2048, STAGE = WARPS * UNIT;
// Stages of the ring; the partial sums (two buffers) and the tables lie behind it.
__host__ __device__ constexpr int ring_stages(int f, int octets) { return f == F_INT4 && octets == 2 ? 4 : 5; }
__host__ __device__ constexpr size_t part_bytes(int f, int octets) { return (size_t)WARPS * 512 * (f == F_INT4 ? 2 : 1) * octets; }
__host__ __device__ constexpr size_t front_bytes(int f, int octets) {
  return (size_t)ring_stages(f, octets) * STAGE + 2 * part_bytes(f, octets);
}

// One barrier over the grid; `arrive` may come well before `wait`.  Thread 0 of each CTA, between barriers of the CTA.
__device__ __forceinline__ void grid_arrive(unsigned* counter) {
  __threadfence();
  atomicAdd(counter, 1u);
}
__device__ __forceinline__ bool grid_wait(unsigned* counter, unsigned target) {
  uint32_t seen = 0, looks = 0;
  do {
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(seen) : "l"(counter) : "memory");
  } while (seen < target && ++looks < POLL_LIMIT);
  __threadfence();
  return seen >= target;
}

// The copies, from the weights' tensor maps.
__device__ __forceinline__ void copy_box(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
               ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
__device__ __forceinline__ void copy_box(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
               ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3) : "memory");
}
// A barrier of some of the CTA's warps.
template <int ID, int N> __device__ __forceinline__ void warps_meet() { asm volatile("bar.sync %0, %1;" ::"n"(ID), "n"(N * 32) : "memory"); }

struct SmallMaps { CUtensorMap gate, up, down; };  // dense and int8: gate and up rows in one

template <int F, int OCT, typename OutT>
__global__ void __launch_bounds__(THREADS, 1) moe_small_layer(const SmallArgs A, const __grid_constant__ SmallMaps maps) {
  using namespace tc5;
  using Acc = typename std::conditional<F == F_INT8, int, float>::type;
  constexpr int SIZE = Fmt<F>::SIZE, UNIT_K = Fmt<F>::UNIT_K, UNIT2_K = Fmt<F>::UNIT2_K, MT = Fmt<F>::MT;
  constexpr bool W4 = F == F_INT4;
  constexpr int STAGES = ring_stages(F, OCT);
  constexpr int HP = F == F_INT8 ? 1 : 2;          // 16-byte pieces of h per step and lane in the down projection
  extern __shared__ uint8_t small_smem_raw[];
  uint8_t* const small_smem = small_smem_raw + ((1024u - (smem_addr(small_smem_raw) & 1023u)) & 1023u);   // the copies' swizzle
  uint8_t* part = small_smem + STAGES * STAGE;
  const Tables tab(small_smem + front_bytes(F, OCT), A.T, A.E, A.K);
  __shared__ int s_hits, s_ok, s_abort;
  __shared__ __align__(8) uint64_t s_bars[2 * STAGES + 4];
  const uint32_t bars = smem_addr(s_bars), ring = smem_addr(small_smem);
  auto full = [&](int i) { return bars + 8u * i; };
  auto empty = [&](int i) { return bars + 8u * (STAGES + i); };
  auto pfull = [&](int i) { return bars + 8u * (2 * STAGES + i); };        // partial sums written
  auto pfree = [&](int i) { return bars + 8u * (2 * STAGES + 2 + i); };    // and read
  const int tid = threadIdx.x, lane = tid & 31, warp = (int)uniform(tid >> 5), g = lane >> 2, q4 = lane & 3;
  const int T = A.T, H = A.H, I = A.I, E = A.E, K = A.K, G = (int)gridDim.x, cta = (int)blockIdx.x;
  volatile int* abort_flag = &s_abort;

  // ------------------------------------------------------------------ who goes where
  if (tid == THREADS - 1) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(full(i), 1);
      mbar_init(empty(i), WARPS);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(pfull(i), WARPS);
      mbar_init(pfree(i), FINISH);
    }
    s_abort = 0;
    mbar_init_fence();
  }
  for (int e = tid; e < E; e += THREADS) tab.mask[e] = 0;
  if (warp < T) {
    const float* row = A.logits + warp * E;
    if (E <= 128) select_experts<4>(row, E, K, A.renorm, lane, tab.ids + warp * MAX_K, tab.w + warp * MAX_K);
    else select_experts<MAX_E / 32>(row, E, K, A.renorm, lane, tab.ids + warp * MAX_K, tab.w + warp * MAX_K);
  }
  __syncthreads();
  if (tid < T * MAX_K && lane < K) atomicOr(&tab.mask[tab.ids[tid]], 1u << warp);      // warp: the token
  __syncthreads();
  if (warp == 0) {
    int n = 0;
    for (int e0 = 0; e0 < E; e0 += 32) {
      const uint32_t m = e0 + lane < E ? tab.mask[e0 + lane] : 0u;
      const unsigned any = __ballot_sync(0xffffffffu, m != 0);
      const int at = n + __popc(any & ((1u << lane) - 1u));
      if (m != 0) {
        tab.hit[at] = (uint16_t)(e0 + lane);
        tab.pos[e0 + lane] = (uint16_t)at;
        tab.count[at] = (uint8_t)__popc(m);
      }
      n += __popc(any);
    }
    if (lane == 0) s_hits = n;
  }
  __syncthreads();
  if (tid < T * MAX_K && lane < K) {
    const int e = tab.ids[tid];
    tab.slot[tab.pos[e] * MAX_T + __popc(tab.mask[e] & ((1u << warp) - 1u))] = (uint16_t)tid;
  }
  __syncthreads();
  const int hits = s_hits;
  auto row_of = [&](int slot) { return (slot >> 5) * K + (slot & 31); };   // row of h
  static_assert(MAX_K == 32 && MAX_T * MAX_K <= THREADS, "a slot is a thread");

  // ------------------------------------------------------------------ the work
  // Gate and up: the columns of h of all experts hit, one after the other, are cut into equal ranges (int4: by 16 columns).
  // A CTA walks its range in tiles of A.tile columns; `ksplit` warps share a tile's k in units, so that `at_once` tiles are in
  // work, for `passes` stages.  Down: a CTA's output columns (rows of the weights; int4: by 16), 16 at a time; the (expert,
  // unit of k) pairs of a tile are dealt out to the warps in turn.
  const int lo = W4 ? (int)((int64_t)hits * (I / 16) * cta / G) * 16 : (int)((int64_t)hits * I * cta / G);
  const int hi = W4 ? (int)((int64_t)hits * (I / 16) * (cta + 1) / G) * 16 : (int)((int64_t)hits * I * (cta + 1) / G);
  const int out_lo = W4 ? (int)((int64_t)(H / 16) * cta / G) * 16 : (int)((int64_t)H * cta / G);
  const int out_hi = W4 ? (int)((int64_t)(H / 16) * (cta + 1) / G) * 16 : (int)((int64_t)H * (cta + 1) / G);
  const int units = (H + UNIT_K - 1) / UNIT_K, units2 = (I + UNIT2_K - 1) / UNIT2_K;
  const int TW = A.tile;
  int tiles;
  {
    const int p0 = lo / I, p1 = hi / I, r0 = lo - p0 * I, r1 = hi - p1 * I;
    tiles = p0 == p1 ? (hi - lo + TW - 1) / TW
                     : (I - r0 + TW - 1) / TW + (p1 - p0 - 1) * ((I + TW - 1) / TW) + (r1 + TW - 1) / TW;
  }
  int ksplit = WARPS;
  while (ksplit / 2 >= units) ksplit >>= 1;
  const int at_once = WARPS / ksplit, passes = (units + ksplit - 1) / ksplit, rounds = (tiles + at_once - 1) / at_once;
  const int tasks = hits * units2;
  struct Walk { int pos, place, end; };            // column over all experts, the expert's place, where its columns end
  auto width = [&](const Walk& c) { return min(TW, min(c.end, hi) - c.pos); };
  auto next_tile = [&](Walk& c) {
    c.pos += width(c);
    if (c.pos == c.end) { ++c.place; c.end += I; }
  };
  auto skip_tiles = [&](Walk& c, int n) {
    for (int i = 0; i < n && c.pos < hi; ++i) next_tile(c);
  };
  Walk walk;
  walk.pos = lo;
  walk.place = lo / I;
  walk.end = (walk.place + 1) * I;

  if (warp == WARPS + FINISH) {
    // ------------------------------------------------------------------ copies: first gate and up, then down
    // Weights only, so they run on through the barrier over the grid.  One elected lane issues, from uniform registers.
    const bool leader = elect_one();
    int stage = 0, filled = 0;
    uint32_t phase = 0;
    bool ok = true;
    auto next_stage = [&] {
      ++filled;
      if (++stage == STAGES) { stage = 0; phase ^= 1u; }
    };
    for (int round = 0; round < rounds && ok; ++round) {
      for (int pass = 0; pass < passes && ok; ++pass) {
        ok = mbar_wait_warp(empty(stage), phase ^ 1u, abort_flag, A.d_status);
        if (!ok) break;
        const int u0 = pass * ksplit, n = min(ksplit, units - u0), live = min(at_once, tiles - round * at_once);
        const uint32_t dst = ring + stage * STAGE, bar = full(stage);
        if (leader) mbar_expect_tx(bar, W4 ? live * 2 * A.box_rows * 64 : live * n * 2 * TW * 128);
        Walk c = walk;
        for (int i = 0; i < live; ++i) {
          const int e = (int)uniform(tab.hit[c.place]), col = (int)uniform(c.pos - (c.end - I));
          const uint32_t at = dst + i * ksplit * UNIT;
          if (W4) {
            if (leader) {
              copy_box(at, &maps.gate, bar, col, u0 * 16, e);
              copy_box(at + ksplit * (UNIT / 2), &maps.up, bar, col, u0 * 16, e);
            }
          } else {
            for (int u = 0; u < n; ++u)
              if (leader) copy_box(at + u * UNIT, &maps.gate, bar, (u0 + u) * UNIT_K, col, 0, e);
          }
          next_tile(c);
        }
        __syncwarp();
        next_stage();
      }
      skip_tiles(walk, at_once);
    }
    for (int row0 = out_lo; row0 < out_hi && ok; row0 += 16) {
      int place = 0, u = 0;
      for (int task = 0; task < tasks && ok; task += WARPS) {
        ok = mbar_wait_warp(empty(stage), phase ^ 1u, abort_flag, A.d_status);
        if (!ok) break;
        const int live = min(WARPS, tasks - task);
        const uint32_t dst = ring + stage * STAGE, bar = full(stage);
        if (leader) mbar_expect_tx(bar, live * (W4 ? UNIT : A.box_rows * 128));
        for (int i = 0; i < live; ++i) {
          const int e = (int)uniform(tab.hit[place]);
          if (leader) {
            if (W4) copy_box(dst + i * UNIT, &maps.down, bar, row0, u * 32, e);
            else copy_box(dst + i * UNIT, &maps.down, bar, u * UNIT2_K, row0, e);
          }
          if (++u == units2) { u = 0; ++place; }
        }
        __syncwarp();
        next_stage();
      }
    }
    // nothing is on its way any more when the CTA ends
    for (int f = max(0, filled - STAGES); f < filled; ++f)
      mbar_wait_limited(full(f % STAGES), (uint32_t)(f / STAGES) & 1u, ok ? SPIN_LIMIT : 1u << 16);
    return;
  }

  auto zero_pair = [](uint32_t z) {                // -(128 + z), twice
    const float v = -(128.0f + (float)(z & 15u));
    return __floats2bfloat162_rn(v, v);
  };
  // A lane's two 16-byte pieces of row `line` of a unit (rows of 128 bytes, swizzled by the copies).
  auto piece = [&](const uint8_t* unit, int line, int s) {
    return *reinterpret_cast<const uint4*>(unit + line * 128 + (((2 * q4 + s) ^ (line & 7)) << 4));
  };
  int stage = 0;
  uint32_t phase = 0;
  bool ok = true;                                  // a wait that ran out: the rest is walked through without waiting
  auto release = [&] {
    __syncwarp();
    if (lane == 0) mbar_arrive(empty(stage));
    if (++stage == STAGES) { stage = 0; phase ^= 1u; }
  };

  if (warp < WARPS) {
    // ------------------------------------------------------------------ gate and up projections
    const int kw = warp % ksplit, tg = warp / ksplit;
    skip_tiles(walk, tg);
    const uint8_t* rows = F == F_INT8 ? reinterpret_cast<const uint8_t*>(A.xq) : reinterpret_cast<const uint8_t*>(A.x);
    // x of the lane's token for a unit (column o * 8 + g of the expert); int4: the group's scales and zero points too
    constexpr int XS = W4 ? 4 : 2;
    auto load_x = [&](uint4 (&b)[XS], int place, int u, int o) {
      const bool live = 8 * o + g < tab.count[place];
      const uint8_t* row = rows + (size_t)(live ? tab.slot[place * MAX_T + 8 * o + g] >> 5 : 0) * H * SIZE;
#pragma unroll
      for (int s = 0; s < XS; ++s) {
        const int k = W4 ? u * 256 + 64 * s + 16 * q4 : u * 128 + 32 * q4 + 16 * s;      // bytes
        b[s] = live && k < H * SIZE ? __ldg(reinterpret_cast<const uint4*>(row + k)) : make_uint4(0u, 0u, 0u, 0u);
      }
    };
    auto load_sz = [&](uint32_t (&sz)[4], const Walk& c, int u) {
      if constexpr (W4) {
        const size_t n = (size_t)(c.pos - (c.end - I)) + 2 * g, row = (size_t)tab.hit[c.place] * (H / A.group) + u * 128 / A.group;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          sz[j] = __ldg(reinterpret_cast<const uint32_t*>(A.sc[j] + row * I + n));
          sz[2 + j] = (uint32_t)__ldg(A.qz[j] + row * (I / 8) + (n >> 3)) >> (4 * (n & 7));
        }
      }
    };
    uint4 b[XS], nb[XS];
    uint32_t sz[4] = {}, nsz[4] = {};
    if (walk.pos < hi && kw < units) {
      load_x(b, walk.place, kw, 0);
      load_sz(sz, walk, kw);
    }
    for (int round = 0; round < rounds; ++round) {
      const bool mine = walk.pos < hi;
      Walk nxt = walk;
      skip_tiles(nxt, at_once);
      Acc acc[OCT][MT][4] = {};
      for (int pass = 0; pass < passes; ++pass) {
        const int u = pass * ksplit + kw;
        // of the unit after this one
        const bool last = pass + 1 == passes;
        const Walk& c = last ? nxt : walk;
        const int nu = last ? kw : u + ksplit;
        if (c.pos < hi && nu < units) {
          load_x(nb, c.place, nu, 0);
          load_sz(nsz, c, nu);
        }
        if (ok) ok = mbar_wait_warp(full(stage), phase, abort_flag, A.d_status);
        if (mine && u < units) {
          const uint8_t* unit = small_smem + stage * STAGE + (W4 ? tg * ksplit * UNIT + kw * (UNIT / 2) : warp * UNIT);
#pragma unroll
          for (int o = 0; o < OCT; ++o) {
            if (o == 1) {
              if (tab.count[walk.place] <= 8) break;
              load_x(b, walk.place, u, 1);
            }
            if constexpr (W4) {
              float grp[MT][4] = {};
#pragma unroll
              for (int s = 0; s < 4; ++s) {
                const uint4 x = pair_up(b[s]);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                  const uint2 w = *reinterpret_cast<const uint2*>(unit + j * ksplit * (UNIT / 2) + (4 * s + q4) * 64 + 8 * g);
                  uint32_t v0[4], v1[4];
                  unpack_int4(w.x, zero_pair(sz[2 + j]), v0);
                  unpack_int4(w.y, zero_pair(sz[2 + j] >> 4), v1);
                  mma_bf16(grp[j % MT], v0[0], v1[0], v0[1], v1[1], x.x, x.y);
                  mma_bf16(grp[j % MT], v0[2], v1[2], v0[3], v1[3], x.z, x.w);
                }
              }
#pragma unroll
              for (int j = 0; j < 2; ++j) {        // a unit lies inside a quantisation group
                const float2 sc = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&sz[j]));
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[o][j % MT][i] = fmaf(grp[j % MT][i], i < 2 ? sc.x : sc.y, acc[o][j % MT][i]);
              }
            } else {
#pragma unroll
              for (int s = 0; s < 2; ++s) {
                const uint4 r = piece(unit, g, s), r8 = piece(unit, TW + g, s);
                if constexpr (F == F_INT8) {
                  mma_s8(acc[o][0], r.x, r8.x, r.y, r8.y, b[s].x, b[s].y);
                  mma_s8(acc[o][0], r.z, r8.z, r.w, r8.w, b[s].z, b[s].w);
                } else if constexpr (F == F_F16) {
                  mma_f16(acc[o][0], r.x, r8.x, r.y, r8.y, b[s].x, b[s].y);
                  mma_f16(acc[o][0], r.z, r8.z, r.w, r8.w, b[s].z, b[s].w);
                } else {
                  mma_bf16(acc[o][0], r.x, r8.x, r.y, r8.y, b[s].x, b[s].y);
                  mma_bf16(acc[o][0], r.z, r8.z, r.w, r8.w, b[s].z, b[s].w);
                }
              }
            }
          }
        }
        release();
#pragma unroll
        for (int s = 0; s < XS; ++s) b[s] = nb[s];
#pragma unroll
        for (int j = 0; j < 4; ++j) sz[j] = nsz[j];
      }
      const int buf = round & 1;
      if (ok) ok = mbar_wait_warp(pfree(buf), ((round >> 1) & 1) ^ 1u, abort_flag, A.d_status);
#pragma unroll
      for (int o = 0; o < OCT; ++o)
#pragma unroll
        for (int j = 0; j < MT; ++j)
          *reinterpret_cast<int4*>(part + buf * part_bytes(F, OCT) + (((warp * OCT + o) * MT + j) * 32 + lane) * 16) =
              *reinterpret_cast<const int4*>(acc[o][j]);
      __syncwarp();
      if (lane == 0) mbar_arrive(pfull(buf));
      walk = nxt;
    }
  } else {
    // ------------------------------------------------------------------ sums over the warps, SwiGLU
    // A warp takes a tile's octet of tokens: a lane a fragment position, its sums over the warps in order.
    for (int round = 0; round < rounds; ++round) {
      const int buf = round & 1;
      if (ok) ok = mbar_wait_warp(pfull(buf), (round >> 1) & 1, abort_flag, A.d_status);
      const int live_tiles = min(at_once, tiles - round * at_once);
      for (int slot = 0; slot < live_tiles; ++slot) {
        const int place = walk.place, col0 = walk.pos - (walk.end - I), cols = width(walk);
        next_tile(walk);
        const size_t e = tab.hit[place];
#pragma unroll
        for (int o = 0; o < OCT; ++o) {
          const int live = (int)tab.count[place] - 8 * o;                  // columns of this octet
          if (live <= 0 || (slot * OCT + o) % FINISH != warp - WARPS) continue;
          Acc sum[MT][4] = {};
#pragma unroll 8
          for (int w = 0; w < ksplit; ++w)
#pragma unroll
            for (int j = 0; j < MT; ++j) {
              const int4 raw = *reinterpret_cast<const int4*>(part + buf * part_bytes(F, OCT) +
                                                              ((((slot * ksplit + w) * OCT + o) * MT + j) * 32 + lane) * 16);
              const Acc* c = reinterpret_cast<const Acc*>(&raw);
#pragma unroll
              for (int i = 0; i < 4; ++i) sum[j][i] += c[i];
            }
#pragma unroll
          for (int i = 0; i < (W4 ? 4 : 2); ++i) {
            const int n = 2 * q4 + (i & 1), col = W4 ? 2 * g + (i >> 1) : g;
            float v = 0.0f;
            const int code = n < live ? tab.slot[place * MAX_T + 8 * o + n] : 0;
            const size_t row = row_of(code);
            if (n < live && col < cols) {
              float gv, uv;
              if constexpr (F == F_INT8) {
                const float* s = A.s13 + e * 2 * I + col0 + col;
                const float sx = A.xs[code >> 5];
                gv = __fmul_rn(__fmul_rn(__int2float_rn(sum[0][i]), sx), s[0]);
                uv = __fmul_rn(__fmul_rn(__int2float_rn(sum[0][2 + i]), sx), s[I]);
              } else {
                gv = (float)sum[0][i];
                uv = W4 ? (float)sum[MT - 1][i] : (float)sum[0][(2 + i) & 3];
              }
              const float p = expf(-fabsf(gv));
              v = __fdividef(gv < 0.0f ? p * gv : gv, 1.0f + p) * uv;
              if (F == F_BF16 || W4) {
                __nv_bfloat16* h = reinterpret_cast<__nv_bfloat16*>(A.h) + row * 2 * I + col0 + col;
                const __nv_bfloat16 high = __float2bfloat16_rn(v);
                h[0] = high;
                h[I] = __float2bfloat16_rn(__hisinf(high) ? 0.0f : v - __bfloat162float(high));
              } else {
                reinterpret_cast<float*>(A.h)[row * I + col0 + col] = v;
              }
            }
            if (F == F_INT8) {                     // the row's largest |h|: first over the columns of the tile
              uint32_t bits = abs_bits(v);
#pragma unroll
              for (int s = 4; s < 32; s <<= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, s));
              if (g == 0 && n < live) atomicMax(A.amax + row, bits);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(pfree(buf));
    }
  }

  // ------------------------------------------------------------------ every h is there
  warps_meet<1, WARPS + FINISH>();
  if (tid == 0) {
    grid_arrive(A.counter);
    s_ok = grid_wait(A.counter, (unsigned)G);
  }
  warps_meet<1, WARPS + FINISH>();
  if (F == F_INT8 && s_ok != 0) {                  // rows of h to int8, a warp a row over the whole grid, and a second barrier
    for (int row = cta * WARPS + warp; row < T * K && warp < WARPS; row += G * WARPS) {
      const RowScale r = row_scale(__ldcg(A.amax + row));
      const float* src = reinterpret_cast<const float*>(A.h) + (size_t)row * I;
#pragma unroll 4
      for (int k = 4 * lane; k < I; k += 128) {
        const float4 v = __ldcg(reinterpret_cast<const float4*>(src + k));
        *reinterpret_cast<uint32_t*>(A.hq + (size_t)row * I + k) =
            ((uint32_t)quantize(v.x, r) & 0xffu) | ((uint32_t)quantize(v.y, r) & 0xffu) << 8 |
            ((uint32_t)quantize(v.z, r) & 0xffu) << 16 | ((uint32_t)quantize(v.w, r) & 0xffu) << 24;
      }
    }
    warps_meet<1, WARPS + FINISH>();
    if (tid == 0) {
      grid_arrive(A.counter);
      s_ok = grid_wait(A.counter, 2u * (unsigned)G);
    }
    warps_meet<1, WARPS + FINISH>();
  }
  if (warp >= WARPS) return;
  if (s_ok == 0) {
    if (tid == 0 && A.d_status != nullptr) atomicOr(A.d_status, (int)MQ_DEV_WAIT_EXPIRED);
    return;
  }

  // ------------------------------------------------------------------ down projection and weighted sum
  // A warp's sums of a tile, [tokens, 16 columns], are its own piece of shared memory, to which a unit's columns are added
  // with their tokens' weights.  A token that did not choose the expert takes nothing from it, whatever its weights hold.
  float* mine = reinterpret_cast<float*>(part) + warp * (128 * OCT);
  constexpr int HS = 2;                            // steps that are loaded together; int4: a quarter of a unit
  constexpr int QUARTERS = W4 ? 4 : 1;
  auto load_h = [&](uint4 (&b)[HS][HP], int place, int u, int quarter, int o) {
    const bool live = 8 * o + g < tab.count[place];
    const size_t row = live ? row_of(tab.slot[place * MAX_T + 8 * o + g]) : 0;
#pragma unroll
    for (int s = 0; s < HS; ++s) {
      const int k = W4 ? u * UNIT2_K + 64 * quarter + 32 * s + 8 * q4 : u * UNIT2_K + (32 / SIZE) * q4 + (16 / SIZE) * s;
      const bool in = live && k < I;
#pragma unroll
      for (int p = 0; p < HP; ++p) {
        b[s][p] = make_uint4(0u, 0u, 0u, 0u);
        if (in) {
          const uint8_t* src;
          if (F == F_INT8) src = reinterpret_cast<const uint8_t*>(A.hq) + row * I + k;
          else if (F == F_F16) src = reinterpret_cast<const uint8_t*>(A.h) + (row * I + k) * 4 + 16 * p;
          else src = reinterpret_cast<const uint8_t*>(A.h) + ((row * 2 + p) * I + k) * 2;
          b[s][p] = __ldcg(reinterpret_cast<const uint4*>(src));
        }
      }
    }
  };
  uint4 b[HS][HP], nb[HS][HP];
  int place = warp / units2, u = warp - place * units2;
  const int step_place = WARPS / units2, step_u = WARPS - step_place * units2;
  if (warp < tasks) load_h(b, place, u, 0, 0);
  for (int row0 = out_lo; row0 < out_hi; row0 += 16) {
    for (int i = lane; i < 128 * OCT; i += 32) mine[i] = 0.0f;
    __syncwarp();
    for (int task = warp; task - warp < tasks; task += WARPS) {
      int np = place + step_place, nu = u + step_u;
      if (nu >= units2) { nu -= units2; ++np; }
      const bool live_task = task < tasks;
      if (task + WARPS >= tasks) {                 // the next tile's first
        np = warp / units2;
        nu = warp - np * units2;
      }
      uint32_t sc[2] = {}, zp[2] = {};
      if constexpr (W4) {
        if (live_task) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const size_t n = (size_t)row0 + 2 * g, row = (size_t)tab.hit[place] * (I / A.group) + min(u * 256 + 128 * j, I - 1) / A.group;
            sc[j] = __ldg(reinterpret_cast<const uint32_t*>(A.sc[2] + row * H + n));
            zp[j] = (uint32_t)__ldg(A.qz[2] + row * (H / 8) + (n >> 3)) >> (4 * (n & 7));
          }
        }
      }
      if (ok) ok = mbar_wait_warp(full(stage), phase, abort_flag, A.d_status);
      const uint8_t* unit = small_smem + stage * STAGE + warp * UNIT;
      if (live_task) {
        Acc acc[OCT][4] = {};
        const bool second = OCT == 2 && tab.count[place] > 8;
#pragma unroll
        for (int quarter = 0; quarter < QUARTERS; ++quarter) {
          if (quarter + 1 < QUARTERS) load_h(nb, place, u, quarter + 1, 0);
          else if (np < hits) load_h(nb, np, nu, 0, 0);
#pragma unroll
          for (int o = 0; o < OCT; ++o) {
            if (o == 1) {
              if (!second) break;
              load_h(b, place, u, quarter, 1);
            }
            float grp[4] = {};
#pragma unroll
            for (int s = 0; s < HS; ++s) {
              if constexpr (W4) {
                const uint4 hi4 = pair_up(b[s][0]), lo4 = pair_up(b[s][HP - 1]);
                const uint2 w = *reinterpret_cast<const uint2*>(unit + (8 * quarter + 4 * s + q4) * 64 + 8 * g);
                uint32_t v0[4], v1[4];
                unpack_int4(w.x, zero_pair(zp[quarter / 2]), v0);
                unpack_int4(w.y, zero_pair(zp[quarter / 2] >> 4), v1);
                mma_bf16(grp, v0[0], v1[0], v0[1], v1[1], lo4.x, lo4.y);
                mma_bf16(grp, v0[2], v1[2], v0[3], v1[3], lo4.z, lo4.w);
                mma_bf16(grp, v0[0], v1[0], v0[1], v1[1], hi4.x, hi4.y);
                mma_bf16(grp, v0[2], v1[2], v0[3], v1[3], hi4.z, hi4.w);
              } else {
                const uint4 r4 = piece(unit, g, s), r84 = piece(unit, 8 + g, s);
                if constexpr (F == F_INT8) {
                  const uint4 x = b[s][0];
                  mma_s8(acc[o], r4.x, r84.x, r4.y, r84.y, x.x, x.y);
                  mma_s8(acc[o], r4.z, r84.z, r4.w, r84.w, x.z, x.w);
                } else if constexpr (F == F_F16) {
                  const uint32_t r[4] = {r4.x, r4.y, r4.z, r4.w}, r8[4] = {r84.x, r84.y, r84.z, r84.w};
                  const uint32_t x[8] = {b[s][0].x, b[s][0].y, b[s][0].z, b[s][0].w, b[s][HP - 1].x, b[s][HP - 1].y, b[s][HP - 1].z, b[s][HP - 1].w};
#pragma unroll
                  for (int p = 0; p < 4; ++p) {
                    // a tf32 number is the upper 19 bits of an fp32 one: fp16 fits, h is a sum of two
                    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&r[p]));
                    const float2 a8 = __half22float2(*reinterpret_cast<const __half2*>(&r8[p]));
                    const float v0 = __uint_as_float(x[2 * p]), v1 = __uint_as_float(x[2 * p + 1]);
                    const uint32_t h0 = x[2 * p] & 0xffffe000u, h1 = x[2 * p + 1] & 0xffffe000u;
                    const uint32_t l0 = isinf(v0) ? 0u : __float_as_uint(v0 - __uint_as_float(h0)) & 0xffffe000u;
                    const uint32_t l1 = isinf(v1) ? 0u : __float_as_uint(v1 - __uint_as_float(h1)) & 0xffffe000u;
                    const uint32_t a0 = __float_as_uint(a.x), a1 = __float_as_uint(a8.x), a2 = __float_as_uint(a.y), a3 = __float_as_uint(a8.y);
                    mma_tf32(acc[o], a0, a1, a2, a3, l0, l1);
                    mma_tf32(acc[o], a0, a1, a2, a3, h0, h1);
                  }
                } else {
                  const uint4 h4 = b[s][0], l4 = b[s][HP - 1];
                  mma_bf16(acc[o], r4.x, r84.x, r4.y, r84.y, l4.x, l4.y);
                  mma_bf16(acc[o], r4.z, r84.z, r4.w, r84.w, l4.z, l4.w);
                  mma_bf16(acc[o], r4.x, r84.x, r4.y, r84.y, h4.x, h4.y);
                  mma_bf16(acc[o], r4.z, r84.z, r4.w, r84.w, h4.z, h4.w);
                }
              }
            }
            if constexpr (W4) {
              const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&sc[quarter / 2]));
#pragma unroll
              for (int i = 0; i < 4; ++i) acc[o][i] = fmaf(grp[i], i < 2 ? f.x : f.y, acc[o][i]);
            }
          }
#pragma unroll
          for (int s = 0; s < HS; ++s)
#pragma unroll
            for (int p = 0; p < HP; ++p) b[s][p] = nb[s][p];
        }
#pragma unroll
        for (int o = 0; o < OCT; ++o) {
          const int live = (int)tab.count[place] - 8 * o;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int n = 2 * q4 + (i & 1);
            if (n < live) {
              const int slot = tab.slot[place * MAX_T + 8 * o + n];
              const int col = W4 ? 2 * g + (i >> 1) : g + 8 * (i >> 1);
              float v = (float)acc[o][i];
              if (F == F_INT8)
                v = v * scale_of(__ldcg(A.amax + row_of(slot))) *
                    (row0 + col < out_hi ? A.s2[(size_t)tab.hit[place] * H + row0 + col] : 0.0f);
              float* to = mine + (slot >> 5) * 16 + col;
              *to = fmaf(v, tab.w[slot], *to);
            }
          }
        }
      } else if (np < hits) {
        load_h(b, np, nu, 0, 0);
      }
      release();
      place = np;
      u = nu;
    }
    warps_meet<2, WARPS>();
    // the warps' sums, in order, then the one rounding
    if (tid < 128 * OCT) {
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) v += reinterpret_cast<const float*>(part)[w * (128 * OCT) + tid];
      const int tok = tid / 16, col = row0 + tid % 16;
      if (tok < T && col < out_hi) {
        const size_t at = (size_t)tok * H + col;
        if (A.residual != nullptr) v += to_float<OutT>(reinterpret_cast<const OutT*>(A.residual)[at]);
        reinterpret_cast<OutT*>(A.out)[at] = from_float<OutT>(v);
      }
    }
    if (row0 + 16 < out_hi) warps_meet<2, WARPS>();
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
    case F_INT8: return H % 16 == 0 && I % 16 == 0 && H <= 131071 && I <= 131071;
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
  const bool int8 = format_of(L) == F_INT8;
  A.xq = int8 ? (int8_t*)take((size_t)(T * L.hidden)) : nullptr;
  A.hq = int8 ? (int8_t*)take(S * (size_t)L.inter) : nullptr;
  return used;
}

bool small_layer_ok(const mq_moe_layer* L) {
  return L != nullptr && L->hidden > 0 && L->inter > 0 && L->experts > 0 && L->top_k > 0 && L->group_size >= 0 &&
         valid_dtype(L->dtype) && valid_dtype(L->router_dtype) && !(L->int8_experts && L->group_size > 0);
}

bool small_map(CUtensorMap* map, CUtensorMapDataType type, const void* base, int rank, const cuuint64_t* dims,
               const cuuint64_t* strides, const cuuint32_t* box, bool swizzle) {
  EncodeTiledFn fn = tensor_map_encoder();
  const cuuint32_t estr[4] = {1u, 1u, 1u, 1u};
  return fn && fn(map, type, (cuuint32_t)rank, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Chooses the tile shapes and describes the weights to the copies.
template <int F>
bool small_maps(SmallArgs& A, int sms, SmallMaps& m) {
  const cuuint64_t H = (cuuint64_t)A.H, I = (cuuint64_t)A.I, E = (cuuint64_t)A.E;
  if constexpr (F == F_INT4) {
    A.tile = 16;
    A.box_rows = A.H / 8 < 256 ? A.H / 8 : 256;
    const cuuint64_t in_dims[3] = {I, H / 8, E}, in_strides[2] = {I * 4, I * (H / 8) * 4};
    const cuuint64_t out_dims[3] = {H, I / 8, E}, out_strides[2] = {H * 4, H * (I / 8) * 4};
    const cuuint32_t in_box[3] = {16, (cuuint32_t)A.box_rows, 1}, out_box[3] = {16, 32, 1};
    return small_map(&m.gate, CU_TENSOR_MAP_DATA_TYPE_INT32, A.qw[0], 3, in_dims, in_strides, in_box, false) &&
           small_map(&m.up, CU_TENSOR_MAP_DATA_TYPE_INT32, A.qw[1], 3, in_dims, in_strides, in_box, false) &&
           small_map(&m.down, CU_TENSOR_MAP_DATA_TYPE_INT32, A.qw[2], 3, out_dims, out_strides, out_box, false);
  } else {
    constexpr int SIZE = Fmt<F>::SIZE;
    const CUtensorMapDataType type = F == F_INT8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                     : F == F_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    // one token hits top_k experts: the tiles of a CTA's share can be made equal
    A.tile = 8;
    if (A.T == 1) {
      const int share = (int)(((int64_t)A.K * A.I + sms - 1) / sms), n = (share + 7) / 8;
      A.tile = (share + n - 1) / n;
    }
    const int rows = (A.H + sms - 1) / sms;
    A.box_rows = rows < 16 ? rows : 16;
    const cuuint64_t in_dims[4] = {H, I, 2, E}, in_strides[3] = {H * SIZE, I * H * SIZE, 2 * I * H * SIZE};
    const cuuint64_t out_dims[3] = {I, H, E}, out_strides[2] = {I * SIZE, H * I * SIZE};
    const cuuint32_t in_box[4] = {128 / SIZE, (cuuint32_t)A.tile, 2, 1}, out_box[3] = {128 / SIZE, (cuuint32_t)A.box_rows, 1};
    return small_map(&m.gate, type, A.w13, 4, in_dims, in_strides, in_box, true) &&
           small_map(&m.down, type, A.w2, 3, out_dims, out_strides, out_box, true);
  }
}

template <int F, int OCT, typename OutT>
int launch_layer(const SmallArgs& A, cudaStream_t st) {
  const size_t smem = front_bytes(F, OCT) + Tables::bytes(A.T, A.E, A.K) + 1024;
  cudaError_t e = cudaFuncSetAttribute(moe_small_layer<F, OCT, OutT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  int dev = 0, sms = 0;
  if (e == cudaSuccess) e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e == cudaSuccess) {
    SmallArgs args = A;
    SmallMaps maps = {};
    if (!small_maps<F>(args, sms, maps)) return MQ_ERR_DRIVER_ENTRY;
    void* argv[] = {&args, &maps};
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
