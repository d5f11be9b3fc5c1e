// The whole MoE layer for up to 16 tokens in two launches: router, top-k, gate/up + SwiGLU, down, weighted sum and
// residual (mini_qwen/model/layers/moe.py:49-68 and model/qwen3_moe.py:63-66 of the reference), on bf16 or fp16 experts,
// on int4 ones (W4A16) or on int8 ones (W8A8).
//
//   logits[t, e] = x[t] . router[e] (+ bias[e]);  p = softmax(logits);  the top_k largest logits, equal ones by ascending id
//   h[t, k] = silu(x[t] . gate[e]) * (x[t] . up[e])
//   out[t] = round(sum_k weight[t, k] * (h[t, k] . down[e]) + residual[t])
//
// Everything between the inputs and the one rounding at the end is held in fp32: the tensor cores' fp32 sums, and h as the sum
// of three bf16 numbers of eight bits each, which is the fp32 number itself.  (With two of them up to 2^-17 of h was lost, and a
// few in a thousand bf16 results came out a step off; the third costs 0.5 us at one token, 2 us at 16, 6 with int4 experts.)
// fp16 experts: two tf32 numbers, 2^-20 at most, and nothing is left to gain: the results of two numbers rounded to nearest,
// 2^-22, miss their step as often (1 in 400; with fp32 throughout 1 in 500).  W8A8: x and h are quantised per token (int8.cuh),
// the sums are int32.
//
// What bounds it is reading the weights of the experts that are hit; a chain of four to eight dependent launches spends more
// than that on latencies.  So:
//   * launch 1, a CTA per expert: logits.  Spare CTAs quantise the rows (W8A8) and clear the counters of launch 2;
//   * launch 2, one CTA per SM, all resident (a cooperative launch): every CTA selects the experts for itself; the gate/up
//     rows of all experts hit are dealt out evenly, to the row, so that no CTA has more than its share of bytes; one barrier
//     over the grid; then each CTA takes a few output columns of ALL experts hit, so the sum over experts stays inside the
//     CTA: no atomics, no second pass, the same bits every time;
//   * the weights come by tensor-map copies, issued by two warps, through a ring of 128 to 192 KB that runs on through the
//     barrier, so that the first weights of the down projection arrive under it.  Eight warps multiply: a lane's 16-byte
//     pieces are, in a suitable order of k, the fragments of mma.sync (tokens are its 8 columns), so the tensor cores cost
//     nothing here, and all tokens of an expert cost one pass over its weights.  Four warps finish the tiles of h.
// Time is lost where a warp does one thing after the other: each unit of weights (4 KB) costs it some 1000 cycles of waiting,
// table look-ups and sums, against 1040 in which the SM's share of the memory's bandwidth brings eight.  Hence units of 4 KB
// (with 2 KB and twice the warps the down projection took 66 us for 16 tokens, now 42); x, h, scales and addresses looked up
// a unit ahead; quotients of the scales kept from the barrier on (four divisions a lane in each unit: 22 us); scales that
// come from afar asked for by the copying warps.  Copies alone: 7.0 to 7.5 TB/s.
// Measured, hidden 2048, inter 768, 128 experts, top-8, weights out of L2, both launches in a graph: bf16 experts, 1 token 26 us,
// 8 tokens 86 us, 16 tokens 130 us (765 MB: 5.9 TB/s); int8, 1 token 23 us, 16 tokens 89 us; fp16, 16 tokens 136 us; int4
// (unpacked in registers: bound by instructions), 1 token 23 us, 8 tokens 77 us, 13 tokens 110 us.
// Every wait is bounded; when one runs out, MQ_DEV_WAIT_EXPIRED is set and the output is invalid.
#include "int8.cuh"
#include "tc5.cuh"

namespace mq {
namespace {

using namespace int8;

constexpr int MAX_T = 16, MAX_E = 1024, MAX_K = 32;
constexpr int WARPS = 8;                           // that multiply a stage of the ring
constexpr int FINISH = 4;                          // that finish the tiles of h, in turn
constexpr int COPY = 2;                            // that issue the copies
constexpr int ROUTER_THREADS = 256;
constexpr uint32_t POLL_LIMIT = 1u << 22;          // looks at the barrier: about two seconds

enum Format { F_BF16, F_F16, F_INT8, F_INT4 };

// Who does what, by warps: [0, WARPS) multiply, the first FINISH of [WARPS, MEET) finish, the last COPY copy.  For the down
// projection the warps of [WARPS, MEET) are a second team that takes the stages of the ring in turn with the first: for 16
// tokens on bf16 experts 42 us instead of 52, fp16 51 for 62, int4 and 8 tokens 29 for 31 (its work on a stage, one thing after
// the other, takes longer than the stage's copies).  int4 experts of more than eight tokens need more than the 96 registers of
// a thread that this leaves.  (Both teams at gate and up as well, each finishing its tiles itself: bf16 78 us, 73 so.)
template <int F, int OCT> struct Roles {
  static constexpr int TEAMS = F == F_INT4 && OCT == 2 ? 1 : 2, ALL = TEAMS * WARPS, MEET = TEAMS == 2 ? ALL : WARPS + FINISH;
  static constexpr int THREADS = TEAMS == 2 ? (MEET + COPY) * 32 : MAX_T * 32;             // at least a warp for each token
  static_assert(WARPS + FINISH <= MEET && MEET + COPY <= THREADS / 32 && MAX_T <= THREADS / 32, "a warp for each role");
};

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
  uint32_t group_mul;                              // 2^32 over the 128s in a group, rounded up; 0: one
  unsigned* counter;                               // workspace from here on
  uint32_t* amax;                                  // [T * K] largest |h| of a slot, as bits
  float* logits;                                   // [T, E]
  int8_t* xq;                                      // [T, H]
  int8_t* hq;                                      // [T * K, I]
  float *xs, *hs;                                  // scales: [T], [T * K]
  void* h;                                         // [T * K, 3, I] parts of h, bf16; fp16 experts: [T * K, 2, I], tf32; int8: fp32 [T * K, I]
  int32_t* d_status;
};

// ---- launch 1 -------------------------------------------------------------------------------------------

// Eight values as fp32; `left` of them exist.
template <typename V>
__device__ __forceinline__ void load8(const V* p, bool vec, int64_t left, float (&v)[8]) {
  if (vec && left >= 8) {
    if constexpr (sizeof(V) == 4) {
      const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const uint4 a = *reinterpret_cast<const uint4*>(p);
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float2 f;
        if constexpr (std::is_same<V, __half>::value) f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
        else f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[j]));
        v[2 * j] = f.x;
        v[2 * j + 1] = f.y;
      }
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = j < left ? to_float<V>(p[j]) : 0.0f;
}

// The types are the kernel's, so that nothing branches between the loads of the tokens: they are all under way at a time.
template <int TN, typename X, typename R>          // tokens, rounded up
__global__ void __launch_bounds__(ROUTER_THREADS) moe_small_router(const SmallArgs A, int router_vec) {
  __shared__ float part[ROUTER_THREADS / 32][TN];
  __shared__ uint32_t top[ROUTER_THREADS / 32];
  const X* const x = reinterpret_cast<const X*>(A.x);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if ((int)blockIdx.x >= A.E) {                    // spare CTAs
    const int t = (int)blockIdx.x - A.E;
    if (t == 0) {
      if (tid == 0) *A.counter = 0;
      for (int i = tid; i < A.T * A.K; i += ROUTER_THREADS) A.amax[i] = 0;
    }
    if (A.xq == nullptr) return;
    uint32_t most = 0;
    for (int k = 8 * tid; k < A.H; k += 8 * ROUTER_THREADS) {
      float v[8];
      load8<X>(x + (size_t)t * A.H + k, true, A.H - k, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) most = max(most, abs_bits(v[j]));
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) top[warp] = most;
    __syncthreads();
    most = 0;
    for (int i = 0; i < ROUTER_THREADS / 32; ++i) most = max(most, top[i]);
    const RowScale r = row_scale(most);
    if (tid == 0) A.xs[t] = r.scale;
    for (int k = 8 * tid; k < A.H; k += 8 * ROUTER_THREADS) {
      float v[8];
      load8<X>(x + (size_t)t * A.H + k, true, A.H - k, v);
      uint32_t w[2];
      quantize<8>(v, r, w);
      *reinterpret_cast<uint2*>(A.xq + (size_t)t * A.H + k) = make_uint2(w[0], w[1]);
    }
    return;
  }
  const int e = (int)blockIdx.x;
  float acc[TN];
#pragma unroll
  for (int t = 0; t < TN; ++t) acc[t] = 0.0f;
  for (int k = 8 * tid; k < A.H; k += 8 * ROUTER_THREADS) {
    float w[8];
    load8<R>(reinterpret_cast<const R*>(A.router) + (size_t)e * A.H + k, router_vec != 0, A.H - k, w);
#pragma unroll
    for (int t = 0; t < TN; ++t) {                 // tokens that are not there: the last one again
      float v[8];
      load8<X>(x + (size_t)min(t, A.T - 1) * A.H + k, true, 8, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[t] = fmaf(v[j], w[j], acc[t]);
    }
  }
  // the lanes' sums: half of the tokens go to the other half of the lanes at each step, then what is left of the lanes
  int t = 0;
#pragma unroll
  for (int n = TN, o = 16; o > 0; o >>= 1) {
    if (n > 1) {
      n /= 2;
      const bool upper = (lane & o) != 0;
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const float keep = upper ? acc[n + i] : acc[i], give = upper ? acc[i] : acc[n + i];
        acc[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
      }
      t += upper ? n : 0;
    } else {
      acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], o);
    }
  }
  if ((lane & (32 / TN - 1)) == 0) part[warp][t] = acc[0];
  __syncthreads();
  if (tid < TN && tid < A.T) {
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < ROUTER_THREADS / 32; ++i) v += part[i][tid];
    if (A.bias != nullptr) v += A.bias[e];
    A.logits[tid * A.E + e] = v;
  }
}

// ---- launch 2 -------------------------------------------------------------------------------------------

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
               "{%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
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
  uint32_t* info;      // [hits] where the expert's slots begin, and how many there are << 16: they are columns 0, 1, ... of its products
  uint16_t* pos;       // [E] its place among the experts hit
  uint16_t* hit;       // [hits] the expert
  uint16_t* slot;      // [T * K] token * MAX_K + which of its experts it is
  uint16_t* ids;       // [T, MAX_K] the tokens' experts
  float* w;            // [T, MAX_K] and their weights
  __host__ __device__ static constexpr size_t bytes(int T, int E, int K) {
    const size_t hits = (size_t)(E < T * K ? E : T * K);
    return hits * 6 + (size_t)E * 6 + (size_t)T * MAX_K * 6 + (size_t)T * K * 2 + 16;
  }
  __device__ Tables(uint8_t* p, int T, int E, int K) {
    const int hits = min(E, T * K);
    w = reinterpret_cast<float*>(p);
    mask = reinterpret_cast<uint32_t*>(w + T * MAX_K);
    info = mask + E;
    slot = reinterpret_cast<uint16_t*>(info + hits);
    ids = slot + T * K;
    pos = ids + T * MAX_K;
    hit = pos + E;
  }
  __device__ __forceinline__ int count(int place) const { return (int)(info[place] >> 16); }
  __device__ __forceinline__ int at(int place, int n) const { return slot[(info[place] & 0xffffu) + n]; }
};

// A unit is what a warp multiplies at a time, in two halves: 256 bytes of k of 16 weight rows (gate and up: 8 of either), or
// int4 words: 256 k of 16 columns (gate and up: of either).  A stage of the ring holds a unit for each warp.
template <int F> struct Fmt {
  static constexpr bool W4 = F == F_INT4;
  static constexpr int SIZE = F == F_INT8 ? 1 : 2;
  static constexpr int UNIT_K = W4 ? 256 : 256 / SIZE, HALF_K = UNIT_K / 2;
  static constexpr int MT = W4 ? 2 : 1;            // accumulator tiles: int4 gate and up apart, else 8 + 8 rows in one
};
constexpr int UNIT = 4096, STAGE = WARPS * UNIT;
// Stages of the ring.  Behind it the partial sums, a buffer for each warp that takes them, and the tables.  The stages are a
// multiple of the teams, so that a place in the ring is the same team's every time and the team has itself seen the place's last
// fill.  (With five stages it could come to a place one fill early, where the parity of the older fill let it through.)
__host__ __device__ constexpr int ring_stages(int f, int octets) { return f == F_INT4 || octets == 2 ? 4 : 6; }
__host__ __device__ constexpr size_t part_bytes(int f, int octets) { return (size_t)WARPS * 512 * (f == F_INT4 ? 2 : 1) * octets; }
__host__ __device__ constexpr size_t front_bytes(int f, int octets) {
  return (size_t)ring_stages(f, octets) * STAGE + FINISH * part_bytes(f, octets);
}

// A barrier over the grid, by one thread of each CTA between barriers of the CTA: its release and acquire stand for all of them.
__device__ __forceinline__ bool grid_meet(unsigned* counter, unsigned target) {
  asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(counter) : "memory");
  uint32_t seen = 0, looks = 0;
  do {
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(seen) : "l"(counter) : "memory");
  } while (seen < target && ++looks < POLL_LIMIT);
  return seen >= target;
}
// For what is read once, from afar, some stages later.
__device__ __forceinline__ void prefetch(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

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

// Four accumulators as bits, and such bits added.
__device__ __forceinline__ int4 raw4(const float (&v)[4]) {
  return make_int4(__float_as_int(v[0]), __float_as_int(v[1]), __float_as_int(v[2]), __float_as_int(v[3]));
}
__device__ __forceinline__ int4 raw4(const int (&v)[4]) { return make_int4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void add4(float (&s)[4], int4 v) {
  s[0] += __int_as_float(v.x); s[1] += __int_as_float(v.y); s[2] += __int_as_float(v.z); s[3] += __int_as_float(v.w);
}
__device__ __forceinline__ void add4(int (&s)[4], int4 v) { s[0] += v.x; s[1] += v.y; s[2] += v.z; s[3] += v.w; }

struct SmallMaps { CUtensorMap gate, up, down; };  // dense and int8: gate and up rows in one

template <int F, int OCT, typename OutT>
__global__ void __launch_bounds__(Roles<F, OCT>::THREADS, 1) moe_small_layer(const SmallArgs A, const __grid_constant__ SmallMaps maps) {
  using namespace tc5;
  using Acc = typename std::conditional<F == F_INT8, int, float>::type;
  constexpr int SIZE = Fmt<F>::SIZE, UNIT_K = Fmt<F>::UNIT_K, HALF_K = Fmt<F>::HALF_K, MT = Fmt<F>::MT;
  constexpr bool W4 = F == F_INT4;
  constexpr int TEAMS = Roles<F, OCT>::TEAMS, ALL = Roles<F, OCT>::ALL, MEET = Roles<F, OCT>::MEET, THREADS = Roles<F, OCT>::THREADS;
  constexpr int STAGES = ring_stages(F, OCT);
  static_assert(STAGES % TEAMS == 0, "a place in the ring belongs to one team");
  extern __shared__ uint8_t small_smem_raw[];
  uint8_t* const small_smem = small_smem_raw + ((1024u - (smem_addr(small_smem_raw) & 1023u)) & 1023u);   // the copies' swizzle
  uint8_t* part = small_smem + STAGES * STAGE;
  const Tables tab(small_smem + front_bytes(F, OCT), A.T, A.E, A.K);
  __shared__ int s_hits, s_ok, s_abort;
  __shared__ __align__(8) uint64_t s_bars[2 * STAGES + 2 * FINISH];
  const uint32_t bars = smem_addr(s_bars), ring = smem_addr(small_smem);
  auto full = [&](int i) { return bars + 8u * i; };
  auto empty = [&](int i) { return bars + 8u * (STAGES + i); };
  auto pfull = [&](int i) { return bars + 8u * (2 * STAGES + i); };        // partial sums written
  auto pfree = [&](int i) { return bars + 8u * (2 * STAGES + FINISH + i); };    // and read
  const int tid = threadIdx.x, lane = tid & 31, warp = (int)uniform(tid >> 5), g = lane >> 2, q4 = lane & 3;
  const int T = A.T, H = A.H, I = A.I, E = A.E, K = A.K, G = (int)gridDim.x, cta = (int)blockIdx.x;
  volatile int* abort_flag = &s_abort;

  // ------------------------------------------------------------------ who goes where
  if (tid == THREADS - 1) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(full(i), COPY);
      mbar_init(empty(i), WARPS);
    }
    for (int i = 0; i < FINISH; ++i) {
      mbar_init(pfull(i), WARPS);
      mbar_init(pfree(i), 1);
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
    int n = 0, slots = 0;
    for (int e0 = 0; e0 < E; e0 += 32) {
      const uint32_t m = e0 + lane < E ? tab.mask[e0 + lane] : 0u;
      const unsigned any = __ballot_sync(0xffffffffu, m != 0);
      if (any == 0) continue;
      int upto = __popc(m);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int below = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += below;
      }
      const int at = n + __popc(any & ((1u << lane) - 1u));
      if (m != 0) {
        tab.hit[at] = (uint16_t)(e0 + lane);
        tab.pos[e0 + lane] = (uint16_t)at;
        tab.info[at] = (uint32_t)(slots + upto - __popc(m)) | (uint32_t)__popc(m) << 16;
      }
      n += __popc(any);
      slots += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane == 0) s_hits = n;
  }
  __syncthreads();
  if (tid < T * MAX_K && lane < K) {
    const int e = tab.ids[tid];
    tab.slot[(tab.info[tab.pos[e]] & 0xffffu) + __popc(tab.mask[e] & ((1u << warp) - 1u))] = (uint16_t)tid;
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
  const int units = (H + UNIT_K - 1) / UNIT_K, units2 = (I + UNIT_K - 1) / UNIT_K;
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
  // int4: quantisation groups along k, and the one that the n-th 128 of k lie in
  const int groups = W4 ? H / A.group : 0, groups2 = W4 ? I / A.group : 0;
  auto group_of = [&](int n) { return A.group_mul != 0 ? (int)__umulhi((uint32_t)n, A.group_mul) : n; };
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

  if (warp >= MEET + COPY) return;

  if (warp >= MEET) {
    // ------------------------------------------------------------------ copies: first gate and up, then down
    // Weights only, so they run on through the barrier over the grid.  The warps take every other unit (int4: gate or up); one
    // elected lane issues, from uniform registers.
    const bool leader = elect_one();
    const int copier = warp - MEET;
    int stage = 0, filled = 0;
    uint32_t phase = 0;
    bool ok = true;
    auto next_stage = [&] {
      __syncwarp();
      ++filled;
      if (++stage == STAGES) { stage = 0; phase ^= 1u; }
    };
    for (int round = 0; round < rounds && ok; ++round) {
      for (int pass = 0; pass < passes; ++pass) {
        ok = mbar_wait_warp(empty(stage), phase ^ 1u, abort_flag, A.d_status);
        if (!ok) break;
        const int u0 = pass * ksplit, n = min(ksplit, units - u0), live = min(at_once, tiles - round * at_once);
        const uint32_t dst = ring + stage * STAGE, bar = full(stage);
        if (leader) mbar_expect_tx(bar, W4 ? live * A.box_rows * 64 : (live * n + 1 - copier) / 2 * 4 * TW * 128);
        int turn = copier;
        Walk c = walk;
        for (int i = 0; i < live; ++i) {
          const int e = (int)uniform(tab.hit[c.place]), col = (int)uniform(c.pos - (c.end - I));
          const uint32_t at = dst + i * ksplit * UNIT;
          if (W4) {
            if (leader) copy_box(at + copier * ksplit * (UNIT / 2), copier == 0 ? &maps.gate : &maps.up, bar, col, u0 * 32, e);
            if (pass == 0) {                       // the tile's scales and zero points
              for (int j = lane; j < groups; j += 32) {
                const size_t row = (size_t)e * groups + j;
                prefetch(A.sc[copier] + row * I + col);
                prefetch(A.qz[copier] + row * (I / 8) + (col >> 3));
              }
            }
          } else {
            for (int u = 0; u < n; ++u) {
              if (leader && (turn++ & 1) == 0) {
                copy_box(at + u * UNIT, &maps.gate, bar, (u0 + u) * UNIT_K, col, 0, e);
                copy_box(at + u * UNIT + UNIT / 2, &maps.gate, bar, (u0 + u) * UNIT_K + HALF_K, col, 0, e);
              }
            }
            if (F == F_INT8 && pass == 0 && copier == 1 && lane < 4) prefetch(A.s13 + ((size_t)e * 2 + (lane & 1)) * I + min(col + 7 * (lane >> 1), I - 1));
          }
          next_tile(c);
        }
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
        if (leader) mbar_expect_tx(bar, (live + 1 - copier) / 2 * (W4 ? 2048 : A.box_rows * 256));
        for (int i = 0; i < live; ++i) {
          const bool turn = (i & 1) == copier;
          const int e = turn ? (int)uniform(tab.hit[place]) : 0;
          if (leader && turn) {
            if (W4) {
              copy_box(dst + i * UNIT, &maps.down, bar, row0, u * 32, e);
            } else {
              copy_box(dst + i * UNIT, &maps.down, bar, u * UNIT_K, row0, e);
              copy_box(dst + i * UNIT + UNIT / 2, &maps.down, bar, u * UNIT_K + HALF_K, row0, e);
            }
          }
          if (W4 && turn && lane < 4) {            // the unit's scales and zero points
            const size_t row = (size_t)e * groups2 + min(group_of(2 * u + (lane & 1)), groups2 - 1);
            if (lane < 2) prefetch(A.sc[2] + row * H + row0);
            else prefetch(A.qz[2] + row * (H / 8) + (row0 >> 3));
          }
          if (F == F_INT8 && turn && lane < 2) prefetch(A.s2 + (size_t)e * H + min(row0 + 15 * lane, out_hi - 1));
          if (++u == units2) { u = 0; ++place; }
        }
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
    if (ok && lane == 0) mbar_arrive(empty(stage));
    if (++stage == STAGES) { stage = 0; phase ^= 1u; }
  };

  if (warp < WARPS) {
    // ------------------------------------------------------------------ gate and up projections
    // What a unit needs beside its weights is loaded a unit ahead, into the registers of the unit just done: x of the lane's
    // token (column g of the expert, o * 8 + g of its second octet); int4: the scales and zero points of its two groups.  Where
    // they lie is worked out a tile ahead: a warp's own instructions, one after the other, are what takes the time here.
    const int kw = warp % ksplit, tg = warp / ksplit;
    skip_tiles(walk, tg);
    const uint8_t* const rows = F == F_INT8 ? reinterpret_cast<const uint8_t*>(A.xq) : reinterpret_cast<const uint8_t*>(A.x);
    constexpr int XS = W4 ? 8 : 4, XH = XS / 2;    // 16-byte pieces of a unit, of a half
    const int x_lane = W4 ? 16 * q4 : 32 * q4, x_row = H * SIZE;
    auto x_offset = [](int s) { return W4 ? 64 * s : (s >> 1) * 128 + (s & 1) * 16; };
    auto row_at = [&](int place, int n) -> const uint8_t* {
      return n < tab.count(place) ? rows + (size_t)(tab.at(place, n) >> 5) * x_row + x_lane : nullptr;
    };
    auto load_x = [&](uint4 (&x)[XS], const uint8_t* row, int u) {
      const int at = u * (W4 ? 512 : 256), left = row != nullptr ? x_row - x_lane - at : 0;
#pragma unroll
      for (int s = 0; s < XS; ++s)
        x[s] = x_offset(s) < left ? __ldg(reinterpret_cast<const uint4*>(row + at + x_offset(s))) : make_uint4(0u, 0u, 0u, 0u);
    };
    struct Ahead {
      Walk w;
      int pass;
      const uint8_t* row;                          // of x
      size_t scale, zero;                          // int4: of the tile's columns in the first group
    } ahead{walk, 0, nullptr, 0, 0};
    auto look_ahead = [&] {                        // a new tile
      if (ahead.w.pos >= hi) return;
      ahead.row = row_at(ahead.w.place, g);
      if constexpr (W4) {
        const size_t n = (size_t)(ahead.w.pos - (ahead.w.end - I)) + 2 * g, first = (size_t)tab.hit[ahead.w.place] * groups;
        ahead.scale = first * I + n;
        ahead.zero = first * (I / 8) + (n >> 3);
      }
    };
    uint4 x[XS];
    uint32_t scale[2][2] = {}, zero[2][2] = {};    // [gate or up][half]
    auto load_ahead = [&] {
      const int u = ahead.pass * ksplit + kw;
      if (ahead.w.pos < hi && u < units) {
        load_x(x, ahead.row, u);
        if constexpr (W4) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int r = min(group_of(2 * u + half), groups - 1);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              scale[j][half] = __ldg(reinterpret_cast<const uint32_t*>(A.sc[j] + ahead.scale + (size_t)r * I));
              zero[j][half] = (uint32_t)__ldg(A.qz[j] + ahead.zero + (size_t)r * (I / 8));
            }
          }
        }
      }
      if (++ahead.pass == passes) {
        ahead.pass = 0;
        skip_tiles(ahead.w, at_once);
        look_ahead();
      }
    };
    auto multiply_dense = [&](Acc (&to)[2][4], const uint4 (&w)[8], const uint4 (&b)[XS]) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {                // two chains of sums
        Acc (&c)[4] = to[i >> 1];
        const uint4 r = w[2 * i], r8 = w[2 * i + 1];
        if constexpr (F == F_INT8) {
          mma_s8(c, r.x, r8.x, r.y, r8.y, b[i].x, b[i].y);
          mma_s8(c, r.z, r8.z, r.w, r8.w, b[i].z, b[i].w);
        } else if constexpr (F == F_F16) {
          mma_f16(c, r.x, r8.x, r.y, r8.y, b[i].x, b[i].y);
          mma_f16(c, r.z, r8.z, r.w, r8.w, b[i].z, b[i].w);
        } else {
          mma_bf16(c, r.x, r8.x, r.y, r8.y, b[i].x, b[i].y);
          mma_bf16(c, r.z, r8.z, r.w, r8.w, b[i].z, b[i].w);
        }
      }
    };
    auto multiply_int4 = [&](float (&to)[2][4], const uint8_t* unit, const uint4 (&b)[XS], uint32_t shift) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {       // a half lies inside a quantisation group
        float grp[2][4] = {};
        const __nv_bfloat162 minus[2][2] = {{zero_pair(zero[0][half] >> shift), zero_pair(zero[0][half] >> (shift + 4))},
                                            {zero_pair(zero[1][half] >> shift), zero_pair(zero[1][half] >> (shift + 4))}};
#pragma unroll
        for (int s = 0; s < XH; ++s) {
          const uint4 v = pair_up(b[half * XH + s]);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint2 w = *reinterpret_cast<const uint2*>(unit + j * ksplit * (UNIT / 2) + (16 * half + 4 * s + q4) * 64 + 8 * g);
            uint32_t v0[4], v1[4];
            unpack_int4(w.x, minus[j][0], v0);
            unpack_int4(w.y, minus[j][1], v1);
            mma_bf16(grp[j], v0[0], v1[0], v0[1], v1[1], v.x, v.y);
            mma_bf16(grp[j], v0[2], v1[2], v0[3], v1[3], v.z, v.w);
          }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float2 sc = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&scale[j][half]));
#pragma unroll
          for (int i = 0; i < 4; ++i) to[j][i] = fmaf(grp[j][i], i < 2 ? sc.x : sc.y, to[j][i]);
        }
      }
    };
    look_ahead();
    load_ahead();
    for (int round = 0; round < rounds; ++round) {
      Acc acc[OCT][2][4] = {};                     // int4: gate, up; else two sums of the same
      const bool mine = walk.pos < hi;
      const bool many = OCT == 2 && mine && tab.count(walk.place) > 8;
      const uint32_t shift = W4 ? 4u * ((walk.pos - (walk.end - I) + 2 * g) & 7) : 0u;
      for (int pass = 0; pass < passes; ++pass) {
        const int u = pass * ksplit + kw;
        const bool live = mine && u < units;
        if (ok) ok = mbar_wait_warp(full(stage), phase, abort_flag, A.d_status);
        if constexpr (W4) {
          const uint8_t* unit = small_smem + stage * STAGE + tg * ksplit * UNIT + kw * (UNIT / 2);
          if (live) {
            multiply_int4(acc[0], unit, x, shift);
            if (many) {
              load_x(x, row_at(walk.place, 8 + g), u);
              multiply_int4(acc[OCT - 1], unit, x, shift);
            }
          }
          release();
        } else {
          const uint8_t* unit = small_smem + stage * STAGE + warp * UNIT;
          uint4 w[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            w[2 * i] = piece(unit + (i >> 1) * (UNIT / 2), g, i & 1);
            w[2 * i + 1] = piece(unit + (i >> 1) * (UNIT / 2), TW + g, i & 1);
          }
          if (live) multiply_dense(acc[0], w, x);
          release();
          if (live && many) {
            load_x(x, row_at(walk.place, 8 + g), u);
            multiply_dense(acc[OCT - 1], w, x);
          }
        }
        load_ahead();
      }
      const int buf = round % FINISH;
      if (ok) ok = mbar_wait_warp(pfree(buf), ((round / FINISH) & 1) ^ 1u, abort_flag, A.d_status);
#pragma unroll
      for (int o = 0; o < OCT; ++o) {
        if (o == 1 && !many) break;
        int4* to = reinterpret_cast<int4*>(part + buf * part_bytes(F, OCT)) + (warp * OCT + o) * MT * 32 + lane;
        if constexpr (W4) {
          to[0] = raw4(acc[o][0]);
          to[32] = raw4(acc[o][1]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[o][0][i] += acc[o][1][i];
          to[0] = raw4(acc[o][0]);
        }
      }
      __syncwarp();
      if (ok && lane == 0) mbar_arrive(pfull(buf));
      skip_tiles(walk, at_once);
    }
  } else if (warp < WARPS + FINISH) {
    // ------------------------------------------------------------------ sums over the warps, SwiGLU
    // The warps take the rounds in turn: a lane a fragment position of a tile, its sums over the warps in order.
    const int buf = warp - WARPS;
    skip_tiles(walk, buf * at_once);
    for (int round = buf; round < rounds; round += FINISH) {
      if (ok) ok = mbar_wait_warp(pfull(buf), (round / FINISH) & 1, abort_flag, A.d_status);
      const int live_tiles = min(at_once, tiles - round * at_once);
      for (int slot = 0; slot < live_tiles; ++slot) {
        const int place = walk.place, col0 = walk.pos - (walk.end - I), cols = width(walk);
        next_tile(walk);
        const size_t e = tab.hit[place];
#pragma unroll
        for (int o = 0; o < OCT; ++o) {
          const int live = tab.count(place) - 8 * o;                  // columns of this octet
          if (live <= 0) continue;
          Acc sum[MT][4] = {};
#pragma unroll 8
          for (int w = 0; w < ksplit; ++w)
#pragma unroll
            for (int j = 0; j < MT; ++j) {
              const int4 raw = *reinterpret_cast<const int4*>(part + buf * part_bytes(F, OCT) +
                                                              ((((slot * ksplit + w) * OCT + o) * MT + j) * 32 + lane) * 16);
              add4(sum[j], raw);
            }
#pragma unroll
          for (int i = 0; i < (W4 ? 4 : 2); ++i) {
            const int n = 2 * q4 + (i & 1), col = W4 ? 2 * g + (i >> 1) : g;
            float v = 0.0f;
            const int code = n < live ? tab.at(place, 8 * o + n) : 0;
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
              if (F == F_BF16 || W4) {             // a bf16 number is the upper 16 bits of an fp32 one; the differences are exact
                uint16_t* h = reinterpret_cast<uint16_t*>(A.h) + row * 3 * I + col0 + col;
                const uint32_t high = __float_as_uint(v) & 0xffff0000u;
                const float rest = isinf(v) ? 0.0f : v - __uint_as_float(high);
                const uint32_t middle = __float_as_uint(rest) & 0xffff0000u;
                h[0] = (uint16_t)(high >> 16);
                h[I] = (uint16_t)(middle >> 16);
                h[2 * I] = (uint16_t)(__float_as_uint(rest - __uint_as_float(middle)) >> 16);
              } else if (F == F_F16) {             // a tf32 number is the upper 19 bits of an fp32 one
                float* h = reinterpret_cast<float*>(A.h) + row * 2 * I + col0 + col;
                const float high = __uint_as_float(__float_as_uint(v) & 0xffffe000u);
                h[0] = high;
                h[I] = isinf(v) ? 0.0f : v - high;
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
      if (ok && lane == 0) mbar_arrive(pfree(buf));
      skip_tiles(walk, (FINISH - 1) * at_once);
    }
  }

  // ------------------------------------------------------------------ every h is there
  warps_meet<1, MEET>();
  if (tid == 0) s_ok = grid_meet(A.counter, (unsigned)G);
  warps_meet<1, MEET>();
  if (F == F_INT8 && s_ok != 0) {                  // h to int8, 128 elements a warp over the whole grid, and a second barrier
    const int pieces = (I + 127) / 128;
    for (int i = warp * G + cta; i < T * K * pieces; i += G * MEET) {
      const int row = i / pieces, k = (i - row * pieces) * 128 + 4 * lane;
      if (k < I) {
        const RowScale r = row_scale(__ldcg(A.amax + row));
        const float4 v = __ldcg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(A.h) + (size_t)row * I + k));
        const float f[4] = {v.x, v.y, v.z, v.w};
        uint32_t q[1];
        quantize<4>(f, r, q);
        *reinterpret_cast<uint32_t*>(A.hq + (size_t)row * I + k) = q[0];
        if (k == 0) A.hs[row] = r.scale;
      }
    }
    warps_meet<1, MEET>();
    if (tid == 0) s_ok = grid_meet(A.counter, 2u * (unsigned)G);
    warps_meet<1, MEET>();
  }
  if (warp >= ALL) return;
  if (s_ok == 0) {
    if (tid == 0 && A.d_status != nullptr) atomicOr(A.d_status, (int)MQ_DEV_WAIT_EXPIRED);
    return;
  }

  // ------------------------------------------------------------------ down projection and weighted sum
  // A warp's sums of a tile, [tokens, 16 columns], are its own piece of shared memory, to which a unit's columns are added
  // with their tokens' weights.  A token that did not choose the expert takes nothing from it, whatever its weights hold.
  float* mine = reinterpret_cast<float*>(part) + warp * (128 * OCT);
  // The eight columns of a product are the parts of h of some tokens, one part after the other: three of two tokens, and two
  // columns without (fp16: two of four tokens; int8: eight tokens).
  constexpr int PARTS = F == F_INT8 ? 1 : F == F_F16 ? 2 : 3;
  constexpr int CHUNK = F == F_INT8 ? 8 : F == F_F16 ? 4 : 2;              // tokens of a product
  constexpr int HS = W4 ? 8 : 4, HH = HS / 2, HV = F == F_F16 ? 2 : 1;     // steps of a unit, of a half; 16-byte pieces of a step
  constexpr int H_ITEM = F == F_INT8 ? 1 : F == F_F16 ? 4 : 2;
  const int h_lane = (W4 ? 8 : 32 / SIZE) * q4, n_lane = g % CHUNK, my_part = g / CHUNK;
  auto h_offset = [](int s) { return W4 ? 32 * s : (s >> 1) * HALF_K + (s & 1) * (16 / SIZE); };
  const uint8_t* const h_rows = F == F_INT8 ? reinterpret_cast<const uint8_t*>(A.hq)
                                            : reinterpret_cast<const uint8_t*>(A.h) + (size_t)min(my_part, PARTS - 1) * I * H_ITEM;
  uint4 h[HS][HV];
  uint32_t scale[2] = {}, zero[2] = {};                                    // int4: of the halves
  float col_scale[2] = {}, row_scale[2] = {};                              // int8: of two columns, of two tokens
  // h of a unit's tokens from `chunk` on, and the scales; the loads are a unit ahead
  auto load_h = [&](int row0, int place, int u, int chunk) {
    const int count = tab.count(place), n = chunk * CHUNK + n_lane;
    const bool live = n < count && my_part < PARTS;
    const int row = live ? row_of(tab.at(place, n)) : 0, k0 = u * UNIT_K + h_lane, left = live ? I - k0 : 0;
    const uint8_t* src = h_rows + ((size_t)row * PARTS * I + k0) * H_ITEM;
#pragma unroll
    for (int s = 0; s < HS; ++s)
#pragma unroll
      for (int p = 0; p < HV; ++p)
        h[s][p] = h_offset(s) < left ? __ldcg(reinterpret_cast<const uint4*>(src + h_offset(s) * H_ITEM + 16 * p)) : make_uint4(0u, 0u, 0u, 0u);
    if constexpr (W4) {
      const size_t c = (size_t)row0 + 2 * g;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const size_t r = (size_t)tab.hit[place] * groups2 + min(group_of(2 * u + half), groups2 - 1);
        scale[half] = __ldg(reinterpret_cast<const uint32_t*>(A.sc[2] + r * H + c));
        zero[half] = (uint32_t)__ldg(A.qz[2] + r * (H / 8) + (c >> 3));
      }
    }
    if constexpr (F == F_INT8) {
      const float* s2 = A.s2 + (size_t)tab.hit[place] * H;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int c = row0 + g + 8 * i, t = chunk * CHUNK + 2 * q4 + i;
        col_scale[i] = c < out_hi ? __ldg(s2 + c) : 0.0f;
        row_scale[i] = t < count ? __ldcg(A.hs + row_of(tab.at(place, t))) : 0.0f;
      }
    }
  };
  // what the unit's sums of two tokens are multiplied by and where they go; none: -1
  struct Target { int to[2]; float weight[2]; };
  auto targets = [&](int place, int chunk) {
    Target t;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int n = 2 * q4 + i, at = chunk * CHUNK + n;
      const bool live = n < CHUNK && at < tab.count(place);
      const int slot = live ? tab.at(place, at) : 0;
      t.weight[i] = tab.w[slot];
      t.to[i] = live ? (slot >> 5) * 16 + (W4 ? 2 * g : g) : -1;
    }
    return t;
  };
  auto add = [&](const Acc (&acc)[4], const Target& t, const float (&of_row)[2], const float (&of_col)[2]) {
    float v[4], old[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = CHUNK == 2 && q4 == PARTS ? 0.0f : (float)acc[i];             // the parts' products together
      if (CHUNK == 2) v[i] += __shfl_xor_sync(0xffffffffu, v[i], 1);
      if (CHUNK <= 4) v[i] += __shfl_xor_sync(0xffffffffu, v[i], 2);
      if (t.to[i & 1] >= 0) old[i] = mine[t.to[i & 1] + (W4 ? 1 : 8) * (i >> 1)];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (F == F_INT8) v[i] = v[i] * of_row[i & 1] * of_col[i >> 1];
      if (t.to[i & 1] >= 0) mine[t.to[i & 1] + (W4 ? 1 : 8) * (i >> 1)] = fmaf(v[i], t.weight[i & 1], old[i]);
    }
    __syncwarp();
  };
  auto multiply_dense = [&](Acc (&sum)[4], const uint4 (&w)[8]) {
    Acc acc[2][4] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      Acc (&c)[4] = acc[i >> 1];
      const uint4 r4 = w[2 * i], r84 = w[2 * i + 1], b = h[i][0];
      if constexpr (F == F_INT8) {
        mma_s8(c, r4.x, r84.x, r4.y, r84.y, b.x, b.y);
        mma_s8(c, r4.z, r84.z, r4.w, r84.w, b.z, b.w);
      } else {
        mma_bf16(c, r4.x, r84.x, r4.y, r84.y, b.x, b.y);
        mma_bf16(c, r4.z, r84.z, r4.w, r84.w, b.z, b.w);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] = acc[0][i] + acc[1][i];
  };
  // fp16 fits into tf32.  Its h takes twice the registers, so the weights are loaded as they are needed.
  auto multiply_f16 = [&](Acc (&sum)[4], const uint8_t* unit) {
    float acc[2][4] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 r4 = piece(unit + (i >> 1) * (UNIT / 2), g, i & 1), r84 = piece(unit + (i >> 1) * (UNIT / 2), 8 + g, i & 1);
      const uint32_t r[4] = {r4.x, r4.y, r4.z, r4.w}, r8[4] = {r84.x, r84.y, r84.z, r84.w};
      const uint4 b = h[i][0], b1 = h[i][HV - 1];
      const uint32_t v[8] = {b.x, b.y, b.z, b.w, b1.x, b1.y, b1.z, b1.w};
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&r[p]));
        const float2 a8 = __half22float2(*reinterpret_cast<const __half2*>(&r8[p]));
        mma_tf32(acc[i & 1], __float_as_uint(a.x), __float_as_uint(a8.x), __float_as_uint(a.y), __float_as_uint(a8.y), v[2 * p], v[2 * p + 1]);
      }
      asm volatile("" ::: "memory");
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] = acc[0][i] + acc[1][i];
  };
  auto multiply_int4 = [&](float (&sum)[4], const uint8_t* unit, uint32_t shift) {
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] = 0.0f;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float grp[2][4] = {};
      const __nv_bfloat162 minus0 = zero_pair(zero[half] >> shift), minus1 = zero_pair(zero[half] >> (shift + 4));
#pragma unroll
      for (int s = 0; s < HH; ++s) {
        const uint4 v = pair_up(h[half * HH + s][0]);
        const uint2 w = *reinterpret_cast<const uint2*>(unit + (16 * half + 4 * s + q4) * 64 + 8 * g);
        uint32_t v0[4], v1[4];
        unpack_int4(w.x, minus0, v0);
        unpack_int4(w.y, minus1, v1);
        mma_bf16(grp[0], v0[0], v1[0], v0[1], v1[1], v.x, v.y);
        mma_bf16(grp[1], v0[2], v1[2], v0[3], v1[3], v.z, v.w);
      }
      const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&scale[half]));
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] = fmaf(grp[0][i] + grp[1][i], i < 2 ? f.x : f.y, sum[i]);
    }
  };
  const int team = warp / WARPS, seat = warp % WARPS;
  const int step_place = WARPS / units2, step_u = WARPS - step_place * units2, turns = (tasks + WARPS - 1) / WARPS;
  const int place0 = seat / units2, u0 = seat - place0 * units2;
  struct At { int row0, turn, place, u; };         // a unit of the warp; there is one only where place < hits
  auto next_unit = [&](At& a) {
    a.place += step_place;
    a.u += step_u;
    if (a.u >= units2) { a.u -= units2; ++a.place; }
    if (++a.turn == turns) {
      a.turn = 0;
      a.row0 += 16;
      a.place = place0;
      a.u = u0;
    }
  };
  At cur{out_lo, 0, place0, u0};
  stage = rounds * passes % STAGES;                // the second team has not counted
  phase = (uint32_t)(rounds * passes / STAGES) & 1u;
  auto skip_stage = [&] {                          // the other team's
    if (++stage == STAGES) { stage = 0; phase ^= 1u; }
    next_unit(cur);
  };
  int turns_left = turns * ((out_hi - out_lo + 15) / 16) - team;           // of this team's next one on
  if (team == 1) skip_stage();
  At ahead = cur;
  Target next = {};
  auto load_ahead = [&] {
    next_unit(ahead);
    if (TEAMS == 2) next_unit(ahead);
    if (ahead.row0 < out_hi && ahead.place < hits) next = targets(ahead.place, 0);
    if (ahead.row0 < out_hi && ahead.place < hits) load_h(ahead.row0, ahead.place, ahead.u, 0);
  };
  if (cur.row0 < out_hi && cur.place < hits) {
    next = targets(cur.place, 0);
    load_h(cur.row0, cur.place, cur.u, 0);
  }
  for (int row0 = out_lo; row0 < out_hi; row0 += 16) {
    for (int i = lane; i < 128 * OCT; i += 32) mine[i] = 0.0f;
    __syncwarp();
    const uint32_t shift = W4 ? 4u * ((row0 + 2 * g) & 7) : 0u;
    for (; turns_left > 0 && cur.row0 == row0; turns_left -= TEAMS) {
      const bool live = cur.place < hits;
      const int chunks = live ? (tab.count(cur.place) + CHUNK - 1) / CHUNK : 0;
      if (ok) ok = mbar_wait_warp(full(stage), phase, abort_flag, A.d_status);
      const uint8_t* unit = small_smem + stage * STAGE + seat * UNIT;
      uint4 w[W4 || F == F_F16 ? 1 : 8];
      if constexpr (!W4 && F != F_F16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[2 * i] = piece(unit + (i >> 1) * (UNIT / 2), g, i & 1);
          w[2 * i + 1] = piece(unit + (i >> 1) * (UNIT / 2), 8 + g, i & 1);
        }
        release();
      }
      for (int chunk = 0; chunk < max(chunks, 1); ++chunk) {               // more than one: loaded as they are needed
        if (chunk > 0) {
          load_h(cur.row0, cur.place, cur.u, chunk);
          next = targets(cur.place, chunk);
        }
        Acc acc[4];
        if (live) {
          if constexpr (W4) multiply_int4(acc, unit, shift);
          else if constexpr (F == F_F16) multiply_f16(acc, unit);
          else multiply_dense(acc, w);
        }
        const float of_row[2] = {row_scale[0], row_scale[1]}, of_col[2] = {col_scale[0], col_scale[1]};
        const Target t = next;
        if (chunk + 1 >= chunks) {
          if (W4 || F == F_F16) release();
          load_ahead();
        }
        if (live) add(acc, t, of_row, of_col);
      }
      next_unit(cur);
      if (TEAMS == 2) skip_stage();
    }
    warps_meet<2, ALL>();
    // the warps' sums, in order, then the one rounding
    if (tid < 128 * OCT) {
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < ALL; ++w) v += reinterpret_cast<const float*>(part)[w * (128 * OCT) + tid];
      const int tok = tid / 16, col = row0 + tid % 16;
      if (tok < T && col < out_hi) {
        const size_t at = (size_t)tok * H + col;
        if (A.residual != nullptr) v += to_float<OutT>(reinterpret_cast<const OutT*>(A.residual)[at]);
        reinterpret_cast<OutT*>(A.out)[at] = from_float<OutT>(v);
      }
    }
    if (row0 + 16 < out_hi) warps_meet<2, ALL>();
  }
}

// ---- host -----------------------------------------------------------------------------------------------

int format_of(const mq_moe_layer& L) {
  if (L.group_size > 0) return F_INT4;
  if (L.int8_experts == 1) return F_INT8;
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
  A.hs = (float*)take(S * 4);
  const bool int8 = format_of(L) == F_INT8;
  A.h = take(S * (size_t)L.inter * (int8 ? 4 : format_of(L) == F_F16 ? 8 : 6));
  A.xq = int8 ? (int8_t*)take((size_t)(T * L.hidden)) : nullptr;
  A.hq = int8 ? (int8_t*)take(S * (size_t)L.inter) : nullptr;
  return used;
}

bool small_layer_ok(const mq_moe_layer* L) {
  return L != nullptr && L->hidden > 0 && L->inter > 0 && L->experts > 0 && L->top_k > 0 && L->group_size >= 0 &&
         valid_dtype(L->dtype) && valid_dtype(L->router_dtype) && !(L->int8_experts == 1 && L->group_size > 0);
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
    int ksplit = WARPS;                            // as the kernel does
    while (ksplit / 2 >= (A.H + Fmt<F>::UNIT_K - 1) / Fmt<F>::UNIT_K) ksplit >>= 1;
    A.box_rows = 32 * ksplit;
    A.group_mul = A.group == 128 ? 0u : (uint32_t)((((uint64_t)1 << 32) + A.group / 128 - 1) / (A.group / 128));
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

template <typename X, typename R>
void launch_router_of(const SmallArgs& A, unsigned grid, int vec, cudaStream_t st) {
  if (A.T == 1) moe_small_router<1, X, R><<<grid, ROUTER_THREADS, 0, st>>>(A, vec);
  else if (A.T <= 4) moe_small_router<4, X, R><<<grid, ROUTER_THREADS, 0, st>>>(A, vec);
  else if (A.T <= 8) moe_small_router<8, X, R><<<grid, ROUTER_THREADS, 0, st>>>(A, vec);
  else moe_small_router<16, X, R><<<grid, ROUTER_THREADS, 0, st>>>(A, vec);
}
template <typename X>
void launch_router(const SmallArgs& A, unsigned grid, int vec, cudaStream_t st) {
  if (A.router_dtype == MQ_F32) launch_router_of<X, float>(A, grid, vec, st);
  else if (A.router_dtype == MQ_BF16) launch_router_of<X, __nv_bfloat16>(A, grid, vec, st);
  else launch_router_of<X, __half>(A, grid, vec, st);
}

template <int F, int OCT, typename OutT>
int launch_layer(const SmallArgs& A, cudaStream_t st) {
  const size_t smem = front_bytes(F, OCT) + Tables::bytes(A.T, A.E, A.K) + 1024;
  // The limit is the kernel's, not the call's: one that went by the call would be lowered by a smaller one on another thread
  // between this line and the launch.  So always the largest.
  constexpr size_t room = front_bytes(F, OCT) + Tables::bytes(8 * OCT, MAX_E, MAX_K) + 1024;
  static_assert(room + 1024 <= 232448, "shared memory of a CTA, and what the kernel has of its own");
  cudaError_t e = cudaFuncSetAttribute(moe_small_layer<F, OCT, OutT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)room);
  int dev = 0, sms = 0;
  if (e == cudaSuccess) e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e == cudaSuccess) {
    SmallArgs args = A;
    SmallMaps maps = {};
    if (!small_maps<F>(args, sms, maps)) return MQ_ERR_DRIVER_ENTRY;
    void* argv[] = {&args, &maps};
    e = cudaLaunchCooperativeKernel((const void*)moe_small_layer<F, OCT, OutT>, dim3(sms), dim3(Roles<F, OCT>::THREADS), argv, smem, st);
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    set_last_cuda_error(e);
    return e == cudaErrorCooperativeLaunchTooLarge ? MQ_ERR_NOT_RESIDENT : MQ_ERR_LAUNCH_FAILED;
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
  if (L.dtype == MQ_F32) launch_router<float>(A, grid, router_vec, st);
  else if (L.dtype == MQ_BF16) launch_router<__nv_bfloat16>(A, grid, router_vec, st);
  else launch_router<__half>(A, grid, router_vec, st);
  const int rc = check_launch();
  if (rc != MQ_OK) return rc;
  return T <= 8 ? launch_format<1>(A, format, st) : launch_format<2>(A, format, st);
}
