// W8A8 products on CTA pairs (tcgen05.mma.cta_group::2, kind::i8): int8 rows times int8 weights into int32 sums in tensor
// memory, scaled by row and by output channel on the way out; for one linear or for rows grouped by expert, optionally with
// the row gather in front and SwiGLU behind.  w8a8.cuh has the arithmetic.
//
// An 8-bit operand block is the same 128 bytes a row as a 16-bit one, holds twice the k, and the tensor cores take the same
// time over it, so the layout is that of grouped_gemm_pair.cu: 256 weight rows over the pair are the MMA's M, tokens its N,
// each CTA stages its own 128 weight rows and half of the tokens (a ring of four stages of 48 KB), and a tile has one of
// these shapes by the rows of its group:
//   TOKENS2   one sub-tile of 256 weight rows against two token tiles (up to 512 rows in all);
//   WEIGHTS2  two sub-tiles against one token tile of 129 to 256 rows (or one sub-tile, where the tiles are kept small);
//   DEEP      one sub-tile, up to 128 rows, 256 k per stage; consecutive tiles alternate between the accumulators.
// K is covered in blocks of 128; what a copy reads past K, past the last row or past the last channel is zero (the tensor
// maps' fill), so K and N need only be multiples of 16.
// With few rows the tiles are kept narrow, so that there is one for every pair (w8_tile_rows).
// What bounds it: with few rows an expert HBM, with many the operands' way from L2 (a pair's stage of 64 KB takes 1.2 times as
// long as its MMAs) and the clock under the power cap.  Measured, int8 rows given, weights out of L2 (hidden 2048, inter 768,
// 128 experts, top-8): gate/up with the gather 58 us for 32 tokens (6.2 TB/s of weights), 70 for 512 (5.8), 115 for 4096 (1.8
// Pop/s); down 40 for 512, 76 for 4096; a linear of 4096 rows, 2048 -> 4096 32 us (2.1 Pop/s), of 500 rows, 4096 -> 2048 10.
// (Weights asked for ahead by tensor-map prefetches to L2: 64 tokens 69 to 87 us instead of 65.)
// Warps: 0 copies, 1 MMA (even CTA), 2-9 epilogue, 10-13 (gathering variant) row copies.  Every wait is bounded: when one
// runs out, MQ_DEV_WAIT_EXPIRED is set, all roles leave their loops, copies in flight are waited for and TMEM is freed.
#include "pair.cuh"
#include "w8a8.cuh"

namespace mq {
namespace {

using namespace tc5;

constexpr int WM = 128;                          // weight rows per sub-tile and CTA = TMEM lanes
constexpr int WK = 128;                          // k per operand block: one 128-byte swizzle span
constexpr int WN = 256;                          // most tokens per MMA
constexpr int W_BLOCK = WM * WK;                 // 16 KB: an operand block
constexpr int W_STAGE = 3 * W_BLOCK;             // A0 | A1 or B1 | B0 (DEEP: A k0 | A k1 | B k0, B k1)
constexpr int W_NST = 4;
constexpr int W_BOX = 32;                        // token rows per box
constexpr int W_BOX_BYTES = W_BOX * WK;
constexpr int W_EPI = 8, W_GATHER = 4;           // warps
constexpr int W_STG = 32 * 64;                   // staged output rows of an epilogue warp
constexpr int W_MAX_E = 1024;
constexpr int W_SORT_E = 256;                    // most groups that are put in order of size
constexpr int W_TABLE = (2 * (W_MAX_E + 1) + W_SORT_E) * 4;
constexpr int W_SMEM = 1024 + W_NST * W_STAGE + W_EPI * W_STG + 256 + ((W_TABLE + 15) & ~15);
static_assert(W_SMEM <= 232448, "shared memory of a CTA");

enum W8Shape { WEIGHTS2, TOKENS2, DEEP };

__device__ __forceinline__ void mma_pair_i8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accum) : "memory");
}
// D int32, A and B signed 8-bit, both K-major
__device__ __forceinline__ uint32_t idesc_s8(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

template <typename T> __device__ __forceinline__ uint32_t pack16(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}
template <> __device__ __forceinline__ uint32_t pack16<__half>(float lo, float hi) {
  const __half2 p = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}
template <> __device__ __forceinline__ uint32_t pack16<float>(float, float) { return 0u; }

// A tile of work.  Chunk c (0, 1) is the token tile of accumulator c; with WEIGHTS2 both are the same rows.
struct W8Tile {
  int expert, unit, shape;                       // unit: first sub-tile (256 weight rows over the pair)
  bool two;                                      // both accumulators are used
  int tok0, ntok;                                // first token row and token rows of the tile
  int n0, n1;                                    // MMA N of the token chunks (multiples of 32; n1 = 0: one chunk)
};

// Tiles are dealt out in the groups' order, the pairs in turn; with skewed groups and more than one round of tiles, largest
// groups first and the pairs back and forth (a tile of 512 rows takes four times one of 128).
struct W8Table {
  __device__ static int weight_of(const W8Args& A, int expert) { return A.period == A.E ? expert : expert % A.period; }
  const int* off;                                // [E + 1]
  const int* group;                              // [E]: the groups by size, or null: in their own order
  const int* first;                              // [E + 1]: first tile of the group in that order
  int E, units, most;                            // most: rows a tile may have (a multiple of 32; above 256: two chunks)
  __device__ static int tiles_of(int n, int units, int most) {
    if (n <= 0) return 0;
    if (most <= WN) return (n + most - 1) / most * units;
    return n <= 128 ? units : n <= WN ? (units + 1) / 2 : (n + most - 1) / most * units;
  }
  __device__ W8Tile locate(int t) const {
    int lo = 0, hi = E;                          // first[lo] <= t < first[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (first[mid] <= t) lo = mid; else hi = mid;
    }
    const int local = t - first[lo], e = group != nullptr ? group[lo] : lo, n = off[e + 1] - off[e];
    W8Tile w;
    w.expert = e;
    w.n1 = 0;
    if (most > WN && n > 128 && n <= WN) {
      w.shape = WEIGHTS2;
      w.unit = 2 * local;
      w.two = w.unit + 1 < units;
      w.tok0 = off[e];
      w.ntok = n;
      w.n0 = (n + 31) & ~31;
      return w;
    }
    // balanced cuts; mostly there is one, and no division to wait for
    const int cuts = n <= most ? 1 : (n + most - 1) / most, cut = cuts == 1 ? 0 : local / units;
    const int width = ((cuts == 1 ? n : (n + cuts - 1) / cuts) + 31) & ~31;
    w.unit = local - cut * units;
    w.tok0 = off[e] + cut * width;
    w.ntok = max(0, min(width, n - cut * width));
    if (width > WN) {
      w.shape = TOKENS2;
      w.n0 = (((w.ntok + 1) >> 1) + 31) & ~31;
      w.n1 = w.ntok > w.n0 ? (w.ntok - w.n0 + 31) & ~31 : 0;
      w.two = w.n1 > 0;
    } else {
      w.shape = width <= 128 ? DEEP : WEIGHTS2;
      w.n0 = max(32, (w.ntok + 31) & ~31);
      w.two = false;
    }
    if (w.n0 < 32) w.n0 = 32;
    return w;
  }
};

template <bool SWIGLU, bool GATHER, typename OutT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__((2 + W_EPI + (GATHER ? W_GATHER : 0)) * 32, 1)
w8a8_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const W8Args A,
                 const int most_rows, int32_t* d_status) {
  constexpr int CW = SWIGLU ? 64 : 128;          // output columns per sub-tile and CTA
  extern __shared__ uint8_t w8_smem_raw[];
  const uint32_t raw = smem_addr(w8_smem_raw);
  const uint32_t ring = (raw + 1023u) & ~1023u;  // the swizzle pattern repeats every 1024 bytes
  uint8_t* ptr = w8_smem_raw + (ring - raw);
  uint8_t* stg_mem = ptr + W_NST * W_STAGE;
  uint8_t* bar_mem = stg_mem + W_EPI * W_STG;
  const uint32_t bars = ring + W_NST * W_STAGE + W_EPI * W_STG;
  auto full = [&](int s) { return bars + 8u * s; };              // waited on by the even CTA's MMA warp only
  auto empty = [&](int s) { return bars + 8u * (W_NST + s); };
  auto tfull = [&](int b) { return bars + 8u * (2 * W_NST + b); };
  auto tempty = [&](int b) { return bars + 8u * (2 * W_NST + 2 + b); };   // even CTA only
  volatile uint32_t* tmem_ptr = reinterpret_cast<volatile uint32_t*>(bar_mem + 8 * (2 * W_NST + 4));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bar_mem + 8 * (2 * W_NST + 4) + 8);
  volatile int* skew_flag = reinterpret_cast<volatile int*>(bar_mem + 8 * (2 * W_NST + 4) + 12);
  int* s_off = reinterpret_cast<int*>(bar_mem + 256);
  int* s_first = s_off + A.E + 1;
  int* s_group = s_first + A.E + 1;

  const int warp = (int)uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int rank = (int)uniform(cluster_rank());
  const int E = A.E, N = A.N, KB = (A.K + WK - 1) / WK;
  const int units = (N + 2 * CW - 1) / (2 * CW);

  if (threadIdx.x == 0) {
    for (int s = 0; s < W_NST; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(tfull(b), 1);
      mbar_init(tempty(b), 2 * W_EPI);
    }
    *abort_flag = 0;
    mbar_init_fence();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_addr((const void*)tmem_ptr)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  for (int e = threadIdx.x; e <= E; e += blockDim.x) s_off[e] = A.offsets == nullptr ? e * A.S : w8_offset(A, e);
  __syncthreads();
  const int pairs = (int)(gridDim.x >> 1), pair = (int)(blockIdx.x >> 1);
  // first[]: exclusive sums of the groups' tile counts; the largest group's rows
  auto count_tiles = [&](const int* order) {
    int carry = 0, top = 0;
    for (int e0 = 0; e0 < E; e0 += 32) {
      const int at = e0 + lane, e = order != nullptr && at < E ? order[at] : at;
      const int n = at < E ? s_off[e + 1] - s_off[e] : 0, c = W8Table::tiles_of(n, units, most_rows);
      top = max(top, n);
      int incl = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      if (at < E) s_first[at] = carry + incl - c;
      carry += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) s_first[E] = carry;
    return __reduce_max_sync(0xffffffffu, top);
  };
  if (warp == 0) {
    const int top = count_tiles(nullptr);
    // skewed: the largest group is over twice the average
    if (lane == 0) *skew_flag = E <= W_SORT_E && s_first[E] > pairs && top > WN && top / 2 > (s_off[E] - s_off[0]) / E;
  }
  fence_before_sync();
  __syncthreads();
  const bool skewed = *skew_flag != 0;
  if (skewed) {                                  // a group's place is the number of larger ones, equals in their order
    int n[W_SORT_E / 32];
#pragma unroll
    for (int j = 0; j < W_SORT_E / 32; ++j) {
      const int e = 32 * j + lane;
      n[j] = e < E ? s_off[e + 1] - s_off[e] : INT32_MIN;
    }
    for (int e = warp; e < E; e += (int)(blockDim.x >> 5)) {
      const int mine = s_off[e + 1] - s_off[e];
      int before = 0;
#pragma unroll
      for (int j = 0; j < W_SORT_E / 32; ++j) before += n[j] > mine || (n[j] == mine && 32 * j + lane < e) ? 1 : 0;
      before = __reduce_add_sync(0xffffffffu, before);
      if (lane == 0) s_group[before] = e;
    }
    __syncthreads();
    if (warp == 0) count_tiles(s_group);
  }
  cluster_sync();                                // barriers, TMEM and table of both CTAs are ready
  fence_after_sync();
  const uint32_t tmem = uniform(*tmem_ptr);
  const W8Table table{s_off, skewed ? s_group : nullptr, s_first, E, units, most_rows};
  const int total = s_first[E];
  auto deal = [&](int i) { return i * pairs + (skewed && (i & 1) != 0 ? pairs - 1 - pair : pair); };   // its i-th tile
  auto steps_of = [&](int shape) { return shape == DEEP ? (KB + 1) / 2 : KB; };                        // ring stages a tile

  if (warp == 0) {
    // ------------------------------------------------------------------ operand copies
    // The whole warp walks the loop and one elected lane issues, so that addresses and coordinates are in uniform registers.
    const bool leader = elect_one();
    const uint32_t full0 = uniform(in_leader(full(0)));
    int stage = 0, filled = 0;
    uint32_t phase = 0;
    bool ok = true;
    // this CTA's 128 weight rows of sub-tile `unit`, 128 k from k
    auto load_a = [&](uint32_t dst, uint32_t bar, int k, int wexpert, int unit) {
      const int c = unit * 2 * CW + rank * CW;
      if (SWIGLU) tma_load_5d_pair(dst, &map_w, bar, k, c / 16, wexpert);
      else tma_load_pair(dst, &map_w, bar, k, wexpert * N + c);
    };
    auto load_b = [&](uint32_t dst, uint32_t bar, int k, int row, int boxes) {
      for (int b = 0; b < boxes; ++b) tma_load_pair(dst + b * W_BOX_BYTES, &map_x, bar, k, row + b * W_BOX);
    };
    for (int nth = 0; deal(nth) < total && ok; ++nth) {
      const W8Tile w = table.locate(deal(nth));
      const int we = (int)uniform(W8Table::weight_of(A, w.expert)), unit = (int)uniform(w.unit), shape = (int)uniform(w.shape);
      const bool two = uniform(w.two) != 0;
      const int h0 = (int)uniform(w.n0 >> 1), h1 = (int)uniform(w.n1 >> 1);     // this CTA's halves of the token chunks
      const int box0 = (h0 + W_BOX - 1) / W_BOX, box1 = (h1 + W_BOX - 1) / W_BOX;   // rows past the half: not read
      const int tok0 = (int)uniform(w.tok0), row0 = tok0 + rank * h0, row1 = tok0 + 2 * h0 + rank * h1;
      const bool both = shape == WEIGHTS2 && two;
      uint32_t bytes = W_BLOCK * (both ? 2 : 1) + (GATHER ? (h0 + h1) * WK : (box0 + box1) * W_BOX_BYTES);
      if (shape == DEEP) bytes *= 2;
      const int steps = steps_of(shape), step = shape == DEEP ? 2 : 1;
      for (int i = 0; i < steps; ++i) {
        ok = mbar_wait_warp(empty(stage), phase ^ 1u, abort_flag, d_status);
        if (!ok) break;
        const uint32_t a = ring + stage * W_STAGE, a1 = a + W_BLOCK, b = a + 2 * W_BLOCK;
        const uint32_t bar = full0 + 8u * stage;
        const int k = i * step * WK;
        if (leader) {
          if (rank == 0) mbar_expect_tx(full(stage), 2 * bytes);           // both CTAs' copies
          load_a(a, bar, k, we, unit);
          if (both) load_a(a1, bar, k, we, unit + 1);
          if (shape == DEEP) load_a(a1, bar, k + WK, we, unit);
          if (!GATHER) {
            load_b(b, bar, k, row0, box0);
            if (shape == DEEP) load_b(b + W_BLOCK / 2, bar, k + WK, row0, box0);
            else load_b(a1, bar, k, row1, box1);
          }
        }
        __syncwarp();
        ++filled;
        if (++stage == W_NST) { stage = 0; phase ^= 1u; }
      }
    }
    // every stage that was filled has been read before the CTA exits; after giving up: the copies have landed
    for (int s = 0; s < W_NST && ok; ++s) {
      ok = mbar_wait_warp(empty(stage), phase ^ 1u, abort_flag, d_status);
      if (++stage == W_NST) { stage = 0; phase ^= 1u; }
    }
    if (!ok && rank == 0) {
      for (int f = max(0, filled - W_NST); f < filled; ++f)
        mbar_wait_limited(full(f % W_NST), (uint32_t)(f / W_NST) & 1u, 1u << 16);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer (even CTA)
    if (rank == 0) {
      const bool leader = elect_one();
      int stage = 0, cur = 0;                    // cur: accumulator of the next single-accumulator tile
      uint32_t phase = 0, used = 0;              // used: parity of the tiles each accumulator has held, a bit each
      bool ok = true;
      for (int nth = 0; deal(nth) < total && ok; ++nth) {
        W8Tile w = table.locate(deal(nth));
        w.shape = (int)uniform(w.shape);
        w.two = uniform(w.two) != 0;
        const int b0 = w.two ? 0 : cur;
        ok = wait_cluster(tempty(b0), ((used >> b0) & 1u) ^ 1u, abort_flag, d_status);
        if (!ok) break;
        fence_after_sync();
        // A stage is four MMAs on (A0, B0) and, unless the tile has one accumulator and 128 k per stage, four more on the
        // operands its shape pairs up.  Everything they are issued with is uniform over the warp.
        const bool second = w.two || w.shape == DEEP;
        const uint32_t acc0 = uniform(tmem + b0 * WN), acc1 = w.shape == DEEP ? acc0 : uniform(tmem + WN);
        const uint32_t id0 = uniform(idesc_s8(2 * WM, w.n0));
        const uint32_t id1 = w.shape == TOKENS2 ? uniform(idesc_s8(2 * WM, w.n1)) : id0;
        const uint32_t a1 = w.shape == TOKENS2 ? 0 : W_BLOCK;                       // offsets inside a stage
        const uint32_t b1 = w.shape == TOKENS2 ? W_BLOCK : 2 * W_BLOCK + (w.shape == DEEP ? W_BLOCK / 2 : 0);
        const int steps = steps_of(w.shape);
        // With two accumulators a tile starts on the first one while the epilogue still drains the second: the first
        // `ahead` stages' MMAs on it go out before the second is waited for.
        const int ahead = w.two ? min(W_NST, steps) : 0;
        auto four = [&](uint32_t acc, uint32_t a, uint32_t b, uint32_t id, uint32_t add) {
          const uint64_t da = smem_desc(a), db = smem_desc(b);
          // 32 k = 32 bytes along the swizzled row: + 2 in the descriptor's address field
          mma_pair_i8(acc, da, db, id, add);
#pragma unroll
          for (int k = 1; k < WK / 32; ++k) mma_pair_i8(acc, da + 2u * k, db + 2u * k, id, 1u);
        };
        for (int i = 0; i < ahead && ok; ++i) {
          int st = stage + i;
          const uint32_t ph = st >= W_NST ? phase ^ 1u : phase;
          if (st >= W_NST) st -= W_NST;
          ok = wait_cluster(full(st), ph, abort_flag, d_status);
          if (!ok) break;
          fence_after_sync();
          const uint32_t s = ring + st * W_STAGE;
          if (leader) {
            four(acc0, s, s + 2 * W_BLOCK, id0, i != 0 ? 1u : 0u);
            if (i == steps - 1) commit_pair(tfull(b0));
          }
          __syncwarp();
        }
        if (ok && w.two) ok = wait_cluster(tempty(1), (used >> 1) ^ 1u, abort_flag, d_status);
        for (int i = 0; i < steps && ok; ++i) {
          if (i >= ahead) ok = wait_cluster(full(stage), phase, abort_flag, d_status);
          if (!ok) break;
          fence_after_sync();
          const uint32_t s = ring + stage * W_STAGE;
          if (leader) {
            if (i >= ahead) four(acc0, s, s + 2 * W_BLOCK, id0, i != 0 ? 1u : 0u);
            if (i >= ahead && w.two && i == steps - 1) commit_pair(tfull(b0));
            if (second) four(acc1, s + a1, s + b1, id1, w.shape == DEEP || i != 0 ? 1u : 0u);
            commit_pair(empty(stage));
            if (i == steps - 1) commit_pair(tfull(w.two ? 1 : b0));
          }
          __syncwarp();
          if (++stage == W_NST) { stage = 0; phase ^= 1u; }
        }
        if (!ok) break;
        used ^= w.two ? 3u : 1u << b0;
        cur = w.two ? 0 : cur ^ 1;
      }
    }
  } else if (GATHER && warp >= 2 + W_EPI) {
    // ------------------------------------------------------------------ row copies of the gathering variant
    // A copy moves four rows x 128 k of x, gathered into four rows of a swizzled operand.  A stage's copies (this CTA's
    // halves of its token chunks; with DEEP one chunk, twice 128 k) are dealt out to the warps; lane i keeps what its warp's
    // copy i needs and hands it over by shuffle, so that the copies are issued from uniform registers.
    // Rows past the group's last repeat it: computed, not stored.
    const bool leader = elect_one();
    const uint32_t full0 = uniform(in_leader(full(0)));
    const int gw = warp - (2 + W_EPI);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    int next[4] = {0, 0, 0, 0}, count_next = 0, shape_next = 0;
    uint32_t at_next = 0;                        // where in a stage the copy lands; bit 0: the second 128 k of the stage
    auto fetch = [&](int t) {
      const W8Tile tl = table.locate(t);
      const int h0 = tl.n0 >> 1, h1 = tl.n1 >> 1, c0 = h0 >> 2, copy = gw + W_GATHER * lane;
      const bool deep = tl.shape == DEEP, later = copy >= c0;               // in the second half of the list
      const int i = later ? copy - c0 : copy, copies = c0 + (deep ? c0 : h1 >> 2);
      at_next = (!later ? 2 * W_BLOCK : deep ? 2 * W_BLOCK + W_BLOCK / 2 + 1 : W_BLOCK) + 512u * i;
      shape_next = tl.shape;
      count_next = (copies - gw + W_GATHER - 1) / W_GATHER;                 // this warp's (at most 16)
      if (copy < copies) {
        const int first = tl.tok0 + (later && !deep ? tl.n0 + rank * h1 : rank * h0) + 4 * i;
        const int last = max(0, min(tl.tok0 + tl.ntok, A.S) - 1);
#pragma unroll
        for (int j = 0; j < 4; ++j) next[j] = (int)w8_source(A, min(first + j, last));
      }
    };
    if (pair < total) fetch(pair);
    for (int nth = 0; deal(nth) < total && ok; ++nth) {
      int row[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) row[i] = next[i];
      const uint32_t at = at_next;
      const int count = (int)uniform(count_next), shape = (int)uniform(shape_next);
      const int steps = steps_of(shape), step = shape == DEEP ? 2 : 1;
      if (deal(nth + 1) < total) fetch(deal(nth + 1));   // the next tile's positions travel under this tile's copies
      for (int s_at = 0; s_at < steps; ++s_at) {
        ok = mbar_wait_warp(empty(stage), phase ^ 1u, abort_flag, d_status);
        if (!ok) break;
        const uint32_t s = ring + stage * W_STAGE, bar = full0 + 8u * stage;
#pragma unroll 4
        for (int i = 0; i < count; ++i) {
          int r[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) r[j] = __shfl_sync(0xffffffffu, row[j], i);
          const uint32_t d = __shfl_sync(0xffffffffu, at, i);
          if (leader) tma_gather4_pair(s + (d & ~1u), &map_x, bar, (s_at * step + (int)(d & 1u)) * WK, r);
        }
        __syncwarp();
        if (++stage == W_NST) { stage = 0; phase ^= 1u; }
      }
    }
  } else if (warp < 2 + W_EPI) {
    // ------------------------------------------------------------------ epilogue
    // Two groups of four warps drain the even and the odd 32-token blocks of an accumulator.  A warp holds 32 of the CTA's
    // 128 lanes (weight rows) and works by itself: it scales its sums in the fragment layout (a lane holds rows lane / 4 and
    // lane / 4 + 8 of each 16, and tokens 2 (lane % 4) and the next of each 8), and for 16-bit results stmatrix.trans turns
    // the block into token-major rows in its own staging space (16-byte pieces placed so that both ways are free of bank
    // conflicts): 64 bytes of 32 output columns, or 32 bytes of 16 columns with SwiGLU (lanes 0..15 are gate rows, 16..31 the
    // up rows of the same columns).  fp32 results are stored from the fragments, eight columns a token at a time.
    const int quad = warp & 3, group = (warp - 2) >> 2;
    constexpr int PIECES = SWIGLU ? 2 : 4, ROWB = 16 * PIECES;             // of a staged token row
    uint8_t* stg = stg_mem + (warp - 2) * W_STG;
    const uint32_t stg_s = smem_addr(stg);
    const int mi = lane >> 3, ri = lane & 7;
    auto place = [&](int tok, int piece) { return (uint32_t)(tok * ROWB + ((piece ^ ((tok * PIECES >> 3) & (PIECES - 1))) << 4)); };
    // two tokens' sums times their scales, times the channel's (as w8_value, two at a time)
    auto scaled = [](uint32_t lo, uint32_t hi, f32x2 rows, float channel) {
      return unpack2(mul2(mul2(pack2(__int2float_rn((int)lo), __int2float_rn((int)hi)), rows), pack2(channel, channel)));
    };
    OutT* out = reinterpret_cast<OutT*>(A.out);
    // An accumulator's share of a tile: its token rows, this warp's columns, and the scales the lane needs.
    struct Chunk {
      int row0, nrow, col0;                        // first token row and token rows; first output column of the warp
      float ws[2][2];                              // of the lane's weight rows: [half][row, row + 8]; SwiGLU: half 0 gate, half 1 up
      float xs[4];                                 // of the token that the lane stands for in each block
    };
    auto chunk_of = [&](const W8Tile& w, int c) {
      Chunk k;
      const bool second_rows = c == 1 && w.shape == TOKENS2;
      k.row0 = w.tok0 + (second_rows ? w.n0 : 0);
      k.nrow = second_rows ? w.ntok - w.n0 : min(w.ntok, w.n0);
      k.col0 = (w.unit + (c == 1 && w.shape == WEIGHTS2 ? 1 : 0)) * 2 * CW + rank * CW + quad * (CW / 4);
      const float* ws = A.w_scale + (size_t)W8Table::weight_of(A, w.expert) * (SWIGLU ? 2 * N : N);
#pragma unroll
      for (int hl = 0; hl < 2; ++hl)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int col = k.col0 + (SWIGLU ? 0 : 16 * hl) + 8 * j + (lane >> 2);
          k.ws[hl][j] = col < N ? ws[SWIGLU && hl == 1 ? N + col : col] : 0.0f;
        }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 32 * group + 64 * i + lane;
        k.xs[i] = r < k.nrow ? A.x_scale[w8_source(A, k.row0 + r)] : 0.0f;
      }
      return k;
    };
    uint32_t used = 0;
    int cur = 0, nth = 0, c = 0;
    bool ok = true;
    W8Tile w;
    Chunk k;
    if (deal(0) < total) {
      w = table.locate(deal(0));
      k = chunk_of(w, 0);
    }
    while (deal(nth) < total) {
      const int b = c == 1 ? 1 : w.two ? 0 : cur;
      // the next chunk's scales come from afar (its rows through the permutation): they travel while this one is finished
      const bool same = c == 0 && w.two;
      W8Tile next = w;
      if (!same && deal(nth + 1) < total) next = table.locate(deal(nth + 1));
      Chunk ahead = k;
      if (same || deal(nth + 1) < total) ahead = chunk_of(next, same ? 1 : 0);
      ok = mbar_wait_warp(tfull(b), (used >> b) & 1u, abort_flag, d_status);
      if (!ok) break;
      used ^= 1u << b;
      fence_after_sync();
      const int blocks = max(0, (k.nrow - 32 * group + 63) >> 6);          // of 32 tokens, every other one
      constexpr int PACKED = SWIGLU ? 8 : 16;
      // Blocks leave tensor memory two at a time.  The accumulator is free once the last two are in registers, and what follows
      // runs under the next tile's MMAs.
      auto load = [&](int i0, uint32_t (&f)[2][2][16]) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (i0 + i < blocks) {
            const uint32_t ta = tmem + b * WN + ((uint32_t)(quad * 32) << 16) + 32 * group + 64 * (i0 + i);
            tmem_ld_frag(ta, f[i][0]);
            tmem_ld_frag(ta + (16u << 16), f[i][1]);
          }
        }
        tmem_ld_wait();
      };
      auto release = [&] {
        fence_before_sync();
        __syncwarp();
        // relaxed: the sums are in registers, and a release would wait for the stores of the chunk before and the loads for the
        // next (half of the finishing warps' time)
        if (lane == 0) arrive_cluster_relaxed(in_leader(tempty(b)));
      };
      auto scale = [&](int i0, const uint32_t (&f)[2][2][16], uint32_t (&v)[2][PACKED]) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (i0 + i < blocks) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {                                  // token octets
              const f32x2 s01 = pack2(__shfl_sync(0xffffffffu, k.xs[i0 + i], 8 * j + 2 * (lane & 3)),
                                      __shfl_sync(0xffffffffu, k.xs[i0 + i], 8 * j + 2 * (lane & 3) + 1));
#pragma unroll
              for (int q = 0; q < 2; ++q) {                                // weight rows lane / 4 and lane / 4 + 8
                const float2 x = scaled(f[i][0][4 * j + 2 * q], f[i][0][4 * j + 2 * q + 1], s01, k.ws[0][q]);
                const float2 y = scaled(f[i][1][4 * j + 2 * q], f[i][1][4 * j + 2 * q + 1], s01, k.ws[1][q]);
                const float a0 = SWIGLU ? w8_swiglu<OutT>(x.x, y.x) : x.x, a1 = SWIGLU ? w8_swiglu<OutT>(x.y, y.y) : x.y;
                if (sizeof(OutT) == 4) {
                  const int r = 32 * group + 64 * (i0 + i) + 8 * j + 2 * (lane & 3), col = k.col0 + 8 * q + (lane >> 2);
                  float* o = reinterpret_cast<float*>(out) + (size_t)(k.row0 + r) * N + col;
                  if (r < k.nrow && col < N) o[0] = a0;
                  if (r + 1 < k.nrow && col < N) o[N] = a1;
                  if (!SWIGLU && r < k.nrow && col + 16 < N) o[16] = y.x;
                  if (!SWIGLU && r + 1 < k.nrow && col + 16 < N) o[N + 16] = y.y;
                } else {
                  v[i][2 * j + q] = pack16<OutT>(a0, a1);
                  if (!SWIGLU) v[i][(8 + 2 * j + q) % PACKED] = pack16<OutT>(y.x, y.y);
                }
              }
            }
          }
        }
      };
      auto store = [&](int i0, const uint32_t (&v)[2][PACKED]) {
        if (sizeof(OutT) == 4) return;                                     // stored from the fragments
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (i0 + i < blocks) {
            const int r = 32 * group + 64 * (i0 + i);
            __syncwarp();                                                  // the previous block's rows have been read
#pragma unroll
            for (int j2 = 0; j2 < 2; ++j2) {                               // token octets (0, 1) and (2, 3)
              const int tok = 8 * (2 * j2 + (mi >> 1)) + ri;
#pragma unroll
              for (int hl = 0; hl < (SWIGLU ? 1 : 2); ++hl)
                stmatrix_x4_trans(stg_s + place(tok, 2 * hl + (mi & 1)), v[i][(8 * hl + 4 * j2) % PACKED],
                                  v[i][(8 * hl + 4 * j2 + 1) % PACKED], v[i][(8 * hl + 4 * j2 + 2) % PACKED],
                                  v[i][(8 * hl + 4 * j2 + 3) % PACKED]);
            }
            __syncwarp();
#pragma unroll
            for (int q = 0; q < PIECES; ++q) {
              const int row = (32 / PIECES) * q + lane / PIECES, p = lane % PIECES;
              if (row < k.nrow - r && k.col0 + p * 8 < N)
                *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(out) + (size_t)(k.row0 + r + row) * N + k.col0 + p * 8) =
                    *reinterpret_cast<const uint4*>(stg + place(row, p));
            }
          }
        }
      };
      uint32_t f[2][2][16], v[2][PACKED];
      load(0, f);
      if (blocks > 2) {
        scale(0, f, v);
        load(2, f);
        release();
        store(0, v);
        scale(2, f, v);
        store(2, v);
      } else {
        release();
        scale(0, f, v);
        store(0, v);
      }
      if (same) {
        c = 1;
      } else {
        cur = w.two ? 0 : cur ^ 1;
        c = 0;
        ++nth;
        w = next;
      }
      k = ahead;
    }
  }

  fence_before_sync();
  __syncthreads();
  cluster_sync();                                // nothing of the pair is in flight towards either CTA any more
  if (warp == 1) {
    fence_after_sync();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// 2-D int8 row-major [rows, cols] tensor, boxes of 128 columns x box_rows rows, 128-byte swizzle.
bool w8_map(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int box_rows) {
  EncodeTiledFn fn = tensor_map_encoder();
  if (!fn) return false;
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)cols};
  cuuint32_t box[2] = {(cuuint32_t)WK, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1u, 1u};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Gate and up rows [experts, 2, N, K] as [experts, N / 16 groups, 2, 16, K]: a box is four groups, 16 gate rows and the 16 up
// rows of the same columns in turn: the 128 lanes of a sub-tile.
bool w8_map_gate_up(CUtensorMap* map, const void* base, int64_t experts, int64_t N, int64_t K) {
  EncodeTiledFn fn = tensor_map_encoder();
  if (!fn) return false;
  const cuuint64_t row = (cuuint64_t)K;
  cuuint64_t dims[5] = {(cuuint64_t)K, 16, 2, (cuuint64_t)(N / 16), (cuuint64_t)experts};
  cuuint64_t strides[4] = {row, row * N, row * 16, row * 2 * N};
  cuuint32_t box[5] = {(cuuint32_t)WK, 16, 2, 4, 1};
  cuuint32_t estr[5] = {1u, 1u, 1u, 1u, 1u};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 5, const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Rows a tile may have: the width at which the rounds of tiles take the shortest time, by a model of a tile in clocks (the
// MMAs' 2 a row and block of 128 k, or the copies' time where that is longer, and a fixed part) and of the last epilogue, which
// nothing hides (16 a row, 40 with SwiGLU), from the mean group.  Of 24 sizes tried with every width the slowest choice took 7 %
// longer than the best one (2048 tokens, 16 experts, top-4, K 1024, 512 columns: 19.8 us with 256 rows, 18.5 with 128, 24.4 with
// 512).
int w8_tile_rows(int64_t S, int64_t E, int64_t units, int64_t KB, int64_t pairs, bool swiglu) {
  const int64_t groups = E < S ? E : S, n = (S + groups - 1) / groups;
  int best = 512;
  double best_time = 0.0;
  for (int width = 512; width >= 32; width -= width > 256 ? 256 : 32) {
    const int64_t cuts = (n + width - 1) / width;
    const double rows = (double)((((n + cuts - 1) / cuts) + 31) & ~(int64_t)31);
    double tiles = (double)(groups * cuts * units), stage = 2.0 * rows > 300.0 + 1.2 * rows ? 2.0 * rows : 300.0 + 1.2 * rows;
    if (width > 256 && n > 128 && n <= 256) {              // two sub-tiles to a tile
      tiles *= 0.5;
      stage *= 2.0;
    }
    const double rounds = tiles <= (double)pairs ? 1.0 : tiles / (double)pairs + 0.5;
    const double time = rounds * ((double)KB * stage + 1500.0) + rows * (swiglu ? 40.0 : 16.0);
    if (width == 512 || time < best_time * 0.98) {
      best = width;
      best_time = time;
    }
  }
  return best;
}

}  // namespace

// Whole 16-byte pieces of every row of the operands and the result; coordinates and tile counts are 32-bit.  Against the small
// tiles of w8a8.cu, which it is measured against at 1 to 256 rows, K 2048 to 131056 and N 16 to 4096, it is nowhere the slower one
// (us, here | there: K 2048, N 16 8.4 | 8.4 for any of these rows; one row of K 2048, N 4096 10.1 | 12.7, 256 rows 11.2 | 27.2; one
// row of K 32768, N 64 38.7 | 102.8).
bool w8a8_pair_covers(const W8Args& A, bool swiglu) {
  return A.K % 16 == 0 && A.N % 16 == 0 && aligned16(A.x) && aligned16(A.w) && aligned16(A.out) && A.E <= W_MAX_E &&
         (int64_t)A.period * A.N * 2 < ((int64_t)1 << 31) &&
         ((int64_t)A.S / 32 + A.E) * (A.N / (swiglu ? 128 : 256) + 1) < ((int64_t)1 << 30);
}

int w8a8_pair(const W8Args& A, bool swiglu, int out_dtype, int32_t* d_status, cudaStream_t st) {
  CUtensorMap map_x, map_w;
  const bool gather = A.perm != nullptr;
  // a gathered copy takes its rows one by one: boxes of one row
  if (!w8_map(&map_x, A.x, A.T, A.K, gather ? 1 : W_BOX) ||
      !(swiglu ? w8_map_gate_up(&map_w, A.w, A.period, A.N, A.K) : w8_map(&map_w, A.w, (int64_t)A.period * A.N, A.K, WM)))
    return MQ_ERR_DRIVER_ENTRY;
  const int64_t units = (A.N + (swiglu ? 128 : 256) - 1) / (swiglu ? 128 : 256), pairs = device_sm_count() / 2;
  const int most = w8_tile_rows(A.S, A.E, units, (A.K + WK - 1) / WK, pairs, swiglu);
  const int64_t tiles = ((int64_t)A.S / (most < 256 ? most : 256) + (A.E < A.S ? A.E : A.S)) * units;      // at most
  const int grid = 2 * (int)(tiles < pairs ? tiles : pairs);
#define MQ_W8_LAUNCH(SW, GA, T)                                                                                       \
  do {                                                                                                               \
    cudaFuncSetAttribute(w8a8_pair_kernel<SW, GA, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, W_SMEM);          \
    w8a8_pair_kernel<SW, GA, T>                                                                                      \
        <<<grid, (2 + W_EPI + (GA ? W_GATHER : 0)) * 32, W_SMEM, st>>>(map_x, map_w, A, most, d_status);             \
  } while (0)
#define MQ_W8_TYPES(SW, GA)                                            \
  do {                                                                 \
    if (out_dtype == MQ_BF16) MQ_W8_LAUNCH(SW, GA, __nv_bfloat16);     \
    else if (out_dtype == MQ_F16) MQ_W8_LAUNCH(SW, GA, __half);        \
    else MQ_W8_LAUNCH(SW, GA, float);                                  \
  } while (0)
  if (swiglu && gather) MQ_W8_TYPES(true, true);
  else if (swiglu) MQ_W8_TYPES(true, false);
  else if (gather) return MQ_ERR_UNSUPPORTED_SHAPE;
  else MQ_W8_TYPES(false, false);
#undef MQ_W8_TYPES
#undef MQ_W8_LAUNCH
  return check_launch();
}

}  // namespace mq
