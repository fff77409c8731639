// Attention of new tokens over a cache in 8 bits with block scales (b8.cuh).
//
//   x_tk = log2(e) scale 2^eK(k) q_t . K_k,   out_t = sum_k 2^x_tk 2^eV(k) V_k / sum_k 2^x_tk
//
// over the keys that token t sees.  The codes go to the tensor cores as they lie in memory (kind::f8f6f4): the
// other operand of each product is split into 8-bit numbers instead.
//   * A query row, scaled by a power of two to a largest magnitude of 224..448, is the sum of two e4m3 numbers, to
//     2^-10, that is 2^-18 of its largest element: for bf16 rows exact down to elements 2^-10 of the largest.
//   * A weight is the sum of three e5m2 numbers (2^-9 of its value, half a bf16 step; the type's range keeps what is
//     2^-27 of the largest).  Weights carry the values' exponent, w = 2^(x + eV - M), so that the tensor cores
//     add codes, and M follows the largest x + eV: contributions keep their size against one another whatever the
//     sizes of the blocks' values are.  The sum of the softmax is held against mu = M - E, E the largest eV so far.
//
// A tile is kT tokens of a sequence x the 16 query heads of a KV head.  Keys are the M side of both products:
//     S^T (128 keys x 16 kT)   = K . Q^T            both K-major, K in 128-byte-swizzled TMA tiles
//     O^T (128 features x 16 kT) += V^T . W^T       V is MN-major as it lies, W is written [key][column] by the softmax
// so that few query rows cost few tensor clocks, and a softmax thread has a key of its own, with the tile's columns
// in registers: a decode step's exponentials are spread over all lanes.
//
// A CTA (2 per SM) takes an even share of the whole call's cost, units of 128 keys plus kStart per tile, whatever the
// lengths are; pieces of a tile go to a workspace and are joined by a second kernel.  Warps: 0 looks blocks up and
// issues TMA, 1 issues MMAs, 2..5 are the softmax (thread = key = feature).
#include "b8.cuh"

namespace ifv2 {
namespace {

using namespace b8;
using namespace tc;

constexpr int kUnit = 2 * kBlockN;               // keys of a step
constexpr int kTileBytes = kUnit * kHeadDim;
constexpr int kThreads = 192;
constexpr int kMaxGrid = 2 * kNumSMs;
constexpr int kStart = 2;                        // units that the start of a tile costs
constexpr int kMinShare = 3;                     // least cost of a CTA's share
constexpr int kMaxMaskWords = 128;               // 524288 keys
constexpr int kPlanThreads = 1024;
constexpr int kJoinThreads = 128;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kUnset = -1e30f;                 // reference of a column that has seen no key
constexpr float kTop = 10.f, kMost = 32768.f;    // a new reference puts the largest weight at 2^kTop; it moves past kMost
constexpr int kDeepest = -90;                    // eV - E that the sum's range has room for

struct B8AttnParams {
  const __nv_bfloat16* q;
  const uint8_t *k_scale, *v_scale;
  __nv_bfloat16* out;
  float* lse;
  const int32_t *cu_q, *seqlens, *block_table;
  const unsigned long long* mask;
  int bt_stride, words, batch, heads_k, length, causal;
  int64_t total_q, pages;
  float scale_log2;
  int most_chunks;                               // tiles of one head that the workspace has room for
  // workspace
  int32_t* first_chunk;                          // (batch + 1) chunks of kT tokens before each sequence
  int32_t* first_tile;                           // (kMaxGrid) tile that a CTA begins with; behind it, the CTAs that work
  int4* tiles;                                   // sequence, row of the first token, keys of the last one, tokens << 16 | head
  int64_t* start;                                // (tiles + 1) cost before each tile
  float *part_o, *part_lse;                      // two pieces per CTA: (2 grid, 16 kT, 128), (2 grid, 16 kT)
};

__device__ __forceinline__ int grid_share(int64_t cost) {
  return (int)min(max(cost / kMinShare, (int64_t)1), (int64_t)kMaxGrid);
}
__device__ __forceinline__ int64_t share_start(int64_t cost, int g, int grid) { return cost * g / grid; }

// Tokens of sequence b (cu_q is clamped to the rows there are).
__device__ __forceinline__ int tokens_of(const B8AttnParams& p, int b, int& row0) {
  row0 = (int)min(max((int64_t)p.cu_q[b], (int64_t)0), p.total_q);
  return max((int)min((int64_t)p.cu_q[b + 1], p.total_q) - row0, 0);
}

// ------------------------------------------------------------------------------- plan --
// Union of the block masks of `tokens` rows, word w; bits from block `blocks` on are not there.
__device__ __forceinline__ unsigned long long union_word(const B8AttnParams& p, int head, int64_t row, int tokens, int w, int blocks) {
  if (w * 64 >= blocks) return 0;
  const unsigned long long* m = p.mask + ((int64_t)head * p.total_q + row) * p.words + w;
  unsigned long long u = 0;
  for (int t = 0; t < tokens; ++t) u |= __ldg(m + (int64_t)t * p.words);
  return blocks - w * 64 < 64 ? u & ((1ull << (blocks - w * 64)) - 1) : u;
}

template <int kT>
__device__ __forceinline__ int4 tile_of(const B8AttnParams& p, const int32_t* first_chunk, int tile) {
  const int chunk = tile / p.heads_k, head = tile - chunk * p.heads_k;
  int b = 0, row0;                                // largest b with first_chunk[b] <= chunk
  for (int hi = p.batch; hi - b > 1;) {
    const int mid = (b + hi) >> 1;
    if (first_chunk[mid] <= chunk) b = mid; else hi = mid;
  }
  const int n = tokens_of(p, b, row0), t0 = (chunk - first_chunk[b]) * kT, tokens = min(kT, n - t0);
  const int64_t cap = p.block_table ? (int64_t)p.bt_stride * p.length : p.length;
  const int len = (int)min((int64_t)max(p.seqlens[b], 0), cap);
  return make_int4(b, row0 + t0, max(p.causal ? len - n + t0 + tokens : len, 0), tokens << 16 | head);
}

__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* scratch) {      // inclusive, over kPlanThreads
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t o = __shfl_up_sync(0xFFFFFFFFu, v, d);
    if (lane >= d) v += o;
  }
  if (lane == 31) scratch[warp] = v;
  __syncthreads();
  if (warp == 0) {
    int64_t w = scratch[lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t o = __shfl_up_sync(0xFFFFFFFFu, w, d);
      if (lane >= d) w += o;
    }
    scratch[lane] = w;
  }
  __syncthreads();
  if (warp > 0) v += scratch[warp - 1];
  return v;
}

// One CTA: chunks per sequence, tiles and their costs, and where each CTA of the attention begins.
template <int kT>
__global__ void __launch_bounds__(kPlanThreads) b8_plan_kernel(const B8AttnParams p) {
  __shared__ int64_t scratch[32], s_total;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int64_t before = 0;
  for (int base = 0; base < p.batch; base += kPlanThreads) {
    const int b = base + tid;
    int row0;
    const int64_t n = b < p.batch ? ceil_div(tokens_of(p, b, row0), kT) : 0;
    const int64_t upto = before + block_scan(n, scratch);
    if (b < p.batch) p.first_chunk[b] = (int)min(upto - n, (int64_t)p.most_chunks);
    if (tid == kPlanThreads - 1) s_total = upto;
    __syncthreads();
    before = s_total;
    __syncthreads();
  }
  const int chunks = (int)min(before, (int64_t)p.most_chunks);
  if (tid == 0) p.first_chunk[p.batch] = chunks;
  __syncthreads();
  const int tiles = chunks * p.heads_k;
  before = 0;
  for (int base = 0; base < tiles; base += kPlanThreads) {
    const int i = base + tid;
    int64_t cost = 0;
    if (i < tiles) {
      const int4 t = tile_of<kT>(p, p.first_chunk, i);
      p.tiles[i] = t;
      cost = kStart + ceil_div(t.z, kUnit);
    }
    if (p.mask) {                                  // a warp per tile counts its blocks
      __syncthreads();
      for (int j = base + warp; j < min(base + kPlanThreads, tiles); j += kPlanThreads / 32) {
        const int4 t = p.tiles[j];
        const int blocks = ceil_div(t.z, kBlockN);
        int count = 0;
        for (int w = lane; w * 64 < blocks && w < p.words; w += 32)
          count += __popcll(union_word(p, t.w & 0xFFFF, t.y, t.w >> 16, w, blocks));
        count = __reduce_add_sync(0xFFFFFFFFu, count);
        if (lane == 0) p.start[j] = kStart + ceil_div(count, 2);
      }
      __syncthreads();
      if (i < tiles) cost = p.start[i];
      __syncthreads();
    }
    const int64_t upto = before + block_scan(cost, scratch);
    if (i < tiles) p.start[i] = upto - cost;
    if (tid == kPlanThreads - 1) s_total = upto;
    __syncthreads();
    before = s_total;
    __syncthreads();
  }
  if (tid == 0) p.start[tiles] = before;
  __syncthreads();
  const int grid = tiles ? grid_share(before) : 0;
  if (tid == 0) p.first_tile[kMaxGrid] = grid, p.first_tile[kMaxGrid + 1] = tiles;
  for (int g = tid; g < grid; g += kPlanThreads) {
    const int64_t at = share_start(before, g, grid);
    int lo = 0, hi = tiles;                        // start[lo] <= at < start[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (p.start[mid] <= at) lo = mid; else hi = mid;
    }
    p.first_tile[g] = lo;
  }
}

// -------------------------------------------------------------------------- attention --
template <int kT>
struct Shape {
  static constexpr int kN = kGroup * kT;           // columns
  static constexpr int kStages = kT == 1 ? 3 : 2;
  static constexpr int kQBytes = kN * kHeadDim;    // one of two terms
  static constexpr int kPBytes = kN * kUnit;       // one of three terms
  static constexpr int kQ = 0, kP = 2 * kQBytes, kRing = (kP + 3 * kPBytes + 1023) / 1024 * 1024;
  static constexpr int kSmem = kRing + kStages * 2 * kTileBytes + 1024;
  static constexpr int kTmem = kT == 1 ? 64 : kT == 2 ? 128 : 256;
};

// A block on its way through the CTA: written by the producer, read by the softmax.
struct __align__(16) Block {
  float k_scale;                                   // 2^eK, or NaN
  int e_v;                                         // eV, kNanByte: NaN block
  int valid;                                       // keys (0: the block only fills a unit)
  int pos;                                         // position of its first key
  uint32_t tokens;                                 // tokens that attend it
  uint32_t pad[3];
};

__device__ __forceinline__ bool give_up_wait(uint64_t* bar, uint32_t parity, volatile int* gave_up) {
  if (mbar_try_wait(bar, parity)) return true;
  if (*gave_up) return false;
  return mbar_wait(bar, parity, gave_up, nullptr, 0);
}

// All lanes of a warp (the TMEM instructions behind it want them together).
__device__ __forceinline__ bool give_up_wait_warp(uint64_t* bar, uint32_t parity, volatile int* gave_up) {
  return __all_sync(0xFFFFFFFFu, give_up_wait(bar, parity, gave_up));
}

__device__ __forceinline__ void softmax_sync() { asm volatile("barrier.cta.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ bool softmax_any(bool x) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r) : "r"((uint32_t)x) : "memory");
  return r != 0;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 2^e for any e (0 and inf outside the range)
__device__ __forceinline__ float pow2i(int e) { return e < -126 ? 0.f : e > 127 ? INFINITY : __uint_as_float((uint32_t)(e + 127) << 23); }

// Floats as integers of the same order, for redux.
__device__ __forceinline__ int ordered(float x) {
  const int i = __float_as_int(x);
  return i ^ ((i >> 31) & 0x7FFFFFFF);
}
__device__ __forceinline__ float from_ordered(int i) { return __int_as_float(i ^ ((i >> 31) & 0x7FFFFFFF)); }

// Four weights to the three e5m2 terms, a byte each.  e5m2 is the upper half of an fp16 number, so that what a term
// leaves over is one subtraction, without a rounding.
__device__ __forceinline__ void split4(float a, float b, float c, float d, uint32_t (&term)[3]) {
  uint32_t lo, hi;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(d), "f"(c));
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    uint16_t x, y;
    asm("cvt.rn.satfinite.e5m2x2.f16x2 %0, %1;" : "=h"(x) : "r"(lo));
    asm("cvt.rn.satfinite.e5m2x2.f16x2 %0, %1;" : "=h"(y) : "r"(hi));
    term[i] = (uint32_t)x | (uint32_t)y << 16;
    if (i < 2) {
      asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(lo) : "r"(__byte_perm(term[i], 0u, 0x1404)));
      asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(hi) : "r"(__byte_perm(term[i], 0u, 0x3424)));
    }
  }
}

// Column sums over the 32 lanes: v[kN] per lane -> for kN >= 32 columns first .. first + kN / 32 - 1 in v[0 ..] of each lane,
// for 16 column `first` in v[0].  Half the columns go to the other lane in each step.
template <int kN>
__device__ __forceinline__ int column_sums(float (&v)[kN], int lane) {
  int first = 0;
  int n = kN;
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) {
    const bool up = lane & s;
    if (n > 1) {
      n >>= 1;
#pragma unroll
      for (int i = 0; i < kN / 2; ++i) {
        if (i >= n) continue;
        const float mine = up ? v[i + n] : v[i], other = up ? v[i] : v[i + n];
        v[i] = mine + __shfl_xor_sync(0xFFFFFFFFu, other, s);
      }
      if (up) first += n;
    } else {
      v[0] += __shfl_xor_sync(0xFFFFFFFFu, v[0], s);
    }
  }
  return first;
}

template <int kN>
__device__ __forceinline__ void load_columns(uint32_t taddr, uint32_t (&r)[kN]) {
  if constexpr (kN == 16) { tmem_ld16(taddr, r); tmem_wait_ld(); }
  else if constexpr (kN == 32) tmem_ld32_wait(taddr, r);
  else tmem_ld64_wait(taddr, r);
}

template <int kT, int kCode>
__global__ void __launch_bounds__(kThreads, 2)
b8_attn_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const B8AttnParams p) {
  using S = Shape<kT>;
  constexpr int kN = S::kN, kStages = S::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ uint64_t bar_full[kStages], bar_empty[kStages], bar_s[2], bar_sfree[2], bar_p, bar_pv, bar_q, bar_drain;
  __shared__ Block s_block[kStages][2];
  __shared__ float s_c[kN], s_mu[kN], s_fl[kN], s_fo[kN], s_red[4][kN];
  __shared__ uint32_t s_tmem;
  __shared__ int s_gave_up;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int grid = p.first_tile[kMaxGrid];
  if ((int)blockIdx.x >= grid) return;

  if (tid == 0) {
    s_gave_up = 0;
    for (int i = 0; i < kStages; ++i) mbar_init(&bar_full[i], 1), mbar_init(&bar_empty[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&bar_s[i], 1), mbar_init(&bar_sfree[i], 4);
    mbar_init(&bar_p, 4);
    mbar_init(&bar_pv, 1);
    mbar_init(&bar_q, 4);
    mbar_init(&bar_drain, 1);
    fence_barrier_init();
    prefetch_tensormap(&k_map);
    prefetch_tensormap(&v_map);
  }
  if (warp == 1) {
    tmem_alloc(&s_tmem, S::kTmem);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_s = s_tmem, tmem_o = s_tmem + 2 * kN;
  const int tiles = p.first_tile[kMaxGrid + 1];
  const int64_t cost = p.start[tiles], lo = share_start(cost, blockIdx.x, grid), hi = share_start(cost, blockIdx.x + 1, grid);
  const int tile0 = p.first_tile[blockIdx.x];
  // units [a, z) of a tile that lie in this CTA's share
  const auto units = [&](int tile, int& a, int& z) {
    const int64_t s = p.start[tile] + kStart;
    a = (int)max(lo - s, (int64_t)0);
    z = max((int)min(hi - s, p.start[tile + 1] - s), a);
  };

  if (warp == 0) {
    // ---------------------------------------------------------------- producer
    int n = 0;                                     // units so far
    for (int tile = tile0; tile < tiles && p.start[tile] < hi && !s_gave_up; ++tile) {
      const int4 t = p.tiles[tile];
      const int b = t.x, head = t.w & 0xFFFF, tokens = t.w >> 16, blocks = ceil_div(t.z, kBlockN);
      int a, z;
      units(tile, a, z);
      if (a == z) continue;
      // the tile's blocks: all, or those of the union of its tokens' masks, 4 words of it per lane
      unsigned long long u[4] = {0, 0, 0, 0};
      int upto = 0, total = blocks;
      if (p.mask) {
        int count = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int w = 4 * lane + i;
          if (w < p.words) u[i] = union_word(p, head, t.y, tokens, w, blocks);
          count += __popcll(u[i]);
        }
        upto = count;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int o = __shfl_up_sync(0xFFFFFFFFu, upto, d);
          if (lane >= d) upto += o;
        }
        total = __shfl_sync(0xFFFFFFFFu, upto, 31);
      }
      const auto nth_block = [&](int k) {          // all lanes, each with its k
        if (!p.mask) return k;
        int at = 0;                                // lane whose words hold it: first with upto > k
#pragma unroll
        for (int d = 16; d > 0; d >>= 1)
          if (__shfl_sync(0xFFFFFFFFu, upto, (at + d - 1) & 31) <= k) at += d;
        at &= 31;
        const int before = __shfl_sync(0xFFFFFFFFu, upto, (at + 31) & 31);
        int left = k - (at ? before : 0), block = 256 * at;
        unsigned long long word = 0;
        bool found = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const unsigned long long w = __shfl_sync(0xFFFFFFFFu, u[i], at);
          const int c = __popcll(w);
          if (!found) {
            if (left < c) found = true, word = w;
            else left -= c, block += 64;
          }
        }
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) {         // its left-th bit
          const int c = __popcll(word & ((1ull << d) - 1));
          if (left >= c) left -= c, word >>= d, block += d;
        }
        return block;
      };
      const auto page_of = [&](int block) {
        const int64_t pos = (int64_t)block * kBlockN;
        return p.block_table ? __ldg(p.block_table + (int64_t)b * p.bt_stride + pos / p.length) : b;
      };
      for (int k0 = 2 * a; k0 < 2 * z; k0 += 32) { // 32 blocks at a time, one per lane
        const int k = k0 + lane;
        const bool there = k < total;
        const int block = nth_block(there ? k : total - 1);
        const int page = page_of(block);
        const bool bad = page < 0 || page >= p.pages;
        const int place = p.block_table ? (block * kBlockN) % p.length : block * kBlockN;
        const int64_t row = ((int64_t)(bad ? 0 : page) * p.heads_k + head) * p.length + place;
        Block r;
        r.pos = block * kBlockN;
        r.valid = there ? min(kBlockN, t.z - r.pos) : 0;
        const int kb = bad ? kNanByte : __ldg(p.k_scale + row / kBlockN), vb = bad ? kNanByte : __ldg(p.v_scale + row / kBlockN);
        r.k_scale = q8::scale_value(kb);
        r.e_v = vb == kNanByte ? kNanByte : vb - 127;
        r.tokens = (1u << tokens) - 1;
        if (p.mask && kT > 1) {
          r.tokens = 0;
          const unsigned long long* m = p.mask + ((int64_t)head * p.total_q + t.y) * p.words + (block >> 6);
          for (int i = 0; i < tokens; ++i) r.tokens |= (uint32_t)((__ldg(m + (int64_t)i * p.words) >> (block & 63)) & 1) << i;
        }
        for (int j = 0; j < min(32, 2 * z - k0); j += 2, ++n) {
          const int stage = n % kStages;
          if (!give_up_wait_warp(&bar_empty[stage], ((n / kStages) & 1) ^ 1, &s_gave_up)) break;
          if ((lane & ~1) == j) s_block[stage][lane & 1] = r;
          const int row0 = (int)__shfl_sync(0xFFFFFFFFu, row, j), row1 = (int)__shfl_sync(0xFFFFFFFFu, row, j + 1);
          __syncwarp();
          if (lane == 0) {
            uint8_t* kt = smem + S::kRing + stage * 2 * kTileBytes;
            mbar_expect_tx(&bar_full[stage], 2 * kTileBytes);
            tma_load_2d(kt, &k_map, &bar_full[stage], 0, row0);
            tma_load_2d(kt + kTileBytes / 2, &k_map, &bar_full[stage], 0, row1);
            tma_load_2d(kt + kTileBytes, &v_map, &bar_full[stage], 0, row0);
            tma_load_2d(kt + kTileBytes + kTileBytes / 2, &v_map, &bar_full[stage], 0, row1);
          }
        }
        if (*(volatile int*)&s_gave_up) break;
      }
    }
    if (*(volatile int*)&s_gave_up)                // copies that are under way land before the CTA ends
      for (int i = max(n - kStages, 0); i < n; ++i) mbar_wait_drain(&bar_full[i % kStages], (i / kStages) & 1);
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMAs
    if (elect_one()) {
      const uint32_t base = smem_u32(smem);
      constexpr uint32_t kIdescS = umma_idesc_f8(128, kN, kCode, kE4m3, false, false);
      constexpr uint32_t kIdescO = umma_idesc_f8(128, kN, kCode, kE5m2, true, true);
      bool ok = true;
      int n = 0, item = 0;
      const auto values = [&](int unit, bool first) {        // O += W V of a unit
        const int stage = unit % kStages;
        ok = ok && give_up_wait(&bar_p, unit & 1, &s_gave_up);
        if (!ok) return;
        tc_fence_after();
        const uint32_t v = base + S::kRing + stage * 2 * kTileBytes + kTileBytes;
#pragma unroll
        for (int i = 0; i < 3; ++i)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            umma_f8_ss(tmem_o, umma_desc_sw128(v + kk * 4096, 16, 1024),
                       umma_desc_noswz_mn8(base + S::kP + i * S::kPBytes + kk * 512, 16 * kUnit), kIdescO, !first || i + kk > 0);
        umma_commit(&bar_empty[stage]);
        umma_commit(&bar_pv);
      };
      for (int tile = tile0; ok && tile < tiles && p.start[tile] < hi; ++tile) {
        int a, z;
        units(tile, a, z);
        if (a == z) continue;
        ok = ok && give_up_wait(&bar_q, item & 1, &s_gave_up);
        for (int i = a; ok && i < z; ++i, ++n) {
          const int stage = n % kStages;
          ok = give_up_wait(&bar_full[stage], (n / kStages) & 1, &s_gave_up) &&
               give_up_wait(&bar_sfree[n & 1], ((n >> 1) & 1) ^ 1, &s_gave_up);
          if (!ok) break;
          tc_fence_after();
          const uint32_t k = base + S::kRing + stage * 2 * kTileBytes;
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              umma_f8_ss(tmem_s + (n & 1) * kN, umma_desc_sw128(k + kk * 32, 16, 1024),
                         umma_desc_sw128(base + S::kQ + j * S::kQBytes + kk * 32, 16, 1024), kIdescS, j + kk > 0);
          umma_commit(&bar_s[n & 1]);
          if (i > a) values(n - 1, i - 1 == a);
        }
        values(n - 1, z - 1 == a);
        ++item;
      }
      if (!ok) {
        umma_commit(&bar_drain);
        mbar_wait_drain(&bar_drain, 0);
      }
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- softmax
    // A wait that gave up only makes the results NaN: every thread keeps to the same loops and barriers.
    const int quad = warp & 3, r = quad * 32 + lane;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const int stid = tid - 64;
    const int heads = p.heads_k * kGroup;

    // Query rows of a tile: 8 threads per row, 16 values each.
    const auto write_query = [&](const int4& t) {
      const int head = t.w & 0xFFFF, tokens = t.w >> 16;
#pragma unroll
      for (int i = 0; i < kT; ++i) {
        const int col = i * 16 + (stid >> 3), c = stid & 7;
        uint4 x[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
        if (i < tokens) {
          const uint4* src = reinterpret_cast<const uint4*>(p.q + ((int64_t)(t.y + i) * heads + head * kGroup + (stid >> 3)) * kHeadDim + c * 16);
          x[0] = __ldg(src);
          x[1] = __ldg(src + 1);
        }
        const uint32_t* w = reinterpret_cast<const uint32_t*>(x);
        uint32_t m2 = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m2 = __vmaxu2(m2, w[j] & 0x7FFF7FFFu);
        uint32_t amax = max(m2 & 0xFFFFu, m2 >> 16);
#pragma unroll
        for (int d = 1; d < 8; d <<= 1) amax = max(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, d));
        const int byte = scale_byte<kE4m3>(amax << 16);
        const float inv = byte == kNanByte ? 0.f : q8::inverse_scale(byte);
        uint32_t first[4], second[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float y[4] = {__uint_as_float(w[2 * j] << 16), __uint_as_float(w[2 * j] & 0xFFFF0000u),
                        __uint_as_float(w[2 * j + 1] << 16), __uint_as_float(w[2 * j + 1] & 0xFFFF0000u)}, near[4];
          if (byte == kNanByte) y[0] = y[1] = y[2] = y[3] = 0.f;
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = q8::mul_exact(y[e], inv);
          first[j] = encode4<kE4m3>(y, 1.f);
          decode4<kE4m3>(near, first[j]);
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] -= near[e];
          second[j] = encode4<kE4m3>(y, 1.f);
        }
        uint8_t* at = smem + S::kQ + col * kHeadDim + ((c ^ (col & 7)) << 4);
        *reinterpret_cast<uint4*>(at) = make_uint4(first[0], first[1], first[2], first[3]);
        *reinterpret_cast<uint4*>(at + S::kQBytes) = make_uint4(second[0], second[1], second[2], second[3]);
        if (c == 0) s_c[col] = p.scale_log2 * q8::scale_value(byte);
      }
      fence_proxy_async_smem();
      mbar_arrive_warp(&bar_q);
      softmax_sync();
    };

    // the first tile from `tile` on that has units in this share (the issuing warp skips the others too)
    const auto next_query = [&](int tile) {
      for (; tile < tiles && p.start[tile] < hi; ++tile) {
        int a, z;
        units(tile, a, z);
        if (z > a) {
          write_query(p.tiles[tile]);
          return;
        }
      }
    };
    int n = 0;
    next_query(tile0);
    for (int tile = tile0; tile < tiles && p.start[tile] < hi; ++tile) {
      const int4 t = p.tiles[tile];
      const int tokens = t.w >> 16;
      int a, z;
      units(tile, a, z);
      float l[kN];
#pragma unroll
      for (int i = 0; i < kN; ++i) l[i] = 0.f;
      if (stid < kN) s_mu[stid] = kUnset;
      softmax_sync();
      int e_ref = -10000, deepest = 0;             // E; least eV - E of the blocks so far
      for (int i = a; i < z; ++i, ++n) {
        const int stage = n % kStages;
        give_up_wait_warp(&bar_full[stage], (n / kStages) & 1, &s_gave_up);
        give_up_wait_warp(&bar_s[n & 1], (n >> 1) & 1, &s_gave_up);
        tc_fence_after();
        uint32_t x[kN];
        load_columns<kN>(tmem_s + (n & 1) * kN + lanes, x);
        tc_fence_before();
        mbar_arrive_warp(&bar_sfree[n & 1]);
        const Block mine = s_block[stage][r >> 6], other = s_block[stage][(r >> 6) ^ 1];
        const int e_mine = mine.valid > 0 && mine.e_v != kNanByte ? mine.e_v : -10000;
        const int e_other = other.valid > 0 && other.e_v != kNanByte ? other.e_v : -10000;
        const int e_new = max(e_ref, max(e_mine, e_other));
        const int in_block = r & 63;
        const bool here = in_block < mine.valid;
        // keys that token i sees end at position t.z - (tokens - 1 - i) if causal, t.z otherwise
        const int reach = t.z - (mine.pos + in_block);         // > 0: the last token sees this key
        const auto sees = [&](int tok) {
          return here && ((mine.tokens >> tok) & 1) && (p.causal ? reach > tokens - 1 - tok : reach > 0);
        };
        const int dv = mine.e_v - e_new;                       // (of no interest without a key or in a NaN block)
        const float v_scale = mine.e_v == kNanByte ? NAN : pow2i(dv), v_ref = pow2i(max(min(dv, 0), kDeepest));
        float w[kN];
        const auto weights = [&]() {
          float most = 0.f;
#pragma unroll
          for (int tok = 0; tok < kT; ++tok) {
            const bool see = sees(tok);
#pragma unroll
            for (int g = 0; g < kGroup; ++g) {
              const int c = tok * kGroup + g;
              const float y = ex2(fmaf(__uint_as_float(x[c]), s_c[c] * mine.k_scale, -s_mu[c]));
              w[c] = see ? y : 0.f;
              most = fmaxf(most, w[c]);
            }
          }
          return most;
        };
        bool moves = e_new != e_ref;
        if (!moves) moves = softmax_any(weights() * v_ref > kMost);
        if (moves) {
          // new references: the largest x + eV of each column, and E
          const int delta = i == a || e_ref == -10000 ? 0 : e_new - e_ref;
          const int bump = i == a ? 0 : max(kDeepest - (deepest - delta), 0);
          deepest = i == a ? 0 : max(deepest - delta, kDeepest);
          if (e_mine > -10000) deepest = max(min(deepest, e_mine - e_new), kDeepest);
          if (e_other > -10000) deepest = max(min(deepest, e_other - e_new), kDeepest);
          const float up = (float)max(min(dv, 0), kDeepest);
#pragma unroll
          for (int tok = 0; tok < kT; ++tok) {
            const bool see = sees(tok);
#pragma unroll
            for (int g = 0; g < kGroup; ++g) {
              const int c = tok * kGroup + g;
              float y = fmaf(__uint_as_float(x[c]), s_c[c] * mine.k_scale, up);
              if (!see || !(y == y)) y = -INFINITY;
              const int top = __reduce_max_sync(0xFFFFFFFFu, ordered(y));
              if (lane == 0) s_red[quad][c] = from_ordered(top);
            }
          }
          softmax_sync();
          if (stid < kN) {
            const float top = fmaxf(fmaxf(s_red[0][stid], s_red[1][stid]), fmaxf(s_red[2][stid], s_red[3][stid]));
            const float mu = s_mu[stid];
            float mu_new = mu, fl = 1.f, fo = 1.f;
            if (mu == kUnset) {
              if (top > -INFINITY) mu_new = top - kTop;
              fl = fo = 0.f;
            } else {
              mu_new = mu + (float)(bump - delta);
              if (top - mu_new > 15.f) mu_new = top - kTop;
              fl = ex2(mu - mu_new);
              fo = ex2(mu - mu_new - (float)delta);
            }
            s_mu[stid] = mu_new;
            s_fl[stid] = fl;
            s_fo[stid] = fo;
          }
          softmax_sync();
#pragma unroll
          for (int c = 0; c < kN; ++c) l[c] = l[c] > 0.f ? l[c] * s_fl[c] : l[c];
          if (i > a) {                             // what is in O so far
            give_up_wait_warp(&bar_pv, (n - 1) & 1, &s_gave_up);
            tc_fence_after();
#pragma unroll
            for (int c0 = 0; c0 < kN; c0 += 16) {
              uint32_t o[16];
              tmem_ld16(tmem_o + lanes + c0, o);
              tmem_wait_ld();
#pragma unroll
              for (int c = 0; c < 16; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * s_fo[c0 + c]);
              tmem_st16(tmem_o + lanes + c0, o);
            }
            tmem_wait_st();
            tc_fence_before();
          }
          e_ref = e_new;
          weights();
        } else {
          if (e_mine > -10000) deepest = max(min(deepest, e_mine - e_ref), kDeepest);
          if (e_other > -10000) deepest = max(min(deepest, e_other - e_ref), kDeepest);
        }
        // the one buffer of weights is free again when the product before has been made
        if (n > 0) give_up_wait_warp(&bar_pv, (n - 1) & 1, &s_gave_up);
#pragma unroll
        for (int tok = 0; tok < kT; ++tok) {
          const bool see = sees(tok);
          uint32_t out[3][4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int c = tok * kGroup + 4 * j + e;
              l[c] += w[c];
              y[e] = see ? w[c] * v_scale : 0.f;
            }
            uint32_t term[3];
            split4(y[0], y[1], y[2], y[3], term);
            out[0][j] = term[0];
            out[1][j] = term[1];
            out[2][j] = term[2];
          }
#pragma unroll
          for (int k = 0; k < 3; ++k)
            *reinterpret_cast<uint4*>(smem + S::kP + k * S::kPBytes + tok * 16 * kUnit + r * 16) =
                make_uint4(out[k][0], out[k][1], out[k][2], out[k][3]);
        }
        if (!here) {                               // a value row that is no key may hold anything: 0 x NaN
          uint4* row = reinterpret_cast<uint4*>(smem + S::kRing + stage * 2 * kTileBytes + kTileBytes + r * kHeadDim);
#pragma unroll
          for (int j = 0; j < 8; ++j) row[j] = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        mbar_arrive_warp(&bar_p);
      }
      // the next tile's query, while the last product runs
      softmax_sync();
      if (z > a) next_query(tile + 1);

      // ---- the tile's results
      const bool whole = lo <= p.start[tile] && hi >= p.start[tile + 1];
      const int piece = 2 * blockIdx.x + (lo <= p.start[tile] ? 1 : 0);
      const int first = column_sums<kN>(l, lane);
      if (kN >= 32) {
#pragma unroll
        for (int j = 0; j < kN / 32; ++j) s_red[quad][first + j] = l[j];
      } else {
        s_red[quad][first] = l[0];                 // (two lanes, one value)
      }
      softmax_sync();
      if (z > a) give_up_wait_warp(&bar_pv, (n - 1) & 1, &s_gave_up);
      tc_fence_after();
      if (stid < kN) {
        const float sum = s_red[0][stid] + s_red[1][stid] + s_red[2][stid] + s_red[3][stid];
        const bool none = sum == 0.f;
        float l2;
        asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(l2) : "f"(sum));
        const float lse2 = none ? -INFINITY : s_mu[stid] + l2;
        s_fl[stid] = none ? 0.f : 1.f / sum;
        const int tok = stid / kGroup;
        if (whole) {
          if (p.lse && tok < tokens) p.lse[(int64_t)(t.y + tok) * heads + (t.w & 0xFFFF) * kGroup + stid % kGroup] = none ? INFINITY : lse2 * kLn2;
        } else {
          p.part_lse[(int64_t)piece * kN + stid] = lse2;
        }
      }
      softmax_sync();
      const float e_half = pow2i(e_ref > -10000 ? e_ref / 2 : 0), e_rest = pow2i(e_ref > -10000 ? e_ref - e_ref / 2 : 0);
#pragma unroll
      for (int c0 = 0; c0 < kN; c0 += 16) {
        uint32_t o[16];
        if (z > a) {
          tmem_ld16(tmem_o + lanes + c0, o);
          tmem_wait_ld();
        }
        if (c0 / kGroup >= tokens) continue;
        const bool lost = *(volatile int*)&s_gave_up;
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          float y = 0.f;
          if (z > a && s_fl[c0 + c] != 0.f) y = q8::mul_exact(q8::mul_exact(__uint_as_float(o[c]) * s_fl[c0 + c], e_half), e_rest);
          if (lost) y = NAN;
          if (whole) p.out[((int64_t)(t.y + c0 / kGroup) * heads + (t.w & 0xFFFF) * kGroup + c) * kHeadDim + r] = __float2bfloat16(y);
          else p.part_o[((int64_t)piece * kN + c0 + c) * kHeadDim + r] = y;
        }
      }
      tc_fence_before();
      softmax_sync();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(s_tmem, S::kTmem);
}

// ------------------------------------------------------------------------------- join --
// The pieces of a tile that shares cut: CTA x of the grid has the tile that share x begins inside, if no earlier share
// does.  A CTA takes 4 of a token's heads.  Also: rows behind the last sequence.
template <int kT>
__global__ void __launch_bounds__(kJoinThreads) b8_join_kernel(const B8AttnParams p) {
  constexpr int kN = kGroup * kT;
  const int tid = threadIdx.x, heads = p.heads_k * kGroup;
  {
    const int64_t row0 = min(max((int64_t)p.cu_q[p.batch], (int64_t)0), p.total_q);
    const int64_t me = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * kJoinThreads + tid, all = (int64_t)gridDim.x * gridDim.y * kJoinThreads;
    uint4* out = reinterpret_cast<uint4*>(p.out);
    for (int64_t i = row0 * heads * 16 + me; i < p.total_q * heads * 16; i += all) out[i] = make_uint4(0, 0, 0, 0);
    if (p.lse)
      for (int64_t i = row0 * heads + me; i < p.total_q * heads; i += all) p.lse[i] = INFINITY;
  }
  const int grid = p.first_tile[kMaxGrid], g = blockIdx.x;
  if (g == 0 || g >= grid) return;
  const int tiles = p.first_tile[kMaxGrid + 1], tile = p.first_tile[g];
  const int64_t cost = p.start[tiles], begin = p.start[tile], end = p.start[tile + 1];
  if (begin >= share_start(cost, g, grid) || begin < share_start(cost, g - 1, grid)) return;
  const int4 t = p.tiles[tile];
  const int tok = blockIdx.y >> 2, col = tok * kGroup + (blockIdx.y & 3) * 4 + (tid >> 5), lane = tid & 31;
  if (tok >= (t.w >> 16)) return;
  // pieces: the second of CTA g - 1, the first of g, g + 1, ...
  int last = g;
  while (last + 1 < grid && share_start(cost, last + 1, grid) < end) ++last;
  const auto piece = [&](int i) { return i < g ? 2 * i + 1 : 2 * i; };
  float most = -INFINITY, nan = 0.f;
  for (int i = g - 1; i <= last; ++i) {
    const float x = p.part_lse[(int64_t)piece(i) * kN + col];
    most = fmaxf(most, x);
    if (!(x == x)) nan = x;
  }
  float sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = g - 1; i <= last; ++i) {
    const float x = p.part_lse[(int64_t)piece(i) * kN + col];
    if (x > -INFINITY) {
      const float f = ex2(x - most);
      const float4 o = reinterpret_cast<const float4*>(p.part_o + ((int64_t)piece(i) * kN + col) * kHeadDim)[lane];
      sum += f;
      acc.x += f * o.x, acc.y += f * o.y, acc.z += f * o.z, acc.w += f * o.w;
    }
  }
  const bool none = most == -INFINITY;
  const float inv = none ? nan : 1.f / sum + nan;
  const int64_t row = (int64_t)(t.y + tok) * heads + (t.w & 0xFFFF) * kGroup + (col & 15);
  uint2 y;
  y.x = pack_bf16(acc.x * inv, acc.y * inv);
  y.y = pack_bf16(acc.z * inv, acc.w * inv);
  reinterpret_cast<uint2*>(p.out + row * kHeadDim)[lane] = y;
  if (p.lse && lane == 0) {
    float l2;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(l2) : "f"(sum));
    p.lse[row] = nan != nan ? nan : none ? INFINITY : (most + l2) * kLn2;
  }
}

// ------------------------------------------------------------------------------- host --
int tokens_per_tile(int max_seqlen_q) { return max_seqlen_q <= 1 ? 1 : max_seqlen_q == 2 ? 2 : 4; }

struct Layout {
  int64_t chunks, tiles_at, start_at, chunk_at, first_at, lse_at, o_at, bytes;
  Layout(int64_t total_q, int batch, int heads_k, int t) {
    const auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
    chunks = ceil_div64(total_q, t) + batch;
    tiles_at = 0;
    start_at = up(tiles_at + 16 * chunks * heads_k);
    chunk_at = up(start_at + 8 * (chunks * heads_k + 1));
    first_at = up(chunk_at + 4 * ((int64_t)batch + 1));
    lse_at = up(first_at + 4 * (kMaxGrid + 2));
    o_at = up(lse_at + 4 * (2 * kMaxGrid) * kGroup * t);
    bytes = o_at + 4ll * (2 * kMaxGrid) * kGroup * t * kHeadDim;
  }
};

template <int kT, int kCode>
int launch(const CUtensorMap& k_map, const CUtensorMap& v_map, const B8AttnParams& p, cudaStream_t stream) {
  constexpr int smem = Shape<kT>::kSmem;
  const cudaError_t e = cudaFuncSetAttribute(b8_attn_kernel<kT, kCode>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return set_error((int)e, "b8_attn: %s", cudaGetErrorString(e));
  b8_plan_kernel<kT><<<1, kPlanThreads, 0, stream>>>(p);
  if (int rc = check_launch("b8_attn (plan)")) return rc;
  b8_attn_kernel<kT, kCode><<<kMaxGrid, kThreads, smem, stream>>>(k_map, v_map, p);
  if (int rc = check_launch("b8_attn")) return rc;
  b8_join_kernel<kT><<<dim3(kMaxGrid, 4 * kT), kJoinThreads, 0, stream>>>(p);
  return check_launch("b8_attn (join)");
}

}  // namespace
}  // namespace ifv2

using namespace ifv2;

extern "C" int64_t ifv2_b8_attn_workspace_bytes(int64_t total_q, int batch, int heads_q, int head_dim, int max_seqlen_q) {
  if (total_q < 0 || batch < 0 || heads_q < 0 || head_dim != kHeadDim) return 0;
  return Layout(total_q, batch, heads_q / kGroup, tokens_per_tile(max_seqlen_q)).bytes;
}

extern "C" int ifv2_b8_attn(const void* q, const void* k_cache, const void* v_cache, const void* k_scale, const void* v_scale,
                            void* out, float* lse, const int32_t* cu_seqlens_q, const int32_t* cache_seqlens,
                            const int32_t* block_table, int block_table_stride, const int64_t* mask, int mask_words, int batch,
                            int64_t total_q, int max_seqlen_q, int64_t num_pages, int64_t length, int code, int heads_q, int heads_k,
                            int head_dim, float softmax_scale, int causal, void* workspace, int64_t workspace_bytes, void* stream) {
  IFV2_REQUIRE(head_dim == kHeadDim && heads_k >= 1 && heads_q == heads_k * kGroup, IFV2_ERR_UNSUPPORTED,
               "b8_attn: head_dim must be %d, with %d query heads per KV head", kHeadDim, kGroup);
  IFV2_REQUIRE(code == kE4m3 || code == kE5m2, IFV2_ERR_INVALID_ARG, "b8_attn: code must be 0 (e4m3) or 1 (e5m2)");
  IFV2_REQUIRE(batch >= 0 && total_q >= 0 && max_seqlen_q >= 0 && num_pages >= 0 && length >= kBlockN && length % kBlockN == 0 &&
               mask_words >= 0 && (block_table == nullptr || block_table_stride >= 1), IFV2_ERR_INVALID_ARG, "b8_attn: bad sizes");
  if (total_q == 0) return IFV2_OK;
  IFV2_REQUIRE(batch >= 1 && q && out && cu_seqlens_q && cache_seqlens && (num_pages == 0 || (k_cache && v_cache && k_scale && v_scale)) &&
               workspace, IFV2_ERR_INVALID_ARG, "b8_attn: null pointer");
  const int64_t cap = block_table ? (int64_t)block_table_stride * length : length;
  IFV2_REQUIRE(num_pages >= 1 && (block_table || num_pages >= batch), IFV2_ERR_INVALID_ARG, "b8_attn: the cache has too few pages");
  IFV2_REQUIRE(heads_k < 32768 && total_q < (1ll << 31) && cap < (1ll << 31) && num_pages * length * heads_k < (1ll << 31),
               IFV2_ERR_TOO_LARGE, "b8_attn: rows of the queries, of a sequence and of the cache must be below 2^31");
  IFV2_REQUIRE(mask == nullptr || mask_words == ceil_div64(cap, 64 * kBlockN), IFV2_ERR_INVALID_ARG,
               "b8_attn: mask rows must have a word per 64 blocks of the capacity");
  IFV2_REQUIRE(mask == nullptr || mask_words <= kMaxMaskWords, IFV2_ERR_TOO_LARGE, "b8_attn: masks over at most %d keys",
               kMaxMaskWords * 64 * kBlockN);
  const int t = tokens_per_tile(max_seqlen_q);
  const Layout at(total_q, batch, heads_k, t);
  IFV2_REQUIRE(at.chunks * heads_k < (1ll << 31), IFV2_ERR_TOO_LARGE, "b8_attn: too many tiles");
  IFV2_REQUIRE(workspace_bytes >= at.bytes, IFV2_ERR_INVALID_ARG, "b8_attn: the workspace is too small");
  IFV2_REQUIRE(((reinterpret_cast<uintptr_t>(workspace) | reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) == 0,
               IFV2_ERR_INVALID_ARG, "b8_attn: q, out and the workspace must begin at multiples of 16 bytes");
  CUtensorMap k_map, v_map;
  const uint64_t rows = (uint64_t)num_pages * heads_k * length;
  int rc = make_tensor_map_rows128(&k_map, k_cache, rows, kBlockN);
  if (rc == IFV2_OK) rc = make_tensor_map_rows128(&v_map, v_cache, rows, kBlockN);
  if (rc != IFV2_OK) return rc;
  char* ws = static_cast<char*>(workspace);
  B8AttnParams p{static_cast<const __nv_bfloat16*>(q), static_cast<const uint8_t*>(k_scale), static_cast<const uint8_t*>(v_scale),
                 static_cast<__nv_bfloat16*>(out), lse, cu_seqlens_q, cache_seqlens, block_table,
                 reinterpret_cast<const unsigned long long*>(mask), block_table_stride, mask_words, batch, heads_k, (int)length, causal,
                 total_q, num_pages, softmax_scale * kLog2e, (int)at.chunks, reinterpret_cast<int32_t*>(ws + at.chunk_at),
                 reinterpret_cast<int32_t*>(ws + at.first_at), reinterpret_cast<int4*>(ws + at.tiles_at),
                 reinterpret_cast<int64_t*>(ws + at.start_at), reinterpret_cast<float*>(ws + at.o_at), reinterpret_cast<float*>(ws + at.lse_at)};
  cudaStream_t s = (cudaStream_t)stream;
#define IFV2_B8(T) (code == kE4m3 ? launch<T, kE4m3>(k_map, v_map, p, s) : launch<T, kE5m2>(k_map, v_map, p, s))
  return t == 1 ? IFV2_B8(1) : t == 2 ? IFV2_B8(2) : IFV2_B8(4);
#undef IFV2_B8
}
