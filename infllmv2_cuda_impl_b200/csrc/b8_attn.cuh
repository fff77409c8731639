// What the kernels of the attention over 8-bit blocks share: how a call is dealt to CTAs, the warp that looks blocks up
// and fetches them, and the numbers that the softmax hands to the tensor cores.
//
//   x_tk = log2(e) scale 2^eK(k) q_t . K_k,   out_t = sum_k 2^x_tk 2^eV(k) V_k / sum_k 2^x_tk
//
// over the keys that token t sees.  The codes go to the tensor cores as they lie in memory (kind::f8f6f4): the
// other operand of each product is split into 8-bit numbers instead.
//   * A query row, scaled by a power of two to a largest magnitude of 224..448, is the sum of two e4m3 numbers, to
//     2^-10, that is 2^-17.8 of its largest element or less: for bf16 rows exact down to elements 2^-9.8 of the largest.
//   * For few tokens a weight is the sum of three e5m2 numbers, to 2^-9 of it (half a bf16 step); for several it is an fp16
//     number and the values' codes become fp16 too (b8_chunk.cu).  e5m2 is the upper byte of an fp16
//     number: a term is a byte, what it leaves over one subtraction.  Weights are 2^(x + eV - M) with M about 2^-10 of the
//     largest so far, at most 2^15, and below 2^-16 they have the type's fixed spacing of 2^-16: 2^-27 of the largest.
//     The values' exponents take part in M, so that contributions keep their size against one another whatever
//     the sizes of the blocks' values are.  The sum of the softmax has a reference of its own for several tokens, and for few is
//     held in units of 2^(M - E) with E near the blocks' eV: that of the first unit, until one is more than 2^kHighest above it.
//
// A tile is up to kT tokens of a sequence x the 16 query heads of a KV head.  A CTA takes an even share of the call's
// cost, units of 128 keys plus kStart per tile, whatever the lengths are; pieces of a tile that shares cut go to a workspace
// and are joined by a second kernel.  Where a sequence has one tile per head (a decode step, drafts) every CTA finds
// its share by itself, from the lengths; otherwise a kernel in front lists the tiles.
#pragma once
#include <atomic>
#include <type_traits>
#include "b8.cuh"
#include "beside.cuh"

namespace ifv2 {
namespace b8 {

using namespace tc;

constexpr int kUnit = 2 * kBlockN;               // keys of a step: two blocks
constexpr int kTileBytes = kUnit * kHeadDim;
constexpr int kStart = 2;                        // units that the start of a tile costs
constexpr int kMaxMaskWords = 128;               // 524288 keys
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kUnset = -1e30f;                 // reference of a row that has seen no key
constexpr float kTop = 10.f, kRoom = 15.f;       // a new reference puts the largest weight at 2^kTop; past 2^kRoom it moves
constexpr int kDeepest = -90, kHighest = 60;     // eV - E that the sum's range has room for
constexpr int kNoScale = -10000, kNanScale = 10000;      // eV of no block, of a NaN block

struct AttnParams {
  const __nv_bfloat16* q;
  const uint8_t *k_scale, *v_scale;
  __nv_bfloat16* out;
  float* lse;
  const int32_t *cu_q, *seqlens, *block_table;
  const unsigned long long* mask;                // (heads_k, total_q, words) or null
  const int32_t* lists;                          // (heads_k, total_q, topk) in place of a mask, or null
  int bt_stride, words, topk, batch, heads_k, length, causal;
  int usual;                                     // blocks that a token is taken to select, where it selects
  uint32_t page_mul;                             // a block's page: umulhi(2 block, page_mul) >> page_shift
  int page_shift;
  int64_t total_q, capacity;
  int pages;
  float scale_log2;
  int least_share;
  int32_t* status;                               // [1]: the first kernel that gave a wait up
  // workspace
  int4* join;                                    // cut tiles: first token's row, tokens << 16 | head, first and last share
  int by_tile;                                   // join has a place per tile (where tiles are few), else per share
  float *part_o, *part_lse;                      // two pieces per CTA: (2 grid, 16 kT, 128), (2 grid, 16 kT)
  int most_chunks;                               // listed tiles of a head that the workspace has room for
  int32_t* first_chunk;                          // (batch + 1) chunks of kT tokens before each sequence
  int32_t* first_tile;                           // tile that a CTA begins with; behind these the number of tiles
  int4* tiles;                                   // sequence, row of the first token, keys of the last one, tokens << 16 | head
  int64_t* start;                                // (tiles + 1) cost before each tile
};

// Shares of a cost: CTA g has [begin(g), begin(g + 1)).  Cost: int where the host knows that a call's fits.
template <typename Cost>
struct Shares {
  Cost each, rest;
  int grid;
  __device__ __forceinline__ void deal(Cost cost, int most, int least) {
    grid = cost >= (Cost)most * least ? most : (int)max((uint32_t)cost / (uint32_t)least, 1u);
    each = sizeof(Cost) == 4 ? (Cost)((uint32_t)cost / (uint32_t)grid) : cost / grid;
    rest = cost - each * grid;
  }
  __device__ __forceinline__ Cost begin(int g) const { return each * g + min((Cost)g, rest); }
};

// Tokens of sequence b (cu_q is clamped to the rows there are).
__device__ __forceinline__ int tokens_of(const AttnParams& p, int b, int& row0) {
  row0 = (int)min(max((int64_t)p.cu_q[b], (int64_t)0), p.total_q);
  return max((int)min((int64_t)p.cu_q[b + 1], p.total_q) - row0, 0);
}
__device__ __forceinline__ int keys_of(const AttnParams& p, int b) {
  return (int)min((int64_t)max(p.seqlens[b], 0), p.capacity);
}

// Word w of the union of the masks of `tokens` rows; bits from block `blocks` on are not there.
__device__ __forceinline__ unsigned long long below(unsigned long long word, int w, int blocks) {
  const int left = blocks - w * 64;
  return left >= 64 ? word : left <= 0 ? 0ull : word & ((1ull << left) - 1);
}
__device__ __forceinline__ unsigned long long union_word(const AttnParams& p, int head, int64_t row, int tokens, int w, int blocks) {
  if (w * 64 >= blocks) return 0;
  const unsigned long long* m = p.mask + ((int64_t)head * p.total_q + row) * p.words + w;
  unsigned long long u = 0;
  for (int t = 0; t < tokens; ++t) u |= *(m + (int64_t)t * p.words);
  return below(u, w, blocks);
}

// ------------------------------------------------------------------------ inside a CTA --
// Bit of a unit whose two blocks are whole, seen by all tokens of the tile and not NaN.
constexpr int kPlain = 0x100;

// A block on its way through the CTA: written by the fetching warp, read by the softmax.
struct __align__(16) Block {
  float k_scale;                                   // 2^eK, or NaN
  int e_v;                                         // eV; kNoScale without keys, kNanScale: NaN block
  int valid;                                       // keys (0: the block only fills a unit), and kPlain
  int e_unit[2];                                   // largest eV of the unit's two blocks; in tiles of two tokens, of each one's
  int pos;                                         // position of its first key
  uint32_t tokens;                                 // tokens that attend it
  uint32_t pad;
};
// A CTA's part of a tile.
struct __align__(16) Item {
  int row, head, tokens, reach;                    // first token, KV head, tokens, keys that the last one sees
  int units;                                       // -1: no more items
  int piece;                                       // -1: the whole tile, else the place of a partial result
};

// (the long form stands apart: what is taken every time has to stay in the instruction cache)
static __device__ __noinline__ bool long_wait(uint64_t* bar, uint32_t parity, volatile int* gave_up) {
  if (*gave_up) return false;
  return mbar_wait(bar, parity, gave_up, nullptr, 0);
}
__device__ __forceinline__ bool bounded_wait(uint64_t* bar, uint32_t parity, volatile int* gave_up) {
  return __builtin_expect(mbar_try_wait(bar, parity), 1) ? true : long_wait(bar, parity, gave_up);
}
// All lanes of a warp (the TMEM instructions behind it want them together).
__device__ __forceinline__ bool bounded_wait_warp(uint64_t* bar, uint32_t parity, volatile int* gave_up) {
  return __all_sync(0xFFFFFFFFu, bounded_wait(bar, parity, gave_up));
}

template <int kThreads>
__device__ __forceinline__ void named_sync() { asm volatile("barrier.cta.sync 1, %0;" ::"n"(kThreads) : "memory"); }
template <int kThreads>
__device__ __forceinline__ bool named_any(bool x) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r) : "r"((uint32_t)x), "n"(kThreads) : "memory");
  return r != 0;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 2^e for any e (0 and inf outside the range)
__device__ __forceinline__ float pow2i(int e) { return e < -126 ? 0.f : e > 127 ? INFINITY : __uint_as_float((uint32_t)(e + 127) << 23); }

// Four weights to their three terms, a byte each.  The first two are cut off, the last is rounded.
__device__ __forceinline__ void split4(float a, float b, float c, float d, uint32_t& t0, uint32_t& t1, uint32_t& t2) {
  uint32_t lo, hi;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(d), "f"(c));
  t0 = __byte_perm(lo, hi, 0x7531);
  asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(lo) : "r"(lo & 0xFF00FF00u));
  asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(hi) : "r"(hi & 0xFF00FF00u));
  t1 = __byte_perm(lo, hi, 0x7531);
  asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(lo) : "r"(lo & 0xFF00FF00u));
  asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(hi) : "r"(hi & 0xFF00FF00u));
  t2 = __byte_perm(lo + 0x00800080u, hi + 0x00800080u, 0x7531);
}

// 16 values of a query row, one of 8 neighbouring lanes' parts, to their two terms at `at` and `at + second` (128-byte-
// swizzled rows); returns the factor that scores of the row get.
__device__ __forceinline__ float write_query16(const uint4 (&x)[2], uint8_t* at, int second_at, float scale_log2) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(x);
  uint32_t m2 = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m2 = __vmaxu2(m2, w[j] & 0x7FFF7FFFu);
  uint32_t amax = max(m2 & 0xFFFFu, m2 >> 16);
#pragma unroll
  for (int d = 1; d < 8; d <<= 1) amax = max(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, d));
  const int byte = amax ? scale_byte<kE4m3>(amax << 16) : 127;
  // (a negative scale turns the query round, so that larger products are larger scores)
  const float inv = byte == kNanByte ? 0.f : scale_log2 < 0.f ? -q8::inverse_scale(byte) : q8::inverse_scale(byte);
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
  *reinterpret_cast<uint4*>(at) = make_uint4(first[0], first[1], first[2], first[3]);
  *reinterpret_cast<uint4*>(at + second_at) = make_uint4(second[0], second[1], second[2], second[3]);
  return q8::mul_exact(fabsf(scale_log2), q8::scale_value(byte));      // (may be subnormal, beside a key's 2^120)
}

// Barriers and records that the roles share.
template <int kT, int kStages>
struct Common {
  uint64_t full[kStages], empty[kStages];          // K and V of a unit
  uint64_t item_full[2], item_empty[2];
  Block block[kStages][2];
  Item item[2];
  unsigned long long words[kT][kMaxMaskWords];     // block lists of the tile's tokens as masks
  uint32_t tmem;
  int gave_up;
};

// ---------------------------------------------------------------------- fetching warp --
// Where a CTA's share begins.  It is worked out before the CTA's barriers and tensor memory are there.
// kListed: tiles come from the kernel in front.
template <int kT, bool kListed, bool kSelected>
struct Deal {
  using Cost = typename std::conditional<kListed, int64_t, int>::type;
  Shares<Cost> shares;
  Cost lo = 0x7FFFFFFF, hi = 0, begin = 0;         // of the share; of the tile it begins in
  int b = 0, head = 0, row = 0, tokens = 0, reach = 0, tile = 0, n_tiles = 0;
  int each = 0;                                    // cost of the sequence's heads
  bool more = false;
  // cost of a head of sequence b
  static __device__ __forceinline__ int cost_of(const AttnParams& p, int b, int& row, int& tokens, int& reach) {
    tokens = min(tokens_of(p, b, row), kT);
    reach = keys_of(p, b);
    int n = ceil_div(reach, kUnit);
    if (kSelected) n = min(n, ceil_div(p.usual * (3 + tokens), 8));
    return tokens ? kStart + n : 0;
  }
  __device__ __forceinline__ void begins(Cost cost, const AttnParams& p) {
    const int me = blockIdx.x;
    shares.deal(max(cost, (Cost)1), gridDim.x, p.least_share);
    lo = me < shares.grid ? shares.begin(me) : cost, hi = me < shares.grid ? shares.begin(me + 1) : cost;
    more = lo < hi && cost > 0;                    // (no tile, no item: the list has none to read)
  }
  // A warp's part of the sequences, and the sum of their costs: all warps of the CTA.  (By one warp 256 sequences took eight
  // trips to memory one after the other.)
  static __device__ __forceinline__ int part(const AttnParams& p) { return ceil_div(p.batch, (int)blockDim.x) * 32; }
  static __device__ __forceinline__ void add_up(const AttnParams& p, int* sums) {
    if (kListed) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = part(p), end = min((warp + 1) * n, p.batch);
    int sum = 0;
#pragma unroll 4
    for (int b = warp * n + lane; b < end; b += 32) {
      int r, t, k;
      sum += cost_of(p, b, r, t, k);
    }
    sum = __reduce_add_sync(0xFFFFFFFFu, sum);
    if (lane == 0) sums[warp] = sum * p.heads_k;
  }
  // From these sums the share, and the sequence that it begins in: one warp.
  __device__ __forceinline__ void work_out(const AttnParams& p, const int* sums) {
    const int lane = threadIdx.x & 31;
    if (kListed) {
      n_tiles = p.first_tile[gridDim.x];
      begins((Cost)p.start[n_tiles], p);
      tile = p.first_tile[blockIdx.x];
      return;
    }
    const auto sum_up_to = [&](int x) {
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xFFFFFFFFu, x, d);
        if (lane >= d) x += o;
      }
      return x;
    };
    const int mine = lane < (int)(blockDim.x >> 5) ? sums[lane] : 0, upto_part = sum_up_to(mine);
    begins(__shfl_sync(0xFFFFFFFFu, upto_part, 31), p);
    if (!more) return;
    const int in = __ffs(__ballot_sync(0xFFFFFFFFu, upto_part > (int)lo)) - 1;
    int before = __shfl_sync(0xFFFFFFFFu, upto_part - mine, in);
    for (int base = in * part(p); base < p.batch; base += 32) {
      int r = 0, t = 0, k = 0, c = 0;
      if (base + lane < p.batch) c = cost_of(p, base + lane, r, t, k);
      const int upto = sum_up_to(c * p.heads_k);
      const uint32_t past = __ballot_sync(0xFFFFFFFFu, before + upto > (int)lo);
      if (past) {
        const int src = __ffs(past) - 1;
        b = base + src;
        row = __shfl_sync(0xFFFFFFFFu, r, src);
        tokens = __shfl_sync(0xFFFFFFFFu, t, src);
        reach = __shfl_sync(0xFFFFFFFFu, k, src);
        each = __shfl_sync(0xFFFFFFFFu, c, src);
        before += __shfl_sync(0xFFFFFFFFu, upto, src) - each * p.heads_k;
        head = (int)((uint32_t)((int)lo - before) / (uint32_t)each);
        begin = before + head * each;
        return;
      }
      before += __shfl_sync(0xFFFFFFFFu, upto, 31);
    }
  }
};

// All lanes of a warp run it.
template <int kT, int kStages, bool kListed, bool kSelected>
__device__ __forceinline__ void fetch(const AttnParams& p, const CUtensorMap* k_map, const CUtensorMap* v_map, Common<kT, kStages>& s,
                                      uint8_t* ring, const Deal<kT, kListed, kSelected>& deal) {
  using D = Deal<kT, kListed, kSelected>;
  using Cost = typename D::Cost;
  const int lane = threadIdx.x & 31, me = blockIdx.x;
  volatile int* gave_up = &s.gave_up;
  const Shares<Cost>& shares = deal.shares;
  const Cost lo = deal.lo, hi = deal.hi;
  int b = deal.b, head = deal.head, row = deal.row, tokens = deal.tokens, reach = deal.reach, tile = deal.tile, each = deal.each;
  Cost begin = deal.begin, end = 0;                // of the tile
  bool more = deal.more;
  int4 cut = make_int4(0, 0, 0, 0);                // (first and last share the same: not cut)
  int n = 0, items = 0;                            // units, items so far
  for (bool first = true; more && !*gave_up; first = false) {
    if (kListed) {
      const int4 t = p.tiles[tile];
      b = t.x, row = t.y, reach = t.z, tokens = t.w >> 16, head = t.w & 0xFFFF;
      begin = p.start[tile], end = p.start[tile + 1];
    } else {
      end = begin + each;
    }
    // the part of the tile that lies in this share, in units of the estimate
    const Cost s0 = begin + kStart;
    const int est = (int)(end - s0);
    const int est_a = (int)min(max(lo - s0, (Cost)0), (Cost)est), est_z = (int)min(max(hi - s0, (Cost)est_a), (Cost)est);
    const int blocks = ceil_div(reach, kBlockN);
    // the tile's blocks: all, or those that its tokens select, 4 words of their union per lane
    unsigned long long u[4] = {0, 0, 0, 0};
    int upto = 0, total = blocks;
    const int32_t* list = nullptr;                 // one token's ascending list, walked as it is
    if (kSelected) {
      if (p.lists && tokens == 1) {
        list = p.lists + ((int64_t)head * p.total_q + row) * p.topk;
        bool ascending = true;                     // blocks of the sequence in front, nothing of it behind
        total = 0;
        for (int base = 0; base < p.topk; base += 32) {
          const int i = base + lane;
          const int x = i < p.topk ? *(list + i) : -1, y = i + 1 < p.topk ? *(list + i + 1) : -1;
          const bool valid = x >= 0 && x < blocks, then = y >= 0 && y < blocks;
          ascending &= valid ? !then || y > x : !then;
          total += __popc(__ballot_sync(0xFFFFFFFFu, valid));
        }
        if (!__all_sync(0xFFFFFFFFu, ascending)) list = nullptr;
      }
      if (list == nullptr) {
        if (p.lists) {
          __syncwarp();
          for (int i = lane; i < tokens * kMaxMaskWords; i += 32) s.words[i / kMaxMaskWords][i % kMaxMaskWords] = 0;
          __syncwarp();
          for (int t = 0; t < tokens; ++t) {
            const int32_t* from = p.lists + ((int64_t)head * p.total_q + row + t) * p.topk;
            for (int i = lane; i < p.topk; i += 32) {
              const int block = *(from + i);
              if (block >= 0 && block < blocks)
                atomicOr(reinterpret_cast<uint32_t*>(s.words[t]) + (block >> 5), 1u << (block & 31));
            }
          }
          __syncwarp();
        }
        int count = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int w = 4 * lane + i;
          if (p.lists)
            for (int t = 0; t < tokens; ++t) u[i] |= s.words[t][w];
          else if (w < p.words)
            u[i] = union_word(p, head, row, tokens, w, blocks);
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
    }
    const int units = ceil_div(total, 2);
    // (a tile's cost is an estimate where blocks are selected: parts are in proportion)
    int a = est_a, z = est_z;
    if (kSelected && est != units) {
      a = est ? (int)((int64_t)est_a * units / est) : 0;
      z = est ? (int)((int64_t)est_z * units / est) : 0;
    }
    const bool whole = lo <= begin && hi >= end;
    const bool begins = begin >= lo;               // the tile begins in this share
    if (p.by_tile ? begins : first && me > 0 && !begins && begin >= shares.begin(me - 1)) {
      int last = me;
      while (last + 1 < shares.grid && shares.begin(last + 1) < end) ++last;
      cut = make_int4(row, tokens << 16 | head, p.by_tile ? me : me - 1, last);
      if (p.by_tile && lane == 0) p.join[b * p.heads_k + head] = cut;
    }
    {
      const int slot = items & 1;
      if (!bounded_wait_warp(&s.item_empty[slot], ((items >> 1) & 1) ^ 1, gave_up)) break;
      if (lane == 0) {
        s.item[slot] = Item{row, head, tokens, reach, z - a, whole ? -1 : 2 * me + (lo <= begin ? 1 : 0)};
        mbar_arrive(&s.item_full[slot]);
      }
      // its query rows, 4096 bytes a token, are on their way when the softmax comes to them
      const __nv_bfloat16* q = p.q + ((int64_t)row * p.heads_k + head) * (kGroup * kHeadDim) + lane * 64;
      for (int i = 0; i < tokens; ++i)
        asm volatile("prefetch.global.L1 [%0];" ::"l"(q + (int64_t)i * p.heads_k * (kGroup * kHeadDim)));
      ++items;
    }
    const auto nth_block = [&](int k) {            // all lanes, each with its k
      if (!kSelected) return k;
      if (list) return *(list + k);
      int at = 0;                                  // lane whose words hold it: the first with upto > k
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
      for (int d = 32; d > 0; d >>= 1) {           // its left-th bit
        const int c = __popcll(word & ((1ull << d) - 1));
        if (left >= c) left -= c, word >>= d, block += d;
      }
      return block;
    };
    // 32 blocks at a time, one per lane; the next ones' pages are looked up while these are fetched, their scales behind that
    int block = 0, page = 0;
    const auto look = [&](int k0) {
      block = nth_block(min(k0 + lane, total - 1));
      const int in_table = (int)(__umulhi(2u * (uint32_t)block, p.page_mul) >> p.page_shift);
      page = p.block_table ? *(p.block_table + (int64_t)b * p.bt_stride + in_table) : b;
    };
    int row_of, kb, vb;
    const auto scales = [&]() {
      const bool bad = page < 0 || page >= p.pages;
      const int in_table = p.block_table ? (int)(__umulhi(2u * (uint32_t)block, p.page_mul) >> p.page_shift) : 0;
      const int place = block * kBlockN - in_table * p.length;
      const int r = (int)(((int64_t)(bad ? 0 : page) * p.heads_k + head) * p.length) + place;
      row_of = r;
      kb = bad ? kNanByte : *(p.k_scale + r / kBlockN);
      vb = bad ? kNanByte : *(p.v_scale + r / kBlockN);
    };
    if (z > a) {
      look(2 * a);
      scales();
    }
    for (int k0 = 2 * a; k0 < 2 * z; k0 += 32) {
      const int now = row_of, many = min(32, 2 * (z - a) - (k0 - 2 * a));
      const bool next = k0 + 32 < 2 * z;
      Block r;
      r.pos = block * kBlockN;
      r.valid = k0 + lane < total ? min(kBlockN, reach - r.pos) : 0;
      r.tokens = (1u << tokens) - 1;
      if (kSelected && kT > 1 && !list) {
        r.tokens = 0;
        const unsigned long long* m = p.mask + ((int64_t)head * p.total_q + row) * p.words + (block >> 6);
        for (int i = 0; i < tokens; ++i) {
          const unsigned long long w = p.lists ? s.words[i][block >> 6] : *(m + (int64_t)i * p.words);
          r.tokens |= (uint32_t)((w >> (block & 63)) & 1) << i;
        }
      }
      if (next) look(k0 + 32);
      // A batch's first kStages - 1 units are asked for before their records are written, whose scales may be on their way
      // still.  (Not more: the next one's copies wait for the products of a unit whose record is among these.)
      const int ahead = min(2 * (kStages - 1), many);
#pragma unroll 1
      for (int j = 0; j < many; j += 2, ++n) {
        const int stage = n % kStages;
        if (!bounded_wait_warp(&s.empty[stage], ((n / kStages) & 1) ^ 1, gave_up)) break;
        const int row0 = __shfl_sync(0xFFFFFFFFu, now, j), row1 = __shfl_sync(0xFFFFFFFFu, now, j + 1);
        if (lane == 0) {
          uint8_t* to = ring + stage * 2 * kTileBytes;
          mbar_expect_tx(&s.full[stage], 2 * kTileBytes);
          tma_load_2d(to, k_map, &s.full[stage], 0, row0);
          tma_load_2d(to + kTileBytes / 2, k_map, &s.full[stage], 0, row1);
          tma_load_2d(to + kTileBytes, v_map, &s.full[stage], 0, row0);
          tma_load_2d(to + kTileBytes + kTileBytes / 2, v_map, &s.full[stage], 0, row1);
        }
        if (j + 2 < ahead) continue;
        int u = j;
        if (j + 2 == ahead) {
          u = 0;
          r.k_scale = q8::scale_value(kb);
          r.e_v = r.valid == 0 ? kNoScale : vb == kNanByte ? kNanScale : vb - 127;
          const bool has = r.e_v != kNanScale && r.e_v != kNoScale;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const int e = has && (kT != 2 || ((r.tokens >> t) & 1)) ? r.e_v : kNoScale;
            r.e_unit[t] = max(e, __shfl_xor_sync(0xFFFFFFFFu, e, 1));
          }
          // (all lanes of a pair have the same)
          const bool plain = r.valid == kBlockN && has && r.k_scale == r.k_scale && r.tokens == (1u << tokens) - 1 &&
                             (!p.causal || r.pos + kBlockN <= reach - (tokens - 1));
          const bool both = __shfl_xor_sync(0xFFFFFFFFu, (int)plain, 1) && plain;
          if (both) r.valid |= kPlain;
          if (next) scales();
        }
        for (; u <= j; u += 2) {
          const int of = (n - (j - u) / 2) % kStages;
          if ((lane & ~1) == u) s.block[of][lane & 1] = r;
          __syncwarp();
          if (lane == 0) mbar_arrive(&s.full[of]);
        }
      }
      if (*gave_up) break;
    }
    // the next tile
    if (end >= hi) break;
    if (kListed) {
      ++tile;
      more = tile < deal.n_tiles;
    } else {
      begin = end;
      if (++head == p.heads_k) {
        head = 0;
        do ++b; while (b < p.batch && (each = D::cost_of(p, b, row, tokens, reach)) == 0);
        more = b < p.batch;
      }
    }
  }
  if (!p.by_tile && lane == 0) p.join[me] = cut;
  const int slot = items & 1;
  if (bounded_wait_warp(&s.item_empty[slot], ((items >> 1) & 1) ^ 1, gave_up) && lane == 0) {
    s.item[slot].units = -1;
    mbar_arrive(&s.item_full[slot]);
  }
  __syncwarp();
  if (*gave_up)                                    // copies that are under way land before the CTA ends
    for (int i = max(n - kStages, 0); i < n; ++i) mbar_wait_drain(&s.full[i % kStages], (i / kStages) & 1);
}

// Each kernel of a call may start beside the one in front of it, the first beside whatever is in front of the call.
__device__ __forceinline__ void wait_inputs() {
  wait_previous();
  fence_proxy_async_global();                      // what that one wrote is read by TMA too
}

// The dynamic shared memory of a kernel is allowed once per device.
inline cudaError_t allow_smem(const void* kernel, int bytes, std::atomic<uint64_t>& done) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (device & 63);
  if (device < 64 && (done.load(std::memory_order_relaxed) & bit)) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && device < 64) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

}  // namespace b8

// b8_decode.cu, b8_chunk.cu: enqueue the attention kernel for tiles of at most 1, 2 or 8 tokens.
int b8_launch_few(const CUtensorMap& k_map, const CUtensorMap& v_map, const b8::AttnParams& p, int tokens, int code, cudaStream_t stream);
int b8_launch_chunk(const CUtensorMap& k_map, const CUtensorMap& v_map, const b8::AttnParams& p, bool listed, int code, cudaStream_t stream);
constexpr int kB8FewGrid = 2 * kNumSMs, kB8ChunkGrid = kNumSMs;

}  // namespace ifv2
