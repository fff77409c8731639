// One new token per sequence over a key-value cache in 8 bits (formulas of the codes: q8.cuh).
//
//   s_t = scale * q . K_t * 2^eK(t),  m = max s,  l = sum exp(s_t - m),  out = sum exp(s_t - m) 2^eV(t) V_t / l
//
// over the positions of the sequence, or those of the 64-key blocks that its mask row selects.  The keys are shared
// by 16 query heads, split over CTAs, and the partial (m, l, M, O) of the splits are joined by a second kernel.
//
// O is a sum over codes, O = sum 2^(z_t - M) V_t with z_t = log2(e) s_t + eV(t) and M about max z: the exponents of the
// values take part in the weights, next to the scores, so that the largest weight is about 1 whatever the values' sizes
// are, and out = O 2^(M - m) / l.  (m and M differ by little more than 127, the range of the exponents.)
//
// Launches: [prepare: long block lists, append where sequences may share rows] -> split -> combine.
#include <type_traits>
#include "beside.cuh"
#include "block_list.cuh"
#include "mma_sync.cuh"
#include "q8.cuh"
#include "rotary.cuh"
#include "tc05.cuh"

namespace ifv2 {
namespace {

using namespace q8;

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kResident = 3;                     // CTAs per SM
constexpr int kUnit = 32;                        // keys that a warp handles at once
constexpr int kSlots = 3;                        // a warp's tiles in shared memory: K, V, next K, next V ... in turn
constexpr int kTileBytes = kUnit * kHeadDim;
constexpr int kSmemBytes = kWarps * kSlots * kTileBytes + 1024;
constexpr int kMaxSplits = 32;                   // CTAs that share the selected blocks of a (sequence, KV head)
constexpr int kMaxCtas = kResident * kNumSMs;    // one wave
constexpr uint32_t kStart = 4;                   // blocks that the start of a head costs (see Deal)
constexpr int kUsualBlocks = 64;                 // blocks that a mask row is taken to select
constexpr int kMaxList = 2 * kThreads;           // longest block list that the split kernel takes itself
constexpr long long kWaitLimit = 1ll << 28;      // clocks; a copy takes microseconds
constexpr int kPartialFloats = kHeadDim + 4;     // O row, m (log2 units), l, exponent of O's units, pad
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLowest = -0x1.fffffep127f;      // the lowest finite number

struct Q8DecodeParams {
  const __nv_bfloat16* q;          // (batch, heads_q, 128)
  uint8_t* k_codes;
  uint8_t* v_codes;
  uint8_t* k_scale;
  uint8_t* v_scale;
  const __nv_bfloat16* k_new;      // (batch, heads_k, 128) new rows that the split kernel appends, or null
  const __nv_bfloat16* v_new;
  const unsigned long long* mask;  // (batch, heads_k, mask_words) or null = all positions
  int mask_words;
  const int32_t* topk_idx;         // (batch, heads_k, topk <= kMaxList) block lists in place of a mask, or null
  int topk;
  const int32_t* cache_seqlens;
  Place place;
  uint32_t page_mul;               // a position's page: umulhi(position, page_mul) >> page_shift
  int page_shift;
  int64_t capacity;
  int batch, heads_k, new_tokens, rotate;
  int splits;                      // CTAs that share a (sequence, KV head) each, or 0: the blocks are dealt (see Deal)
  int most_blocks;                 // a head counts for so many blocks in the deal at most
  RotaryParams rotary;
  float scale_log2;
  float* partial;                  // (batch, heads_k, splits | 2 per CTA, 16, kPartialFloats)
  __nv_bfloat16* out;
  float* lse;                      // (batch, heads_q) or null
};

struct Q8PrepareParams {
  const __nv_bfloat16* k_new;      // (batch, heads_k, 128) or null = no append
  const __nv_bfloat16* v_new;
  uint8_t* k_codes;
  uint8_t* v_codes;
  uint8_t* k_scale;
  uint8_t* v_scale;
  const int32_t* topk_idx;         // (batch, heads_k, topk) or null
  unsigned long long* mask;
  int topk, words;
};

// Keys that sequence b attends.  A length below 0 has none; past the capacity, those that exist (a new token without
// room is neither written nor attended).
__device__ __forceinline__ int keys_of(const Q8DecodeParams& p, int b) {
  const int64_t len = p.cache_seqlens[b];
  return len < 0 ? 0 : (int)min(len + p.new_tokens, p.capacity);
}

// Rows of a token in a warp, features 4 lane .. 4 lane + 3 in each lane: the lane's angles, loaded once for all rows, and
// a row's own and partner features as they come from memory.
struct Angles {
  float c[4], s[4];
  int mate;                        // where the partner's four features are (halves), 0: in the lane itself (neighbours)
  bool on, second;                 // the lane's features turn; they are the second of their pairs (halves)
  __device__ __forceinline__ void load(const RotaryParams& r, int64_t t, int lane) {
    const int half = r.dim / 2, f = 4 * lane;
    on = f < r.dim;
    second = !r.interleaved && f >= half;
    mate = r.interleaved || !on ? 0 : second ? -half : half;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (!on || (r.interleaved && i >= 2)) continue;
      const int pair = r.interleaved ? 2 * lane + i : second ? f - half + i : f + i;
      const int64_t e = r.table_row(t, pair) * half + pair;
      c[i] = __ldg(r.cos_t + e);
      s[i] = __ldg(r.sin_t + e);
    }
  }
};
struct RowPart {
  uint2 own, mate;
  __device__ __forceinline__ void load(const __nv_bfloat16* row, int lane, int mate_at) {
    own = __ldg(reinterpret_cast<const uint2*>(row) + lane);
    if (mate_at != 0) mate = __ldg(reinterpret_cast<const uint2*>(row + 4 * lane + mate_at));
  }
  static __device__ __forceinline__ void widen(float (&x)[4], const uint2& v) {
    x[0] = __uint_as_float(v.x << 16);
    x[1] = __uint_as_float(v.x & 0xFFFF0000u);
    x[2] = __uint_as_float(v.y << 16);
    x[3] = __uint_as_float(v.y & 0xFFFF0000u);
  }
  __device__ __forceinline__ void plain(float (&x)[4]) const { widen(x, own); }
  __device__ __forceinline__ void turned(float (&x)[4], const Angles& a) const {
    widen(x, own);
    if (!a.on) return;
    if (a.mate == 0) {
      rotate2(x[0], x[1], a.c[0], a.s[0]);
      rotate2(x[2], x[3], a.c[1], a.s[1]);
      return;
    }
    float y[4];
    widen(y, mate);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x0 = a.second ? y[i] : x[i], x1 = a.second ? x[i] : y[i];
      rotate2(x0, x1, a.c[i], a.s[i]);
      x[i] = a.second ? x1 : x0;
    }
  }
};

// One CTA per (sequence, KV head): block lists -> mask row; the new key (rotated) and value -> their row.  (The next kernel of the call
// may start beside this one: what it reads of this one's it reads after its wait, which every thread of it makes before it ends.)
template <int kCode>
__global__ void __launch_bounds__(kThreads) q8_prepare_kernel(const Q8PrepareParams a, const Q8DecodeParams p) {
  extern __shared__ unsigned long long row_words[];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
  const int64_t pair = (int64_t)b * p.heads_k + h;
  allow_next();
  if (a.topk_idx != nullptr) {
    for (int w = tid; w < a.words; w += kThreads) row_words[w] = 0ull;
    __syncthreads();
    for (int i = tid; i < a.topk; i += kThreads) {
      const int v = a.topk_idx[pair * a.topk + i];
      if (v >= 0 && v < a.words * 64) atomicOr(&row_words[v >> 6], 1ull << (v & 63));
    }
  }
  if (a.k_new != nullptr && tid < 64) {
    const int64_t len = p.cache_seqlens[b];
    const int64_t row0 = len < p.capacity ? p.place.row0(b, len) : -1;
    if (row0 >= 0) {
      const int64_t row = p.place.row(row0, h);
      const bool is_v = tid >= 32;
      Angles angles;
      angles.mate = 0;
      angles.on = false;
      if (p.rotate && !is_v) angles.load(p.rotary, b, lane);
      RowPart part;
      part.load((is_v ? a.v_new : a.k_new) + pair * kHeadDim, lane, angles.mate);
      float x[4];
      part.turned(x, angles);
      store_row<kCode>(x, (is_v ? a.v_codes : a.k_codes) + row * kHeadDim, (is_v ? a.v_scale : a.k_scale) + row, lane);
    }
  }
  if (a.topk_idx != nullptr) {
    __syncthreads();
    for (int w = tid; w < a.words; w += kThreads) a.mask[pair * a.words + w] = row_words[w];
  }
}

// Blocks of 64 keys that one sequence's head counts for in the deal, and the length of its place there.
__device__ __forceinline__ int blocks_of(const Q8DecodeParams& p, int b) {
  return min((keys_of(p, b) + kBlockN - 1) / kBlockN, p.most_blocks);
}
__device__ __forceinline__ uint32_t extent(int blocks) { return blocks ? kStart + blocks : 0; }

// The blocks of all sequences and heads are one row, sequence by sequence, head by head, and CTA c of `ctas` takes those
// from c total / ctas on: shares of equal cost, blocks and starts of heads, whatever the lengths are (in equal splits, 16
// sequences of 1000 .. 32000 tokens wait for the longest one).  One wave of CTAs: with 1.5, 2 and 3 times as many, 64
// sequences of 4000 tokens take 42, 46 and 52 us instead of 32.  Every warp finds its place by itself, a sequence per lane.
//
// Where a CTA goes from one head to the next it starts over (query, first tiles, join), for about as long as it takes for
// kStart blocks, so a head's place in the row begins with as many that are no work: CTAs whose shares hold more starts
// read fewer bytes.  Without / with them: 16 sequences of
// 1000 .. 32000 tokens 38.2 / 35.3 us, 12 of up to 30000 with 8 KV heads 107 / 98.8, 256 of 100 .. 1000 41.6 / 34.9; 3
// or 5 in place of 4 made no difference beyond 1 %.
//
// Under a selection a head's place is as long as its list can be (a mask: as kUsualBlocks, whatever it selects), and the
// CTAs that share it share the selected blocks in proportion, so that the deal need not wait for their number.
struct Deal {
  uint32_t total, ctas, each, rest;                // total = each * ctas + rest
  // extents: of all sequences, for one KV head (the host keeps the total below 2^31)
  __device__ Deal(uint32_t extents, int heads_k, uint32_t grid) {
    total = extents * heads_k;
    // two blocks are one 32-key unit for each of the four warps
    ctas = max(1u, min(grid, (total + 1) / 2));
    each = total / ctas;
    rest = total - each * ctas;
  }
  __device__ uint32_t first(uint32_t c) const { return c * each + c * rest / ctas; }      // c total / ctas
  // the last c with first(c) <= block, from an estimate that is off by one at most
  __device__ uint32_t cta_of(uint32_t block) const {
    uint32_t c = min((uint32_t)((float)block * ((float)ctas / (float)total)), ctas - 1);
    while (c + 1 < ctas && first(c + 1) <= block) ++c;
    while (first(c) > block) --c;
    return c;
  }
};

// Sequence that holds block `at` of the row, and the row's blocks before it.
__device__ __forceinline__ int find_block(const Q8DecodeParams& p, uint32_t at, uint32_t& before, int lane) {
  before = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 32) {
    const uint32_t n = b0 + lane < p.batch ? extent(blocks_of(p, b0 + lane)) * p.heads_k : 0u;
    uint32_t incl = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t up = __shfl_up_sync(0xFFFFFFFFu, incl, d);
      if (lane >= d) incl += up;
    }
    const uint32_t past = __ballot_sync(0xFFFFFFFFu, before + incl > at);
    if (past) {
      const int src = __ffs(past) - 1;
      before += __shfl_sync(0xFFFFFFFFu, incl - n, src);
      return b0 + src;
    }
    before += __shfl_sync(0xFFFFFFFFu, incl, 31);
  }
  return p.batch;
}

// A block list as the split kernel walks it: the blocks below nblk, ascending, each once; returns their number.  Lists
// come ascending with their unused entries last as a rule, which one look confirms; others are ranked entry by entry.
__device__ __forceinline__ int sort_list(int* list, const int32_t* src, int topk, int nblk) {
  constexpr int kNone = 0x7FFFFFFF;
  const int tid = threadIdx.x;
  int mine[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int i = tid + u * kThreads, x = i < topk ? __ldg(src + i) : -1;
    mine[u] = x >= 0 && x < nblk ? x : kNone;
    list[i] = mine[u];
  }
  int n = __syncthreads_count(mine[0] != kNone);
  n += __syncthreads_count(mine[1] != kNone);
  bool ascending = true;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int i = tid + u * kThreads, next = i + 1 < kMaxList ? list[i + 1] : kNone;
    ascending &= mine[u] < next || next == kNone;
  }
  if (__syncthreads_and(ascending)) return n;
  bool again[2] = {false, false};                 // an entry that stands before already
  for (int u = 0; u < 2; ++u)
    for (int j = 0; j < tid + u * kThreads && j < topk; ++j) again[u] |= list[j] == mine[u];
  __syncthreads();
  for (int u = 0; u < 2; ++u)
    if (again[u]) list[tid + u * kThreads] = mine[u] = kNone;
  n = __syncthreads_count(mine[0] != kNone);
  n += __syncthreads_count(mine[1] != kNone);
  int rank[2] = {0, 0};
  for (int u = 0; u < 2; ++u)
    for (int j = 0; j < topk; ++j) rank[u] += list[j] < mine[u];
  __syncthreads();
  for (int u = 0; u < 2; ++u)
    if (mine[u] != kNone) list[rank[u]] = mine[u];
  __syncthreads();
  return n;
}

// A partial sum in units of 2^m as one in units of 2^top.  Without a finite m it is 0, or NaN and stays so.
__device__ __forceinline__ float join_weight(float m, float top) { return m == -INFINITY ? 1.f : exp2f(m - top); }

// x 2^d, |d| <= 150, in two steps so that neither factor leaves the normal numbers.
__device__ __forceinline__ float times_exp2(float x, float d) {
  const float f = exp2f(0.5f * d);
  return mul_exact(mul_exact(x, f), f);
}

__device__ __forceinline__ void store_out(const Q8DecodeParams& p, int64_t qrow, int d0, const float (&acc)[4], float m, float l,
                                          float unit) {
  // l == 0: no key; NaN: a NaN among them
  const float inv = l == 0.f ? 0.f : 1.f / l;
  float x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = l == 0.f ? 0.f : times_exp2(acc[i] * inv, unit - m);
  *reinterpret_cast<uint2*>(p.out + qrow * kHeadDim + d0) = make_uint2(mmasync::pack2(x[0], x[1]), mmasync::pack2(x[2], x[3]));
  if (p.lse != nullptr && d0 == 0) p.lse[qrow] = l == 0.f ? INFINITY : (m + log2f(l)) * kLn2;
}

// A CTA's blocks of one (sequence, KV head) at a time; each of its four warps streams 32-key units, K and V in turn,
// through its own three slots of shared memory (4 KB, 128-byte swizzle, filled by TMA), so that two tiles are in flight
// while another is worked on.  The 16 query heads are one M tile of mma.sync m16n8k16 in fp16, fp32 sums: codes become fp16
// numbers exactly, a query row is scaled by a power of two so that its largest element is 1 to 2 (exact but for elements
// below 2^-16 of that, which are off by 2^-25 of it at most; a rotated row, which has 24 bits, becomes a sum of two fp16
// rows), scales are applied to the scores and, as exponents, to the weights.  A weight is rounded to fp16 at 2^8 to 2^15
// times its share of the largest, 2^-12 relative down to 2^-22 of that and 2^-33 of it below.
//
// The contraction order over the 128 features is free, so codes 4t .. 4t + 3 of a 16-feature chunk, one 32-bit word
// of ldmatrix, serve as k = 2t, 2t + 1, 2t + 8, 2t + 9; the query is read in the same order.  V comes through the
// transposing 16-bit ldmatrix, a word of which holds two tokens' codes of two neighbouring features: even features
// and odd features of a chunk are the columns of two products.
//
// Bound by HBM where there is much to read, and by about 12 us of start (3 us to the first tile), uneven ends and join
// elsewhere.  e4m3, two KV heads, 64 sequences of 4000 / 16000 / 32000 tokens: 32 / 88.8 / 164 us with the join, 63 / 91 /
// 99 % of the copy bandwidth; without the copies the arithmetic alone takes 77 us at 16000.  Eight heads, 8 sequences of
// 30000 tokens: e4m3 93 us, int8 100 (five instructions for four codes in place of two), with a rotated query 108 and 116
// (three fp16 products for two).
//
// kPage: 0, slots are sequences; 32, pages of a multiple of 32 positions; 16, of 16, so that a tile comes in two boxes.
// kCopied: scale bytes come with K's tile, by copies of their own, where those of a unit are together and begin at a multiple
// of 16 bytes.  As loads they cost more than the 0.8 % that they are of the bytes: 64 sequences of 16000 tokens, two heads,
// take 88.8 us against 95.5.  In pages of 16 copies of 16 bytes cost more: 64 sequences of 32000 tokens 189 us against 184.
template <int kCode, int kPage, bool kRotate, bool kCopied>
__global__ void __launch_bounds__(kThreads, kResident)
q8_split_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Q8DecodeParams p) {
  constexpr int kBox = kPage == 16 ? 16 : 32;      // rows that one copy takes
  allow_next();
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ uint64_t bars[kWarps][kSlots];
  // of the unit at work: scales of the keys in two factors, exponents of the values
  __shared__ __align__(16) float factors[kWarps][3][kUnit];
  // the query as A fragments: [high and low part][16-feature chunk][lane]
  __shared__ uint4 q_frag[kRotate ? 2 : 1][kHeadDim / 16][32];
  __shared__ float q_factor[kGroup];               // 2^x that undoes a row's scaling
  __shared__ __align__(16) uint8_t scale_bytes[kCopied ? kWarps : 1][2][2][kUnit];      // [warp][unit][K, V][key]
  __shared__ int block_list[kMaxList];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  uint8_t* tiles = smem + warp * kSlots * kTileBytes;
  if (lane == 0) {
    if (warp == 0) {
      tc::prefetch_tensormap(&map_k);
      tc::prefetch_tensormap(&map_v);
    }
#pragma unroll
    for (int i = 0; i < kSlots; ++i) tc::mbar_init(&bars[warp][i], kUnit / kBox);
    tc::fence_barrier_init();
  }
  __syncwarp();
  // a lane's places in a tile: 16-byte chunk c of row r lies at chunk c ^ (r & 7)
  const uint32_t tiles32 = tc::smem_u32(tiles);
  uint32_t k_lane[2], v_lane[4];
#pragma unroll
  for (int i = 0; i < 2; ++i) k_lane[i] = (lane & 7) * kHeadDim + (((i * 4 + (lane >> 3)) ^ (lane & 7)) << 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) v_lane[i] = (lane & 15) * kHeadDim + (((i * 2 + (lane >> 4)) ^ (lane & 7)) << 4);
  uint32_t phases = 0;                             // bit i: parity of the next completion of slot i
  bool expired = false;                            // a bounded wait ran out: the result is poisoned

  // the CTA's share: blocks [at, end) of the row of all blocks, or split `split` of the selected blocks
  const bool listed = p.topk_idx != nullptr, selected = listed || p.mask != nullptr, dealt = p.splits == 0;
  int b = 0, h = 0, split = 0;
  uint32_t at = 0, end = 0, before = 0;
  if (dealt) {
    uint32_t extents = 0;
    for (int i = lane; i < p.batch; i += 32) extents += extent(blocks_of(p, i));
    const Deal deal(__reduce_add_sync(0xFFFFFFFFu, extents), p.heads_k, gridDim.x);
    if (deal.total == 0 || blockIdx.x >= deal.ctas) {
      wait_previous();
      return;
    }
    at = deal.first(blockIdx.x);
    end = deal.first(blockIdx.x + 1);
    b = find_block(p, at, before, lane);
  } else {
    split = blockIdx.x % p.splits;
    const int pair = blockIdx.x / p.splits;
    b = pair / p.heads_k;
    h = pair % p.heads_k;
  }

  auto advance = [&](uint32_t by) -> bool {        // to the next head or sequence; false: the share is done
    at += by;
    if (at >= end) return false;
    for (uint32_t len; at - before >= (len = extent(blocks_of(p, b)) * p.heads_k); ++b) before += len;
    return true;
  };
  while (true) {
    const int len = keys_of(p, b);
    uint32_t w0 = split, w1 = split + 1, nw = p.splits, used = 0;      // the CTA's share of the head: w0 .. w1 - 1 of nw
    if (dealt) {
      nw = blocks_of(p, b);
      const uint32_t place = kStart + nw;
      h = (int)((at - before) / place);
      const uint32_t v0 = at - before - h * place, v1 = min(place, v0 + end - at);
      used = v1 - v0;
      if (v1 <= kStart) {                          // (nothing to do for this head)
        wait_previous();
        if (!advance(used)) return;
        continue;
      }
      w0 = max(v0, kStart) - kStart;
      w1 = v1 - kStart;
    }
    const int64_t pair = (int64_t)b * p.heads_k + h;
    // the warp's rows of the query, on their way while the first tiles are asked for
    Angles angles;
    angles.mate = 0;
    if (kRotate) angles.load(p.rotary, b, lane);
    RowPart q_part[kGroup / kWarps];
#pragma unroll
    for (int i = 0; i < kGroup / kWarps; ++i) q_part[i].load(p.q + (pair * kGroup + warp + kWarps * i) * kHeadDim, lane, angles.mate);

    wait_previous();                               // (the mask, or a new row of shared pages)
    const int n_all = (len + kBlockN - 1) / kBlockN;
    BlockList<2, true> list{p.mask ? p.mask + pair * p.mask_words : nullptr, p.mask_words, n_all, -1};
    // blocks to attend, of which this CTA takes numbers j0 .. j1 - 1
    const uint32_t n = listed ? sort_list(block_list, p.topk_idx + pair * p.topk, p.topk, n_all) : list.count(lane);
    const int j0 = n == nw ? w0 : (int)((uint64_t)w0 * n / nw), j1 = n == nw ? w1 : (int)((uint64_t)w1 * n / nw);

    // the new token's row, by the warp whose unit it belongs to (no CTA attends it: by the first warp of the first CTA)
    if (p.k_new != nullptr) {
      const int pos = p.cache_seqlens[b];
      if (pos >= 0 && pos < p.capacity) {
        const int blk = pos / kBlockN;
        const bool attended = !selected || (listed ? n > 0 && block_list[n - 1] == blk
                                                   : blk / 64 < p.mask_words && ((list.words[blk / 64] >> (blk & 63)) & 1ull));
        const int owner = attended ? (((n - 1 - j0) & 1) << 1) | ((pos / kUnit) & 1) : 0;
        if ((attended ? j0 < j1 && j1 == (int)n : w0 == 0) && warp == owner) {
          const int64_t row = ((int64_t)b * p.heads_k + h) * p.place.length + pos;
          RowPart k_part, v_part;
          k_part.load(p.k_new + pair * kHeadDim, lane, angles.mate);
          v_part.load(p.v_new + pair * kHeadDim, lane, 0);
          float x[4];
          if (kRotate) k_part.turned(x, angles);
          else k_part.plain(x);
          store_row<kCode>(x, p.k_codes + row * kHeadDim, p.k_scale + row, lane);
          v_part.plain(x);
          store_row<kCode>(x, p.v_codes + row * kHeadDim, p.v_scale + row, lane);
          __threadfence();
          tc::fence_proxy_async_global();
          __syncwarp();
        }
      }
    }

    // this warp's units: half (warp & 1) of blocks j0 + (warp >> 1), + 2, ...
    int j = j0 + (warp >> 1), lookups = 0;
    auto next_key = [&]() -> int {                 // first key of the next unit, or -1
      while (j < j1) {
        const int blk = listed ? block_list[j] : list.nth(lookups++, j, lane);
        j += 2;
        const int key0 = blk * kBlockN + (warp & 1) * kUnit;
        if (blk >= 0 && key0 < len) return key0;
      }
      return -1;
    };
    // where the key of this lane is (-1: nowhere), and its scale bytes.  (The cache has fewer than 2^31 rows.)
    int slot0 = 0;                                 // row of the head's first position, where slots are sequences
    if (kPage == 0) {
      const int slot = p.place.batch_idx ? __ldg(p.place.batch_idx + b) : b;
      slot0 = slot >= 0 && slot < p.place.slots ? (slot * p.place.heads + h) * p.place.length : -1;
    }
    // entry of the block table for it, read a unit ahead, because what uses it waits for the load (with the page by
    // multiplication: 64 sequences of 32000 tokens in pages of 16 184 us in place of 199)
    auto page_of = [&](int key) -> int { return (int)(__umulhi((uint32_t)key, p.page_mul) >> p.page_shift); };
    auto entry = [&](int key0) -> int {
      const int key = key0 + lane;
      return kPage != 0 && key0 >= 0 && key < len ? __ldg(p.place.block_table + (int64_t)b * p.place.bt_stride + page_of(key)) : -1;
    };
    // The bytes are not touched before the unit's turn either.
    auto locate = [&](int key0, int slot, int& row, uint32_t& kb, uint32_t& vb) {
      row = -1;
      kb = vb = kNanByte;                          // (a page that the cache does not have: NaN; no tile comes for it)
      const int key = key0 + lane;
      if (key < len) {
        if (kPage != 0) {
          if (slot >= 0 && slot < p.place.slots) row = (slot * p.place.heads + h) * p.place.length + key - page_of(key) * p.place.length;
        } else if (slot0 >= 0) {
          row = slot0 + key;
        }
        if (!kCopied && row >= 0) {
          kb = p.k_scale[row];                     // (ordinary loads: this warp or the kernel before wrote the newest)
          vb = p.v_scale[row];
        }
      }
    };
    // starts the copy of the tile whose keys' rows the lanes hold into slot i, which the warp is done reading (what is
    // written there by ordinary stores, the zeros of a tail and the join, is fenced off at the end of a segment)
    int turn = 0;                                  // kCopied: which of its two places the next unit's scale bytes get
    auto fetch = [&](const CUtensorMap& map, int i, int row, auto with_scales) {
      constexpr bool kScales = kCopied && decltype(with_scales)::value;
      __syncwarp();
      if (lane % kBox == 0) {
        uint64_t* bar = &bars[warp][i];
        tc::mbar_expect_tx(bar, row >= 0 ? kBox * kHeadDim + (kScales ? 2 * kUnit : 0) : 0);
        if (row >= 0) {
          tc::tma_load_2d(tiles + i * kTileBytes + lane * kHeadDim, &map, bar, 0, row);
          if (kScales) {
            tc::bulk_load(scale_bytes[warp][turn][0], p.k_scale + row, kUnit, bar);
            tc::bulk_load(scale_bytes[warp][turn][1], p.v_scale + row, kUnit, bar);
          }
        }
      }
      if (kScales) turn ^= 1;
    };
    // waits for slot i's copy; the whole warp gets the same verdict
    auto arrived = [&](int i) -> bool {
      uint64_t* bar = &bars[warp][i];
      const uint32_t parity = (phases >> i) & 1u;
      phases ^= 1u << i;
      if (__all_sync(0xFFFFFFFFu, tc::mbar_try_wait(bar, parity))) return true;
      const long long start = clock64();
      while (!__all_sync(0xFFFFFFFFu, tc::mbar_try_wait_hint(bar, parity, 1000)))
        if (__any_sync(0xFFFFFFFFu, clock64() - start > kWaitLimit)) return false;
      return true;
    };

    // unit at work, the next one and that after it: first keys, rows, scale bytes; slots of K, V and the next K
    int key0 = next_key(), key1 = key0 >= 0 ? next_key() : -1, key2 = -1, row = -1, row1 = -1, slot_k = 0, slot_v = 1, slot_n = 2;
    int entry2 = -1;                               // of the block table
    uint32_t kb = 0, vb = 0, kb1 = 0, vb1 = 0;
    if (key0 >= 0) {
      const int entry0 = entry(key0), entry1 = entry(key1);
      locate(key0, entry0, row, kb, vb);
      fetch(map_k, slot_k, row, std::true_type{});
      fetch(map_v, slot_v, row, std::false_type{});
      if (key1 >= 0) {
        locate(key1, entry1, row1, kb1, vb1);
        fetch(map_k, slot_n, row1, std::true_type{});
        if (kPage != 0) {
          key2 = next_key();
          entry2 = entry(key2);
        }
      }
    }

    // the query rows, rotated, as fp16 with a power of two taken out
#pragma unroll
    for (int n4 = 0; n4 < kGroup / kWarps; ++n4) {
      const int i = warp + kWarps * n4;
      float x[4];
      if (kRotate) q_part[n4].turned(x, angles);
      else q_part[n4].plain(x);
      uint32_t amax = 0;
#pragma unroll
      for (int u = 0; u < 4; ++u) amax = max(amax, abs_bits(x[u]));
      const int e = min(max((int)(__reduce_max_sync(0xFFFFFFFFu, amax) >> 23), 1), 253);      // the largest becomes 1 .. 2
      const float f = __uint_as_float((uint32_t)(254 - e) << 23);
#pragma unroll
      for (int u = 0; u < 4; u += 2) {
        const float y0 = mul_exact(x[u], f), y1 = mul_exact(x[u + 1], f);
        const __half2 y = __floats2half2_rn(y0, y1);
        // features 4 lane + u, + 1 of row i: word (i / 8) + u of fragment lane 4 (i % 8) + lane % 4
        const int at = (i & 7) * 4 + (lane & 3), word = (i >> 3) + u;
        reinterpret_cast<__half2*>(&q_frag[0][lane >> 2][at])[word] = y;
        if (kRotate) {
          const float2 z = __half22float2(y);
          reinterpret_cast<__half2*>(&q_frag[kRotate ? 1 : 0][lane >> 2][at])[word] = __floats2half2_rn(y0 - z.x, y1 - z.y);
        }
      }
      if (lane == 0) q_factor[i] = __uint_as_float((uint32_t)e << 23);
    }
    __syncthreads();
    const float c0 = mul_exact(q_factor[g], p.scale_log2), c1 = mul_exact(q_factor[g + 8], p.scale_log2);

    float o[16][4];
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    bool fresh = true;                             // no unit yet: there are no references
    // rows g and g + 8: reference m, l, and reference M; O's units are 2^(M - 8)
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f, u0 = -INFINITY, u1 = -INFINITY;

    while (key0 >= 0) {
      const uint32_t kt = tiles32 + slot_k * kTileBytes, vt = tiles32 + slot_v * kTileBytes;
      if (!arrived(slot_k)) {
        expired = true;
        break;
      }
      if (kCopied) {
        const int at = key1 >= 0 ? turn : turn ^ 1;          // (the places are given out in turn)
        kb = row >= 0 ? scale_bytes[warp][at][0][lane] : kNanByte;
        vb = row >= 0 ? scale_bytes[warp][at][1][lane] : kNanByte;
      }
      // 2^(kb - 127) = 2^a 2^b: with the query's factor between the two no product leaves the range that the score is in
      factors[warp][0][lane] = kb == kNanByte ? __uint_as_float(0x7FC00000u) : __uint_as_float((64 + kb / 2) << 23);
      factors[warp][1][lane] = __uint_as_float((63 + (kb + 1) / 2) << 23);
      factors[warp][2][lane] = vb == kNanByte ? __uint_as_float(0x7FC00000u) : (float)((int)vb - 127);
      __syncwarp();

      // ---- S = Q . K^T (16 x 32)
      float s[kUnit / 8][4];
#pragma unroll
      for (int nt = 0; nt < kUnit / 8; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
      for (int kp = 0; kp < 2; ++kp) {
        uint32_t w[kUnit / 8][4];
#pragma unroll
        for (int nt = 0; nt < kUnit / 8; ++nt) mmasync::ldmatrix_x4(w[nt], kt + k_lane[kp] + nt * 8 * kHeadDim);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const uint4 hi4 = q_frag[0][kp * 4 + u][lane], lo4 = q_frag[kRotate ? 1 : 0][kp * 4 + u][lane];
          const uint32_t qh[4] = {hi4.x, hi4.y, hi4.z, hi4.w}, ql[4] = {lo4.x, lo4.y, lo4.z, lo4.w};
          uint32_t f[kUnit / 8][2];
#pragma unroll
          for (int nt = 0; nt < kUnit / 8; ++nt) {
            decode_h2<kCode>(f[nt][0], f[nt][1], w[nt][u]);
            mmasync::mma_f16(s[nt], qh, f[nt][0], f[nt][1]);
          }
          if (kRotate) {                           // (after the four others: a sum waits for its last product)
#pragma unroll
            for (int nt = 0; nt < kUnit / 8; ++nt) mmasync::mma_f16(s[nt], ql, f[nt][0], f[nt][1]);
          }
        }
      }

      if (key1 >= 0) fetch(map_v, slot_k, row1, std::false_type{});

      // ---- weights against reference maxima that move only when a weight would pass 2^15: the sum l against m, the
      //      weights of the values against M - 8 (see the file's head).  A unit whose weights pass is done again.
      // pairs for keys 8 nt + 2t, + 1: exponents of values, second factors of keys, scores without it of two rows
      uint64_t ev[kUnit / 8], kb2[kUnit / 8], sp[kUnit / 8][2];
      const uint64_t cc0 = tc::pack_f32x2(c0, c0), cc1 = tc::pack_f32x2(c1, c1);
#pragma unroll
      for (int nt = 0; nt < kUnit / 8; ++nt) {
        const uint64_t ks = *reinterpret_cast<const uint64_t*>(&factors[warp][0][nt * 8 + 2 * t]);
        kb2[nt] = *reinterpret_cast<const uint64_t*>(&factors[warp][1][nt * 8 + 2 * t]);
        ev[nt] = *reinterpret_cast<const uint64_t*>(&factors[warp][2][nt * 8 + 2 * t]);
        sp[nt][0] = mul_exact2(mul_exact2(tc::pack_f32x2(s[nt][0], s[nt][1]), ks), cc0);
        sp[nt][1] = mul_exact2(mul_exact2(tc::pack_f32x2(s[nt][2], s[nt][3]), ks), cc1);
      }
      float sum[2];
      uint32_t pf[kUnit / 16][4];                  // weights as A fragments of the second product
      auto weigh = [&](auto tail) -> bool {
        constexpr bool kTail = decltype(tail)::value;
        __half2 top;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float m = r ? m1 : m0, u = r ? u1 : u0;
          const float n = -m, w = 8.f - u;
          const uint64_t nn = tc::pack_f32x2(n, n), ww = tc::pack_f32x2(w, w);
          uint64_t total = 0;
#pragma unroll
          for (int nt = 0; nt < kUnit / 8; ++nt) {
            float a0, a1, x0, x1;
            tc::unpack_f32x2(tc::fma_f32x2(sp[nt][r], kb2[nt], nn), a0, a1);
            tc::unpack_f32x2(tc::add_f32x2(tc::fma_f32x2(sp[nt][r], kb2[nt], ww), ev[nt]), x0, x1);
            if (kTail) {
              if (key0 + nt * 8 + 2 * t >= len) a0 = x0 = -INFINITY;
              if (key0 + nt * 8 + 2 * t + 1 >= len) a1 = x1 = -INFINITY;
            }
            total = tc::add_f32x2(total, tc::pack_f32x2(exp2f(a0), exp2f(a1)));
            const __half2 y = __floats2half2_rn(exp2f(x0), exp2f(x1));
            top = r == 0 && nt == 0 ? y : __hmax2(top, y);
            pf[nt >> 1][(nt & 1) * 2 + r] = *reinterpret_cast<const uint32_t*>(&y);
          }
          float a0, a1;
          tc::unpack_f32x2(total, a0, a1);
          sum[r] = a0 + a1;
        }
        const float2 y = __half22float2(top);
        return fmaxf(y.x, y.y) > 0x1p15f || fmaxf(sum[0], sum[1]) > 0x1p40f;
      };
      bool again = fresh;
      if (!fresh) again = key0 + kUnit > len ? weigh(std::true_type{}) : weigh(std::false_type{});
      if (__any_sync(0xFFFFFFFFu, again)) {
        // (no reference is -inf: next to scores that are all -inf, or NaN, the first finite one weighs infinitely, and
        // the references move)
        float mx0 = fmaxf(m0, kLowest), mx1 = fmaxf(m1, kLowest), mu0 = fmaxf(u0, kLowest), mu1 = fmaxf(u1, kLowest);
#pragma unroll
        for (int nt = 0; nt < kUnit / 8; ++nt) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if (key0 + nt * 8 + 2 * t + e >= len) continue;
            float a[2], b2[2], ex[2];
            tc::unpack_f32x2(mul_exact2(sp[nt][0], kb2[nt]), a[0], a[1]);
            tc::unpack_f32x2(mul_exact2(sp[nt][1], kb2[nt]), b2[0], b2[1]);
            tc::unpack_f32x2(ev[nt], ex[0], ex[1]);
            mx0 = fmaxf(mx0, a[e]);
            mx1 = fmaxf(mx1, b2[e]);
            mu0 = fmaxf(mu0, a[e] + ex[e]);
            mu1 = fmaxf(mu1, b2[e] + ex[e]);
          }
        }
#pragma unroll
        for (int d = 1; d < 4; d <<= 1) {
          mx0 = fmaxf(mx0, __shfl_xor_sync(0xFFFFFFFFu, mx0, d));
          mx1 = fmaxf(mx1, __shfl_xor_sync(0xFFFFFFFFu, mx1, d));
          mu0 = fmaxf(mu0, __shfl_xor_sync(0xFFFFFFFFu, mu0, d));
          mu1 = fmaxf(mu1, __shfl_xor_sync(0xFFFFFFFFu, mu1, d));
        }
        l0 *= exp2f(m0 - mx0);
        l1 *= exp2f(m1 - mx1);
        const float f0 = exp2f(u0 - mu0), f1 = exp2f(u1 - mu1);
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          o[k][0] *= f0;
          o[k][1] *= f0;
          o[k][2] *= f1;
          o[k][3] *= f1;
        }
        m0 = mx0;
        m1 = mx1;
        u0 = mu0;
        u1 = mu1;
        fresh = false;
        weigh(std::true_type{});
      }
      l0 += sum[0];                                // per lane; added up over the quad at the end
      l1 += sum[1];

      // ---- O += P . V (16 x 128); rows past the last key have weight 0, but their bytes can be NaN codes
      if (!arrived(slot_v)) {
        expired = true;
        break;
      }
      if (key0 + kUnit > len) {
        for (int k = lane; k < kUnit * 8; k += 32)
          if (key0 + (k >> 3) >= len) *reinterpret_cast<uint4*>(tiles + slot_v * kTileBytes + k * 16) = make_uint4(0u, 0u, 0u, 0u);
        __syncwarp();
      }
#pragma unroll
      for (int kk = 0; kk < kUnit / 16; ++kk) {
#pragma unroll
        for (int np = 0; np < 4; ++np) {           // two chunks of 16 features
          uint32_t w[4];
          mmasync::ldmatrix_x4_trans(w, vt + v_lane[np] + kk * 16 * kHeadDim);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            uint32_t e0, e1, d0, d1;
            decode_h2_even_odd<kCode>(e0, d0, w[2 * u]);
            decode_h2_even_odd<kCode>(e1, d1, w[2 * u + 1]);
            mmasync::mma_f16(o[4 * np + 2 * u], pf[kk], e0, e1);
            mmasync::mma_f16(o[4 * np + 2 * u + 1], pf[kk], d0, d1);
          }
        }
      }
      key0 = key1;
      row = row1;
      kb = kb1;
      vb = vb1;
      if (key1 >= 0) {
        key1 = kPage != 0 ? key2 : next_key();
        if (key1 >= 0) {
          locate(key1, entry2, row1, kb1, vb1);
          fetch(map_k, slot_v, row1, std::true_type{});
          if (kPage != 0) {
            key2 = next_key();
            entry2 = entry(key2);
          }
        }
      }
      const int done = slot_k;
      slot_k = slot_n;
      slot_n = slot_v;
      slot_v = done;
    }
    if (expired) {                                 // NaN: visible, not silent; the other copies get their time to land
      l0 = l1 = __uint_as_float(0x7FC00000u);
      const long long start = clock64();
      for (int i = 0; i < kSlots; ++i)
        while (!tc::mbar_try_wait(&bars[warp][i], (phases >> i) & 1u) && clock64() - start < kWaitLimit >> 4) {}
      __syncwarp();
    }
    l0 += __shfl_xor_sync(0xFFFFFFFFu, l0, 1);
    l0 += __shfl_xor_sync(0xFFFFFFFFu, l0, 2);
    l1 += __shfl_xor_sync(0xFFFFFFFFu, l1, 1);
    l1 += __shfl_xor_sync(0xFFFFFFFFu, l1, 2);

    // ---- join the four warps through the slots' memory (all their copies have landed and been read)
    __syncthreads();
    float* stage = reinterpret_cast<float*>(smem);             // [warp][16][kPartialFloats]
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float* w = stage + (warp * kGroup + g + 8 * half) * kPartialFloats;
#pragma unroll
      for (int c = 0; c < 8; ++c)
        *reinterpret_cast<float4*>(w + 16 * c + 4 * t) =
            make_float4(o[2 * c][2 * half], o[2 * c + 1][2 * half], o[2 * c][2 * half + 1], o[2 * c + 1][2 * half + 1]);
      if (t == 0) {
        w[kHeadDim] = half ? m1 : m0;
        w[kHeadDim + 1] = half ? l1 : l0;
        w[kHeadDim + 2] = (half ? u1 : u0) - 8.f;
      }
    }
    __syncthreads();
    // all of the head: the result; in the deal the head's first blocks: the CTA's second place; otherwise its first
    const bool whole = w0 == 0 && w1 == nw;
    const int64_t part = dealt ? 2 * (int64_t)blockIdx.x + (w0 == 0) : (int64_t)blockIdx.x;
    for (int r = warp; r < kGroup; r += kWarps) {              // a row per warp, four features per lane
      const float* src = stage + r * kPartialFloats;
      float m = -INFINITY, unit = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        m = fmaxf(m, src[w * kGroup * kPartialFloats + kHeadDim]);
        unit = fmaxf(unit, src[w * kGroup * kPartialFloats + kHeadDim + 2]);
      }
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float* sw = src + w * kGroup * kPartialFloats;
        l += join_weight(sw[kHeadDim], m) * sw[kHeadDim + 1];
        const float f = join_weight(sw[kHeadDim + 2], unit);
        const float4 v = *reinterpret_cast<const float4*>(sw + 4 * lane);
        acc[0] += f * v.x;
        acc[1] += f * v.y;
        acc[2] += f * v.z;
        acc[3] += f * v.w;
      }
      if (whole) {
        store_out(p, pair * kGroup + r, 4 * lane, acc, m, l, unit);
      } else {
        float* dst = p.partial + (part * kGroup + r) * kPartialFloats;
        *reinterpret_cast<float4*>(dst + 4 * lane) = make_float4(acc[0], acc[1], acc[2], acc[3]);
        if (lane == 0) *reinterpret_cast<float4*>(dst + kHeadDim) = make_float4(m, l, unit, 0.f);
      }
    }
    if (!dealt || !advance(used)) return;
    tc::fence_proxy_async_smem();
    __syncthreads();                               // the stage is read before the next segment's copies land in it
  }
}

// Joins the partial sums of a (sequence, KV head).  kSplitWarps warps share a row's partials, a lane holds four
// features; eight partials' loads are in flight at a time.
template <int kSplitWarps>
__global__ void __launch_bounds__(256) q8_combine_kernel(const Q8DecodeParams p, int split_grid) {
  __shared__ float4 sums[8][32];
  __shared__ float4 stats[8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t pair = blockIdx.y;
  const int b = (int)(pair / p.heads_k), h = (int)(pair % p.heads_k);
  const int r = blockIdx.x * (8 / kSplitWarps) + warp / kSplitWarps, w0 = warp % kSplitWarps;
  int64_t first = pair * p.splits;                  // (of partials)
  int n = p.splits;
  bool start_slot = false;                          // the first partial lies in its CTA's second place
  if (p.splits == 0) {
    uint32_t extents = 0, before = 0;               // of all sequences, of those before b
    for (int i = lane; i < p.batch; i += 32) {
      const uint32_t v = extent(blocks_of(p, i));
      extents += v;
      if (i < b) before += v;
    }
    const Deal deal(__reduce_add_sync(0xFFFFFFFFu, extents), p.heads_k, split_grid);
    const int blocks = blocks_of(p, b);
    n = 0;
    if (blocks) {
      const uint32_t at = __reduce_add_sync(0xFFFFFFFFu, before) * p.heads_k + h * extent(blocks) + kStart;
      first = deal.cta_of(at);
      n = deal.cta_of(at + blocks - 1) - (int)first + 1;
    }
    start_slot = true;
  }
  wait_previous();
  if (start_slot && n == 1) return;                 // one CTA had all of it and wrote the result
  auto partial = [&](int s) -> const float* {
    const int64_t slot = start_slot ? 2 * (first + s) + (s == 0) : first + s;
    return p.partial + (slot * kGroup + r) * kPartialFloats;
  };
  float m = -INFINITY, unit = -INFINITY, acc[4] = {0.f, 0.f, 0.f, 0.f}, l = 0.f;
  constexpr int kBatch = 8;
  for (int s0 = w0; s0 < n; s0 += kBatch * kSplitWarps) {
    float4 v[kBatch], st[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      st[k] = make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
      if (s0 + k * kSplitWarps >= n) continue;
      const float* src = partial(s0 + k * kSplitWarps);
      v[k] = *reinterpret_cast<const float4*>(src + 4 * lane);
      st[k] = *reinterpret_cast<const float4*>(src + kHeadDim);
    }
    float top = m, top_unit = unit;
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      top = fmaxf(top, st[k].x);
      top_unit = fmaxf(top_unit, st[k].z);
    }
    l *= join_weight(m, top);
    const float f0 = join_weight(unit, top_unit);
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] *= f0;
    m = top;
    unit = top_unit;
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      l += join_weight(st[k].x, m) * st[k].y;
      const float f = join_weight(st[k].z, unit);
      acc[0] += f * v[k].x;
      acc[1] += f * v[k].y;
      acc[2] += f * v[k].z;
      acc[3] += f * v[k].w;
    }
  }
  if (kSplitWarps > 1) {
    sums[warp][lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
    if (lane == 0) stats[warp] = make_float4(m, l, unit, 0.f);
    __syncthreads();
    if (w0 != 0) return;
#pragma unroll
    for (int w = 1; w < kSplitWarps; ++w) {
      m = fmaxf(m, stats[warp + w].x);
      unit = fmaxf(unit, stats[warp + w].z);
    }
    l *= join_weight(stats[warp].x, m);
    const float f0 = join_weight(stats[warp].z, unit);
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] *= f0;
#pragma unroll
    for (int w = 1; w < kSplitWarps; ++w) {
      const float4 v = sums[warp + w][lane], st = stats[warp + w];
      l += join_weight(st.x, m) * st.y;
      const float f = join_weight(st.z, unit);
      acc[0] += f * v.x;
      acc[1] += f * v.y;
      acc[2] += f * v.z;
      acc[3] += f * v.w;
    }
  }
  store_out(p, pair * kGroup + r, 4 * lane, acc, m, l, unit);
}

}  // namespace
}  // namespace ifv2

using namespace ifv2;

// CTAs that share a (sequence, KV head) each, or 0: the blocks are dealt.  Without a selection they are.  Selected blocks
// are shared by CTAs of their head alone, as many as fill one wave, because a CTA that goes on to another head starts over:
// 64 blocks in 200 / 400 / 800 pairs 48 / 79 / 152 us, dealt 51 / 90 / 164; 16 blocks in 230 / 256 / 400 pairs 23 / 23 /
// 27, dealt 27 / 28 / 40.  Long lists are dealt where the wave, or the last one, would be 70 % full or less: 64 blocks in
// 150 / 256 / 460 / 600 pairs 44.6 / 68.9 / 129 / 142 us, dealt 41.1 / 60.6 / 102 / 127.
static int plan_splits(int64_t pairs, int blocks) {
  int64_t splits = kMaxCtas / pairs;
  splits = splits < 1 ? 1 : splits > kMaxSplits ? kMaxSplits : splits;
  const int64_t ctas = pairs * splits, waves = ceil_div64(ctas, kMaxCtas);
  return splits < kMaxSplits && blocks >= 48 && 10 * ctas <= 7 * waves * kMaxCtas ? 0 : (int)splits;
}

template <int kCode, bool kRotate>
static auto split_kernel(int page, bool copied) {
  return page == 32 ? q8_split_kernel<kCode, 32, kRotate, true>
       : page == 16 ? q8_split_kernel<kCode, 16, kRotate, false>
       : copied     ? q8_split_kernel<kCode, 0, kRotate, true> : q8_split_kernel<kCode, 0, kRotate, false>;
}

extern "C" int64_t ifv2_q8_decode_workspace_bytes(int batch, int heads_q, int head_dim) {
  if (batch < 0 || heads_q < 0 || head_dim != kHeadDim) return 0;
  // masks: every split of every (sequence, KV head), at most kMaxCtas of them or one each; no mask: two per CTA
  const int64_t pairs = (int64_t)batch * (heads_q / kGroup);
  const int64_t parts = pairs > 2 * kMaxCtas ? pairs : 2 * kMaxCtas;
  return parts * kGroup * kPartialFloats * 4;
}

extern "C" int ifv2_q8_decode(const void* q, void* k_cache, void* v_cache, void* k_scale, void* v_scale, const void* k_new,
                              const void* v_new, const float* rotary_cos, const float* rotary_sin,
                              const int32_t* rotary_positions, int64_t axis_stride, const uint8_t* pair_axis, int axes,
                              int rotary_dim, int64_t table_rows, int interleaved, const int32_t* topk_idx, int topk,
                              int64_t* mask, int mask_words, void* out, float* lse, const int32_t* cache_seqlens,
                              const int32_t* cache_batch_idx, const int32_t* block_table, int block_table_stride,
                              int64_t slots, int64_t length, int code, int batch, int heads_q, int heads_k, int head_dim,
                              float softmax_scale, void* workspace, int64_t workspace_bytes, void* stream) {
  IFV2_REQUIRE(head_dim == kHeadDim, IFV2_ERR_UNSUPPORTED, "q8_decode: head_dim %d not supported (only 128)", head_dim);
  IFV2_REQUIRE(heads_k >= 1 && heads_q == heads_k * kGroup, IFV2_ERR_UNSUPPORTED,
               "q8_decode: heads_q (%d) must be 16 x heads_k (%d)", heads_q, heads_k);
  IFV2_REQUIRE(code == kE4m3 || code == kInt8, IFV2_ERR_INVALID_ARG, "q8_decode: code must be 0 (e4m3) or 1 (int8)");
  IFV2_REQUIRE(batch >= 0 && slots >= 1 && length >= 1, IFV2_ERR_INVALID_ARG, "q8_decode: bad size");
  if (batch == 0) return IFV2_OK;
  IFV2_REQUIRE(q && k_cache && v_cache && k_scale && v_scale && out && cache_seqlens && workspace, IFV2_ERR_INVALID_ARG,
               "q8_decode: null pointer");
  IFV2_REQUIRE((k_new == nullptr) == (v_new == nullptr), IFV2_ERR_INVALID_ARG, "q8_decode: pass both k_new and v_new, or neither");
  const bool rotate = rotary_cos != nullptr;
  IFV2_REQUIRE(rotate == (rotary_sin != nullptr) && (!rotate || k_new), IFV2_ERR_INVALID_ARG,
               "q8_decode: rotation takes both tables and a new key");
  const bool listed = topk_idx != nullptr && topk >= 0 && topk <= kMaxList;      // the split kernel takes short lists as they are
  if (listed) mask = nullptr;
  IFV2_REQUIRE(topk_idx == nullptr || listed || (mask != nullptr && topk >= 0), IFV2_ERR_INVALID_ARG,
               "q8_decode: lists of more than %d blocks need a mask buffer", kMaxList);
  IFV2_REQUIRE(mask == nullptr || mask_words >= 1, IFV2_ERR_INVALID_ARG, "q8_decode: mask_words < 1");
  IFV2_REQUIRE(topk_idx == nullptr || listed || mask_words <= 4096, IFV2_ERR_TOO_LARGE, "q8_decode: more than 4096 mask words");
  if (block_table != nullptr) {
    IFV2_REQUIRE(length % 16 == 0 && block_table_stride >= 1, IFV2_ERR_INVALID_ARG,
                 "q8_decode: page size must be a positive multiple of 16");
    IFV2_REQUIRE(cache_batch_idx == nullptr, IFV2_ERR_UNSUPPORTED, "q8_decode: a paged cache takes no cache_batch_idx");
  } else {
    IFV2_REQUIRE(cache_batch_idx != nullptr || slots >= batch, IFV2_ERR_INVALID_ARG, "q8_decode: fewer slots than sequences");
  }
  IFV2_REQUIRE(length <= INT32_MAX && slots <= INT32_MAX && slots * length <= INT32_MAX / heads_k, IFV2_ERR_TOO_LARGE,
               "q8_decode: the cache has more than 2^31-1 rows");
  const int64_t capacity = block_table != nullptr ? (int64_t)block_table_stride * length : length;
  IFV2_REQUIRE(capacity <= INT32_MAX - kBlockN, IFV2_ERR_TOO_LARGE, "q8_decode: more than 2^31-1 positions");
  IFV2_REQUIRE(batch <= 65535 && heads_k <= 65535 && (int64_t)batch * heads_k <= 65535, IFV2_ERR_TOO_LARGE,
               "q8_decode: more than 65535 sequences x KV heads");
  IFV2_REQUIRE(workspace_bytes >= ifv2_q8_decode_workspace_bytes(batch, heads_q, head_dim), IFV2_ERR_INVALID_ARG,
               "q8_decode: workspace too small");
  for (const void* ptr : {q, (const void*)k_cache, (const void*)v_cache, (const void*)workspace, (const void*)out, k_new, v_new})
    IFV2_REQUIRE(reinterpret_cast<uintptr_t>(ptr) % 16 == 0, IFV2_ERR_INVALID_ARG, "q8_decode: tensors must be 16-byte aligned");
  Q8DecodeParams p{};
  if (rotate) {
    int rc = make_rotary(&p.rotary, "q8_decode", rotary_cos, rotary_sin, rotary_positions ? rotary_positions : cache_seqlens,
                         rotary_positions ? axis_stride : 0, pair_axis, axes, rotary_dim, table_rows, interleaved);
    if (rc) return rc;
  }
  p.rotate = rotate;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.k_codes = static_cast<uint8_t*>(k_cache);
  p.v_codes = static_cast<uint8_t*>(v_cache);
  p.k_scale = static_cast<uint8_t*>(k_scale);
  p.v_scale = static_cast<uint8_t*>(v_scale);
  // Where sequences may share rows (pages, slots by index) the new rows are all written before any is attended; slots
  // that belong to one sequence each get them from the CTA that attends the new token's block.
  const bool shared_rows = block_table != nullptr || cache_batch_idx != nullptr;
  if (!shared_rows) {
    p.k_new = static_cast<const __nv_bfloat16*>(k_new);
    p.v_new = static_cast<const __nv_bfloat16*>(v_new);
  }
  p.mask = reinterpret_cast<const unsigned long long*>(mask);
  p.mask_words = mask_words;
  p.topk_idx = listed ? topk_idx : nullptr;
  p.topk = topk;
  p.cache_seqlens = cache_seqlens;
  p.place = Place{block_table, cache_batch_idx, block_table_stride, heads_k, (int)length, (int)slots};
  p.capacity = capacity;
  // x / d for x < 2^31: with 2^(s - 1) < d <= 2^s and m = floor(2^(31 + s) / d) + 1 < 2^32, x m / 2^(31 + s) is past x / d by
  // less than 2^-s <= 1 / d.  (d = length >= 16 where it is used)
  if (block_table != nullptr) {
    int s = 1;
    while (((int64_t)1 << s) < length) ++s;
    p.page_mul = (uint32_t)(((uint64_t)1 << (31 + s)) / (uint64_t)length + 1);
    p.page_shift = s - 1;
  }
  p.batch = batch;
  p.heads_k = heads_k;
  p.new_tokens = k_new != nullptr;
  p.scale_log2 = softmax_scale * kLog2e;
  p.partial = static_cast<float*>(workspace);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.lse = lse;
  const int64_t pairs = (int64_t)batch * heads_k;
  const int64_t n_blocks = ceil_div64(capacity, kBlockN);
  IFV2_REQUIRE(pairs * (n_blocks + kStart) <= INT32_MAX, IFV2_ERR_TOO_LARGE, "q8_decode: more than 2^31-1 blocks of 64 keys");
  const bool selected = listed || mask != nullptr;
  p.most_blocks = !selected ? (int)n_blocks : topk_idx != nullptr && topk > 0 ? topk : kUsualBlocks;
  p.splits = selected ? plan_splits(pairs, p.most_blocks) : 0;
  cudaStream_t st = (cudaStream_t)stream;
  const bool packed = topk_idx != nullptr && !listed, prepared = (k_new != nullptr && shared_rows) || packed;
  if (prepared) {
    const Q8PrepareParams a{shared_rows ? static_cast<const __nv_bfloat16*>(k_new) : nullptr, static_cast<const __nv_bfloat16*>(v_new),
                            static_cast<uint8_t*>(k_cache), static_cast<uint8_t*>(v_cache), static_cast<uint8_t*>(k_scale),
                            static_cast<uint8_t*>(v_scale), packed ? topk_idx : nullptr, reinterpret_cast<unsigned long long*>(mask), topk, mask_words};
    const size_t smem = packed ? (size_t)mask_words * 8 : 0;
    if (code == kE4m3) q8_prepare_kernel<kE4m3><<<dim3(heads_k, batch), kThreads, smem, st>>>(a, p);
    else q8_prepare_kernel<kInt8><<<dim3(heads_k, batch), kThreads, smem, st>>>(a, p);
    int rc = check_launch("q8_prepare");
    if (rc) return rc;
  }
  // the scale bytes of a unit are together, at a multiple of 16 bytes
  const bool copied = length % kUnit == 0 && ((reinterpret_cast<uintptr_t>(k_scale) | reinterpret_cast<uintptr_t>(v_scale)) & 15) == 0;
  const int page = block_table == nullptr ? 0 : copied ? 32 : 16;
  CUtensorMap map_k, map_v;
  const uint64_t rows = (uint64_t)slots * heads_k * length;
  int rc = make_tensor_map_rows128(&map_k, k_cache, rows, page == 16 ? 16 : 32);
  if (rc == IFV2_OK) rc = make_tensor_map_rows128(&map_v, v_cache, rows, page == 16 ? 16 : 32);
  if (rc) return rc;
  auto kernel = rotate ? (code == kE4m3 ? split_kernel<kE4m3, true>(page, copied) : split_kernel<kInt8, true>(page, copied))
                       : (code == kE4m3 ? split_kernel<kE4m3, false>(page, copied) : split_kernel<kInt8, false>(page, copied));
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
  if (e != cudaSuccess) return set_error((int)e, "q8_decode: %s", cudaGetErrorString(e));
  int64_t grid = pairs * p.splits;
  if (p.splits == 0) {
    grid = pairs * (kStart + (n_blocks < p.most_blocks ? n_blocks : p.most_blocks));
    if (grid > kMaxCtas) grid = kMaxCtas;
  }
  e = launch_kernel(kernel, dim3((unsigned)grid), kThreads, kSmemBytes, st, prepared, map_k, map_v, p);
  if (e != cudaSuccess) return set_error((int)e, "q8_split: launch failed: %s", cudaGetErrorString(e));
  if (p.splits == 1) return IFV2_OK;               // the split kernel wrote the results
  const int64_t per_pair = p.splits ? p.splits : ceil_div64(grid, pairs);
  const int warps = per_pair > 16 ? 8 : per_pair > 6 ? 4 : 1;      // that share a row's partials
  auto join = warps == 8 ? q8_combine_kernel<8> : warps == 4 ? q8_combine_kernel<4> : q8_combine_kernel<1>;
  e = launch_kernel(join, dim3(2 * warps, (unsigned)pairs), 256, 0, st, true, p, (int)grid);
  if (e != cudaSuccess) return set_error((int)e, "q8_combine: launch failed: %s", cudaGetErrorString(e));
  return IFV2_OK;
}
