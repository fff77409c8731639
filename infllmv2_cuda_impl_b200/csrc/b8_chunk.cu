// Attention over 8-bit blocks for several new tokens per sequence: drafts and prompts' chunks (formulas, operands and
// shares: b8_attn.cuh).
//
// Eight tokens x 16 heads are the M side:
//     S (128 rows x 128 keys)      = [Q1 + Q2] . K^T     codes as they lie, two products into one sum (kind::f8f6f4)
//     O (128 rows x 128 features) += W . V               fp16 weights in TMEM, values made fp16 by four warps (kind::f16)
// Here the weights are many (128 x 128 per unit) and the values' codes are not: three 8-bit terms of every weight cost the
// softmax 3.75 instructions for a weight of 6, conversion of V costs 0.75 per code and is shared by all rows.  (For one or two
// tokens it is the other way round, b8_decode.cu.)  fp16 holds a weight to 2^-11 and down to 2^-24.
//
// Units go to two groups of four softmax warps in turn (thread = row).  Each group has a score buffer, its weights over
// the scores, and sums of its own (M, l, O), so that neither waits for the other; the two are put together at the end
// of the tile.  TMEM: two S and two O of 128 columns, all there is, so scores are made by blocks of 64 keys: a block's
// next scores and the product of its weights are under way while the group works on the unit's other block (by whole
// units a group waited 1200 of 4600 clocks for its next scores).  Warps: 0 looks blocks up and issues TMA, 1 issues the MMAs
// of the scores, 2..5 and 6..9 are the groups, 10..13 convert values, 14 issues the MMAs of the values.  (One warp that
// issued both took 1050 clocks for a block's 12 MMAs and their waits, and paced everything.)
//
// What bounds it: a unit takes 2150 clocks.  Its exponentials need 1024 of them in the special-function units, its products 1024
// in the tensor cores, and shared memory 1660 (scores of 64 keys read the query again; values are read, written as fp16 and
// read by the product).  A chunk of 4096 tokens over 32768: 1.85 ms (2.0 under the power cap), 1.1 PFLOP/s of the attention's own
// FLOPs (a third of the products serves the query's second term).  Where tokens select blocks a tile walks the union of theirs, and
// every warp takes the exponentials of all of it: 2048 tokens over 65536, 64 blocks each, 345 us where the selected pairs' FLOPs take 82.  Tried and slower: scores of whole units; 16 softmax warps, two to a row's 32 keys
// each (1880 -> 2167 us: the vote that holds them together); scores fetched from TMEM in halves; masked and unmasked
// forms of the weights' code.
#include "b8_attn.cuh"

namespace ifv2 {
namespace {

using namespace b8;

constexpr int kT = 8, kRows = kT * kGroup;
constexpr int kThreads = 480, kSoftmax = 256;
constexpr int kStages = 3;
constexpr int kQBytes = kRows * kHeadDim;         // one of two terms
constexpr int kVBytes = kUnit * kHeadDim * 2;     // fp16 values of a unit: two halves of 64 features, a row per key
constexpr int kV = 2 * kQBytes, kRing = kV + 2 * kVBytes, kSmem = kRing + kStages * 2 * kTileBytes + 1024;
// Every row has two references.  M is for what goes to the tensor cores: weights are 2^(x + eV - M).  A new one puts the largest
// weight at 2^kFirst; it moves when a block's weights add up to more than kMost.  R is for the sum l = sum 2^(x - R), in which the
// values' sizes have no part: it moves when a score is more than kApart above it.  A block adds 2^(M - R - eV) of its weights' sum;
// that is at most 2^kDeep: where eV is less, the weights are taken with M - R - kDeep in its place, below 2^(kApart - kDeep)
// (nothing in fp16) unless they add up to kLeast, which shows that R is too low.
constexpr float kFirst = 4.f, kMost = 32768.f, kApart = 20.f, kDeep = 86.f, kLeast = 0x1p-30f;

// Instruction descriptor, kind::f16 with fp16 operands, B MN-major.
constexpr uint32_t kIdescValues = (1u << 4) | (1u << 16) | (128u >> 3 << 17) | (128u >> 4 << 24);

// A row's 64 weights of a block as fp16 pairs, 2^(x c + b), 0 from key `see` on; returns their sum.
__device__ __forceinline__ float weights(uint32_t scores, uint32_t (&w)[32], float c, float b, bool all, int see) {
  uint32_t x[64];
  tmem_ld64_wait(scores, x);
  if (!all) {
#pragma unroll
    for (int j = 0; j < kBlockN; ++j)
      if (j >= see) x[j] = 0xFF800000u;
  }
  const uint64_t b2 = pack_f32x2(b, b), c2 = pack_f32x2(c, c);
  uint64_t sum2 = 0, sum2b = 0;
#pragma unroll
  for (int j = 0; j < kBlockN; j += 4) {
    float y[4];
    unpack_f32x2(fma_f32x2(pack_f32x2(x[j], x[j + 1]), c2, b2), y[0], y[1]);
    unpack_f32x2(fma_f32x2(pack_f32x2(x[j + 2], x[j + 3]), c2, b2), y[2], y[3]);
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = ex2(y[e]);
    sum2 = add_f32x2(sum2, pack_f32x2(y[0], y[1]));
    sum2b = add_f32x2(sum2b, pack_f32x2(y[2], y[3]));
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[j / 2]) : "f"(y[1]), "f"(y[0]));
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[j / 2 + 1]) : "f"(y[3]), "f"(y[2]));
  }
  float s0, s1;
  unpack_f32x2(add_f32x2(sum2, sum2b), s0, s1);
  return s0 + s1;
}

template <int kCode, bool kListed, bool kSelected>
__global__ void __launch_bounds__(kThreads, 1)
b8_chunk_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const AttnParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ Common<kT, kStages> s;
  // by group, and by block of a unit
  __shared__ uint64_t bar_s[2][2], bar_p[2][2], bar_v[2][2], bar_pv[2][2], bar_q, bar_drain[2];
  __shared__ float s_c[kRows], s_top[2][kRows], s_lse[2][kRows];       // row's factor; a group's M and log2 of its sum
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  __shared__ int s_cost[kThreads / 32];
  __shared__ Item s_now;                           // the softmax's item, for its end (in registers it was spilled)
  volatile int* gave_up = &s.gave_up;

  if (tid == 64) {
    s.gave_up = 0;
    for (int i = 0; i < kStages; ++i) mbar_init(&s.full[i], 2), mbar_init(&s.empty[i], 9);
    for (int i = 0; i < 2; ++i) {
      for (int h = 0; h < 2; ++h)
        mbar_init(&bar_s[i][h], 1), mbar_init(&bar_p[i][h], 4), mbar_init(&bar_v[i][h], 4), mbar_init(&bar_pv[i][h], 1);
      mbar_init(&s.item_full[i], 1), mbar_init(&s.item_empty[i], 14);
    }
    mbar_init(&bar_q, 8);
    mbar_init(&bar_drain[0], 1), mbar_init(&bar_drain[1], 1);
    fence_barrier_init();
    prefetch_tensormap(&k_map);
    prefetch_tensormap(&v_map);
  }
  if (warp == 1) {
    tmem_alloc(&s.tmem, 512);
    tmem_relinquish();
  }
  wait_inputs();
  Deal<kT, kListed, kSelected> deal;
  deal.add_up(p, s_cost);
  __syncthreads();
  if (warp == 0) deal.work_out(p, s_cost);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  allow_next();
  const uint32_t tmem = s.tmem;                    // S of group g at 128 g, O at 256 + 128 g

  if (warp == 0) {
    fetch<kT, kStages, kListed, kSelected>(p, &k_map, &v_map, s, smem + kRing, deal);
  } else if (warp == 1) {
    // ---------------------------------------------------------------- scores
    if (elect_one()) {
      const uint32_t base = smem_u32(smem);
      constexpr uint32_t kIdescS = umma_idesc_f8(128, kBlockN, kE4m3, kCode, false, false);
      const uint32_t q_lo = umma_desc_lo(base, 16);
      bool ok = true;
      int n0 = 0, queries = 0;
      const auto scores = [&](int n, int h) {                // S of a unit's block
        const int stage = n % kStages;
        ok = ok && bounded_wait(&s.full[stage], (n / kStages) & 1, gave_up);
        if (!ok) return;
        tc_fence_after();
        const uint32_t k_lo = umma_desc_lo(base + kRing + stage * 2 * kTileBytes + h * (kTileBytes / 2), 16);
        const uint32_t to = tmem + 128 * (n & 1) + kBlockN * h;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            umma_f8_ss_lo(to, q_lo + ((j * kQBytes + kk * 32) >> 4), k_lo + ((kk * 32) >> 4), kUmmaDescHi, kIdescS, j + kk > 0);
        umma_commit(&bar_s[n & 1][h]);
        if (h == 1) umma_commit(&s.empty[stage]);
      };
      for (int item = 0; ok; ++item) {
        ok = bounded_wait(&s.item_full[item & 1], (item >> 1) & 1, gave_up);
        const int units = ok ? s.item[item & 1].units : -1;
        if (units < 0) break;
        mbar_arrive(&s.item_empty[item & 1]);
        if (units == 0) continue;
        ok = bounded_wait(&bar_q, queries++ & 1, gave_up);
        // scores are written over weights: the product that reads these is waited for
        for (int n = max(n0 - 2, 0); n < n0; ++n) ok = ok && bounded_wait(&bar_pv[n & 1][1], (n >> 1) & 1, gave_up);
        for (int i = 0; i < min(units, 2); ++i)
          for (int h = 0; h < 2; ++h) scores(n0 + i, h);
#pragma unroll 1
        for (int i = 2; ok && i < units; i += 2)
#pragma unroll 1
          for (int h = 0; ok && h < 2; ++h)
#pragma unroll 1
            for (int u = i; ok && u < min(i + 2, units); ++u) {
              const int n = n0 + u;
              ok = bounded_wait(&bar_pv[n & 1][h], ((n - 2) >> 1) & 1, gave_up);
              scores(n, h);
            }
        n0 += units;
      }
      if (!ok) {
        umma_commit(&bar_drain[0]);
        mbar_wait_drain(&bar_drain[0], 0);
      }
    }
    __syncwarp();
  } else if (warp == 14) {
    // ---------------------------------------------------------------- values
    if (elect_one()) {
      const uint32_t base = smem_u32(smem);
      bool ok = true;
      int n0 = 0;
      for (int item = 0; ok; ++item) {
        ok = bounded_wait(&s.item_full[item & 1], (item >> 1) & 1, gave_up);
        const int units = ok ? s.item[item & 1].units : -1;
        if (units < 0) break;
        mbar_arrive(&s.item_empty[item & 1]);
#pragma unroll 1
        for (int i = 0; ok && i < units; i += 2)
#pragma unroll 1
          for (int h = 0; ok && h < 2; ++h)
#pragma unroll 1
            for (int u = i; ok && u < min(i + 2, units); ++u) {
              const int n = n0 + u, g = n & 1;
              ok = bounded_wait(&bar_v[g][h], (n >> 1) & 1, gave_up) && bounded_wait(&bar_p[g][h], (n >> 1) & 1, gave_up);
              if (!ok) break;
              tc_fence_after();
              const uint32_t v_lo = umma_desc_lo(base + kV + g * kVBytes + h * (kVBytes / 4), kVBytes / 2);
              const uint32_t w = tmem + 128 * g + kBlockN * h;
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                umma_ts_lo(tmem + 256 + 128 * g, w + 8 * kk, v_lo + ((kk * 2048) >> 4), kIdescValues, u >= 2 || h + kk > 0);
              umma_commit(&bar_pv[g][h]);
            }
        n0 += units;
      }
      if (!ok) {
        umma_commit(&bar_drain[1]);
        mbar_wait_drain(&bar_drain[1], 0);
      }
    }
    __syncwarp();
  } else if (warp >= 10) {
    // ---------------------------------------------------------------- values to fp16
    // A warp takes 8 rows x 64 features at a time, a thread 16 features.  Eight neighbouring threads have pieces of two rows whose
    // numbers differ by 5 in the swizzle (bits 0 and 2), so that neither their reads nor their writes, of every other
    // 16-byte piece, meet in a bank.
    const int cwarp = warp - 10, quarter = lane >> 3, c = lane & 3, at = lane & 4 ? quarter ^ 5 : quarter;      // at: row of eight
    const int from0 = (cwarp * 16 + at) * kHeadDim + ((c ^ at) << 4), to0 = (cwarp * 16 + at) * 128 + (((2 * c) ^ at) << 4);
    int n = 0;
    for (int item = 0;; ++item) {
      if (!bounded_wait_warp(&s.item_full[item & 1], (item >> 1) & 1, gave_up)) break;
      const int units = s.item[item & 1].units;
      if (units < 0) break;
      mbar_arrive_warp(&s.item_empty[item & 1]);
      for (int i = 0; i < units; ++i, ++n) {
        const int stage = n % kStages, g = n & 1;
        bounded_wait_warp(&s.full[stage], (n / kStages) & 1, gave_up);
        // (of a page that is not there another one is read in its place: its values may be anything, and count as rows that are no keys)
        int valid[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) valid[h] = s.block[stage][h].e_v == kNanScale ? 0 : s.block[stage][h].valid & 0xFF;
        const uint8_t* tile = smem + kRing + stage * 2 * kTileBytes + kTileBytes;
        uint8_t* place = smem + kV + g * kVBytes;
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          if (n >= 2) bounded_wait_warp(&bar_pv[g][h], ((n - 2) >> 1) & 1, gave_up);      // the block's place is free again
          const int have = (h ? valid[1] : valid[0]) - cwarp * 16 - at;      // > 8 j: the thread's row in step j is a key
          const uint8_t* from = tile + h * (kTileBytes / 2);
          uint8_t* to = place + h * (kVBytes / 4);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int j = i >> 1, half = i & 1;    // eight rows, 64 features
            uint4 x = *reinterpret_cast<const uint4*>(from + (from0 ^ (half << 6)) + j * 8 * kHeadDim);
            // a value row that is no key may hold anything: 0 x NaN
            if (have <= 8 * j) x = make_uint4(0, 0, 0, 0);
            uint32_t y[8];
            const uint32_t* w = reinterpret_cast<const uint32_t*>(&x);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if (kCode == kE4m3) {
                asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
                    : "=r"(y[2 * k]), "=r"(y[2 * k + 1]) : "r"(w[k]));
              } else {                             // the upper bytes of fp16 numbers
                y[2 * k] = __byte_perm(w[k], 0u, 0x1404);
                y[2 * k + 1] = __byte_perm(w[k], 0u, 0x3424);
              }
            }
            uint8_t* at_half = to + half * (kVBytes / 2) + j * 8 * 128;
            *reinterpret_cast<uint4*>(at_half + to0) = make_uint4(y[0], y[1], y[2], y[3]);
            *reinterpret_cast<uint4*>(at_half + (to0 ^ 16)) = make_uint4(y[4], y[5], y[6], y[7]);
          }
          fence_proxy_async_smem();
          mbar_arrive_warp(&bar_v[g][h]);
        }
        mbar_arrive_warp(&s.empty[stage]);
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax
    // A wait that gave up makes the tile's results NaN, the CTA's tiles behind it are not written, and the status block says so.
    // Within an item every thread keeps to the same loops and barriers.
    const int group = (warp - 2) >> 2, quad = warp & 3, r = quad * 32 + lane;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const uint32_t my_s = tmem + 128 * group + lanes, my_o = tmem + 256 + 128 * group + lanes;
    const int stid = tid - 64;
    const int heads = p.heads_k * kGroup;

    // Query rows of an item: 8 threads per row, 16 values each.
    // (two tokens at a time, the next ones' values on their way; code that runs once per tile is kept short, since every line of
    // it comes from far away)
    const auto write_query = [&](const Item& t) {
      const int c = stid & 7, of_pair = stid >> 3;
      const __nv_bfloat16* src = p.q + ((int64_t)(t.row + of_pair / kGroup) * heads + t.head * kGroup + of_pair % kGroup) * kHeadDim + c * 16;
      const auto load = [&](int i, uint4 (&x)[2]) {
        x[0] = x[1] = make_uint4(0, 0, 0, 0);
        if (2 * i + of_pair / kGroup < t.tokens) {
          const uint4* at = reinterpret_cast<const uint4*>(src + (int64_t)2 * i * heads * kHeadDim);
          x[0] = *at, x[1] = *(at + 1);
        }
      };
      uint4 x[2];
      load(0, x);
#pragma unroll 1
      for (int i = 0; 2 * i < t.tokens; ++i) {
        uint4 y[2];
        load(i + 1, y);
        const int row = 32 * i + of_pair;
        const float f = write_query16(x, smem + row * kHeadDim + ((c ^ (row & 7)) << 4), kQBytes, p.scale_log2);
        if (c == 0) s_c[row] = f;
        x[0] = y[0], x[1] = y[1];
      }
      fence_proxy_async_smem();
      mbar_arrive_warp(&bar_q);
    };
    Item next;
    const auto next_item = [&](int item) {
      const bool ok = bounded_wait_warp(&s.item_full[item & 1], (item >> 1) & 1, gave_up);
      if (named_any<kSoftmax>(!ok)) {
        next.units = -1;
        return;
      }
      next = s.item[item & 1];
      mbar_arrive_warp(&s.item_empty[item & 1]);
    };

    // O times f, once the group's product before the one of unit n, block h, has been made
    const auto rescale = [&](float f, int n, int h) {
      bounded_wait_warp(&bar_pv[group][h ^ 1], ((h ? n : n - 2) >> 1) & 1, gave_up);
      tc_fence_after();
#pragma unroll 1
      for (int c0 = 0; c0 < kHeadDim; c0 += 32) {
        uint32_t o[32];
        tmem_ld32_wait(my_o + c0, o);
#pragma unroll
        for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
        tmem_st32(my_o + c0, o);
      }
    };

    int n0 = 0;                                    // units of earlier items
    next_item(0);
    if (next.units > 0) write_query(next);
    named_sync<kSoftmax>();
    for (int item = 0; next.units >= 0; ++item) {
      if (stid == 0) s_now = next;
      const struct { int tokens, reach, units; } t{next.tokens, next.reach, next.units};
      const int tok = r / kGroup;
      // keys that the row sees; rows of tokens that the tile does not have see what the last one does, for nobody
      const int limit = tok < t.tokens && p.causal ? t.reach - (t.tokens - 1 - tok) : t.reach;
      const uint32_t bit = 1u << min(tok, t.tokens - 1);
      const bool idle = 2 * quad >= t.tokens;      // nor does the warp have another
      const float c_row = s_c[r];
      const bool c_nan = !(c_row == c_row);
      float m = kUnset, ref = 0.f, l = 0.f;        // M; R; the sum in units of 2^R
      bool begun = false;                          // O holds something
#pragma unroll 1
      for (int i = (n0 & 1) ^ group; i < t.units; i += 2) {
        const int n = n0 + i, stage = n % kStages;
        bounded_wait_warp(&s.full[stage], (n / kStages) & 1, gave_up);
        const Block blk[2] = {s.block[stage][0], s.block[stage][1]};
        mbar_arrive_warp(&s.empty[stage]);
        if (idle) {                                // (what lies in its rows stays in its rows)
#pragma unroll 1
          for (int h = 0; h < 2; ++h) {
            bounded_wait_warp(&bar_s[group][h], (n >> 1) & 1, gave_up);
            mbar_arrive_warp(&bar_p[group][h]);
          }
          continue;
        }
        // Of both blocks: keys that the row sees, factor of the scores.  Nearly every unit is plain (every row sees all of it, see
        // Block): the rest of this is for the others.
        int seen[2] = {kBlockN, kBlockN};
        float cs[2];
        bool all_seen[2] = {true, true}, odd = false;      // odd: a NaN among the warp's numbers
        if (blk[0].valid & kPlain) {
#pragma unroll
          for (int h = 0; h < 2; ++h) cs[h] = q8::mul_exact(c_row, blk[h].k_scale);
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            seen[h] = blk[h].tokens & bit ? max(min(limit - blk[h].pos, blk[h].valid & 0xFF), 0) : 0;
            all_seen[h] = __all_sync(0xFFFFFFFFu, seen[h] == kBlockN);
            cs[h] = fmaxf(q8::mul_exact(c_row, blk[h].k_scale), 1e-37f);     // (-inf of a masked key times 0 would be NaN)
            odd |= !(blk[h].k_scale == blk[h].k_scale) || blk[h].e_v == kNanScale;
          }
          odd = __any_sync(0xFFFFFFFFu, odd || c_nan);
        }
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          const int see = h ? seen[1] : seen[0], e_v = h ? blk[1].e_v : blk[0].e_v;
          const bool all = h ? all_seen[1] : all_seen[0];
          // (a block without an exponent has no keys or NaN values: any will do)
          const float c = h ? cs[1] : cs[0], ev = e_v > kNoScale && e_v < kNanScale ? (float)e_v : 0.f;
          uint32_t w[32];
          bounded_wait_warp(&bar_s[group][h], (n >> 1) & 1, gave_up);
          tc_fence_after();
          float sum = 0.f, up = 0.f;
#pragma unroll 1
          for (bool again = false;; again = true) {
            if (again) {
              // the row's largest score: new references where it is above the old ones (whole numbers, so that what follows from
              // them is exact)
              float top = -INFINITY;
#pragma unroll 1
              for (int j0 = 0; j0 < kBlockN; j0 += 16) {
                uint32_t x[16];
                tmem_ld16(my_s + kBlockN * h + j0, x);
                tmem_wait_ld();
#pragma unroll
                for (int j = 0; j < 16; ++j)
                  if (j0 + j < see) top = fmaxf(top, __uint_as_float(x[j]));
              }
              const float k_scale = h ? blk[1].k_scale : blk[0].k_scale;
              top = c_nan || !(k_scale == k_scale) ? -INFINITY : top * c;
              float f = 1.f;
              if (top > -INFINITY && (m == kUnset || top - ref > kApart)) {
                const float now = ceilf(top - kFirst);
                l = l > 0.f ? l * ex2(ref - now) : l;
                ref = now;
              }
              if (top + ev - m > kFirst) {
                const float now = ceilf(top + ev - kFirst);
                f = m == kUnset ? 0.f : ex2(m - now);
                m = now;
              }
              __syncwarp();
              if (begun) rescale(f, n, h);
            }
            // 2^-t: the block's sum in units of the row's; past 2^kDeep the block's values are too small to matter, and its
            // weights are taken to be larger than they are, so that the keys still count in l
            const float t = m - ref - ev;
            up = fminf(t, kDeep);
            sum = weights(my_s + kBlockN * h, w, c, -(ref + up), all, see);
            if (again || !(__any_sync(0xFFFFFFFFu, !(sum <= (t > kDeep ? kLeast : kMost))) || odd)) break;
          }
          if (odd) {
            const float k_scale = h ? blk[1].k_scale : blk[0].k_scale;
            const bool nan_key = c_nan || !(k_scale == k_scale), nan_value = e_v == kNanScale;
            if (nan_key) sum = see > 0 ? NAN : 0.f;
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              const uint32_t here = (2 * j < see ? 0xFFFFu : 0u) | (2 * j + 1 < see ? 0xFFFF0000u : 0u);
              if (nan_key || nan_value) w[j] = here & 0x7FFF7FFFu;
            }
          }
          begun = true;
          tmem_st32(my_s + kBlockN * h, w);
          l += sum * ex2(up);
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive_warp(&bar_p[group][h]);
        }
      }
      s_top[group][r] = m;
      s_lse[group][r] = l == 0.f ? -INFINITY : ref + lg2(l);
      // the next item's query, while the last products run (every S of this item has been read)
      next_item(item + 1);
      if (next.units > 0) write_query(next);

      // ---- the item's results: each group has half of the features
      const Item of = s_now;
      const int n1 = n0 + of.units;
      for (int n = max(n1 - 2, n0); n < n1; ++n) bounded_wait_warp(&bar_pv[n & 1][1], (n >> 1) & 1, gave_up);
      tc_fence_after();
      const float lse0 = s_lse[0][r], lse1 = s_lse[1][r];
      const bool lost = *gave_up;                  // a wait ran out: nothing here can be trusted
      const float most = fmaxf(lse0, lse1), nan = lost ? NAN : lse0 != lse0 ? lse0 : lse1 != lse1 ? lse1 : 0.f;
      const bool none = most == -INFINITY;
      const float lse2 = none ? -INFINITY + nan : most + lg2(ex2(lse0 - most) + ex2(lse1 - most)) + nan;
      if (group == 0 && tok < of.tokens) {
        if (of.piece >= 0) p.part_lse[(int64_t)of.piece * kRows + r] = lse2;
        else if (p.lse) p.lse[(int64_t)(of.row + tok) * heads + of.head * kGroup + r % kGroup] = none && nan == 0.f ? INFINITY : lse2 * kLn2;
      }
      // 2^(M - lse) in two steps, so that neither leaves fp32's range; below 0: the group has no key of this row's.  (A product
      // that 2^(M - lse) makes 0 is added all the same: it is NaN where the row sees a NaN block.)
      float f[2];
      bool with[2];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        with[g] = of.units > (g ^ (n0 & 1));        // this group had a unit
        f[g] = none ? nan : ex2(0.5f * (s_top[g][r] - lse2));
        if (s_lse[g][r] == -INFINITY) f[g] = -1.f;
      }
      __nv_bfloat16* out = p.out + ((int64_t)(of.row + tok) * heads + of.head * kGroup + r % kGroup) * kHeadDim + 64 * group;
      float* part = p.part_o + ((int64_t)max(of.piece, 0) * kRows + r) * kHeadDim + 64 * group;
#pragma unroll 1
      for (int c0 = 0; c0 < 64; c0 += 16) {
        float y[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) y[j] = nan;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          if (!with[g]) continue;
          uint32_t o[16];
          __syncwarp();
          tmem_ld16(tmem + 256 + 128 * g + lanes + 64 * group + c0, o);
          tmem_wait_ld();
          if (!(f[g] < 0.f)) {
#pragma unroll
            for (int j = 0; j < 16; ++j) y[j] += q8::mul_exact(q8::mul_exact(__uint_as_float(o[j]), f[g]), f[g]);
          }
        }
        if (tok < of.tokens && of.piece < 0) {
          uint4 a, b;
          a.x = pack_bf16(y[0], y[1]), a.y = pack_bf16(y[2], y[3]), a.z = pack_bf16(y[4], y[5]), a.w = pack_bf16(y[6], y[7]);
          b.x = pack_bf16(y[8], y[9]), b.y = pack_bf16(y[10], y[11]), b.z = pack_bf16(y[12], y[13]), b.w = pack_bf16(y[14], y[15]);
          reinterpret_cast<uint4*>(out + c0)[0] = a;
          reinterpret_cast<uint4*>(out + c0)[1] = b;
        } else if (tok < of.tokens) {
#pragma unroll
          for (int j = 0; j < 16; j += 4) *reinterpret_cast<float4*>(part + c0 + j) = make_float4(y[j], y[j + 1], y[j + 2], y[j + 3]);
        }
      }
      tc_fence_before();
      named_sync<kSoftmax>();
      n0 = n1;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && s.gave_up) atomicCAS(p.status + 1, 0, 102);
  if (warp == 1) tmem_dealloc(s.tmem, 512);
}

template <int kCode, bool kListed, bool kSelected>
int launch(const CUtensorMap& k_map, const CUtensorMap& v_map, const AttnParams& p, cudaStream_t stream) {
  static std::atomic<uint64_t> allowed{0};
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(b8_chunk_kernel<kCode, kListed, kSelected>), kSmem, allowed);
  if (e == cudaSuccess)
    e = launch_beside(b8_chunk_kernel<kCode, kListed, kSelected>, dim3(kB8ChunkGrid), kThreads, kSmem, stream, k_map, v_map, p);
  if (e != cudaSuccess) return set_error((int)e, "b8_attn: %s", cudaGetErrorString(e));
  return check_launch("b8_attn");
}

template <int kCode>
int launch_with(const CUtensorMap& k_map, const CUtensorMap& v_map, const AttnParams& p, bool listed, cudaStream_t stream) {
  const bool selected = p.mask != nullptr || p.lists != nullptr;
  if (listed) return selected ? launch<kCode, true, true>(k_map, v_map, p, stream) : launch<kCode, true, false>(k_map, v_map, p, stream);
  return selected ? launch<kCode, false, true>(k_map, v_map, p, stream) : launch<kCode, false, false>(k_map, v_map, p, stream);
}

}  // namespace

int b8_launch_chunk(const CUtensorMap& k_map, const CUtensorMap& v_map, const AttnParams& p, bool listed, int code, cudaStream_t stream) {
  return code == kE4m3 ? launch_with<kE4m3>(k_map, v_map, p, listed, stream) : launch_with<kE5m2>(k_map, v_map, p, listed, stream);
}

}  // namespace ifv2
