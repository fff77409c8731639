// Attention over 8-bit blocks for one or two new tokens per sequence (formulas, operands and shares: b8_attn.cuh).
//
// Keys are the M side of both products, so that few query rows cost few tensor clocks:
//     S^T (128 keys x 16 kT)            = K . [Q1 + Q2]^T   the query's two terms one after the other
//     O^T (128 features x 3 x 16 kT)   += V^T . [W1 W2 W3]  V is MN-major as it lies; W is written [key][column], its terms
//                                                           side by side, so that four MMAs serve all of them: the next
//                                                           unit's weights wait for this product, not for the scores
// A softmax thread has a key of its own, with the tile's columns in registers: a decode step's exponentials are spread
// over all lanes.  Warps: 0 looks blocks up and issues TMA, 1 issues MMAs, 2..5 are the softmax (thread = key =
// feature).  Two CTAs per SM.
//
// What bounds it is memory, and at both ends latency.  64 sequences of 16000 tokens, 2 KV heads: 87 us with the join, 6.1 TB/s,
// 93 % of the copy bandwidth.  64 selected blocks of 64 sequences, 135 MB: 34-36 us where the bytes take 21: 5 us until the first
// unit is there (lengths, list, page, tile: each a trip to memory of 0.7 us), CTAs that end some us apart, and the join.  Short
// sequences pay for the start and end of tiles: 4096 of 200 tokens 169 us where the bytes take 65.  Two tokens, 64 sequences of
// 16000: 130 us.
// Registers decide: with the columns' factors and references in them 30 words were spilled, and every call took 5 us more.  (The
// two-token forms still spill: four words, eight where blocks are selected.)
// Tried and slower or equal: four sequences per lane in the deal (one sequence +0.6 us, 256 sequences -1.2), joins that
// work the cuts out instead of reading them (+1 to +4 us), going through the join's code once over zeros while it waits (+0.3).
#include "b8_attn.cuh"

namespace ifv2 {
namespace {

using namespace b8;

constexpr int kThreads = 192, kSoftmax = 128;
constexpr float kMostSum = 100.f;                // log2 of the largest part of a sum after a move

template <int kT>
struct Shape {
  static constexpr int kN = kGroup * kT;           // columns
  static constexpr int kStages = kT == 1 ? 3 : 2;
  static constexpr int kQBytes = kN * kHeadDim;    // one of two terms
  static constexpr int kPBytes = kN * kUnit;       // one of three terms
  static constexpr int kQ = 0, kP = 2 * kQBytes, kRing = (kP + 3 * kPBytes + 1023) / 1024 * 1024;
  static constexpr int kSmem = kRing + kStages * 2 * kTileBytes + 1024;
  static constexpr int kO = 2 * kN;                // columns of O behind two S
  static constexpr int kTmem = kT == 1 ? 128 : 256;
};

// Column sums (or maxima) over the 32 lanes: half the columns go to the other lane in each step.  Column `first` is in v[0]
// at the end.
template <bool kMax, int kN>
__device__ __forceinline__ int reduce_columns(float (&v)[kN], int lane) {
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
        const float got = __shfl_xor_sync(0xFFFFFFFFu, other, s);
        v[i] = kMax ? fmaxf(mine, got) : mine + got;
      }
      if (up) first += n;
    } else {
      const float got = __shfl_xor_sync(0xFFFFFFFFu, v[0], s);
      v[0] = kMax ? fmaxf(v[0], got) : v[0] + got;
    }
  }
  return first;
}

template <int kT, int kCode, bool kSelected>
__global__ void __launch_bounds__(kThreads, 2)
b8_few_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const AttnParams p) {
  using S = Shape<kT>;
  constexpr int kN = S::kN, kStages = S::kStages;
  // an E for every token where tokens select blocks: one's values may be far from those of a block that another selects
  constexpr int kE = kSelected ? kT : 1;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ Common<kT, kStages> s;
  __shared__ uint64_t bar_s[2], bar_sfree[2], bar_p, bar_pv, bar_q, bar_drain;
  __shared__ __align__(16) float s_c[kN], s_mu[kN], s_fl[kN], s_fo[kN], s_red[4][kN], s_most[4][kE];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  __shared__ int s_cost[kThreads / 32];
  volatile int* gave_up = &s.gave_up;

  if (tid == 64) {
    s.gave_up = 0;
    for (int i = 0; i < kStages; ++i) mbar_init(&s.full[i], 2), mbar_init(&s.empty[i], 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar_s[i], 1), mbar_init(&bar_sfree[i], 4);
      mbar_init(&s.item_full[i], 1), mbar_init(&s.item_empty[i], 5);
    }
    mbar_init(&bar_p, 4);
    mbar_init(&bar_pv, 1);
    mbar_init(&bar_q, 4);
    mbar_init(&bar_drain, 1);
    fence_barrier_init();
    prefetch_tensormap(&k_map);
    prefetch_tensormap(&v_map);
  }
  if (warp == 1) {
    tmem_alloc(&s.tmem, S::kTmem);
    tmem_relinquish();
  }
  wait_inputs();
  Deal<kT, false, kSelected> deal;
  deal.add_up(p, s_cost);
  __syncthreads();
  if (warp == 0) deal.work_out(p, s_cost);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  allow_next();
  const uint32_t tmem_s = s.tmem, tmem_o = s.tmem + S::kO;

  if (warp == 0) {
    fetch<kT, kStages, false, kSelected>(p, &k_map, &v_map, s, smem + S::kRing, deal);
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMAs
    if (elect_one()) {
      const uint32_t base = smem_u32(smem);
      constexpr uint32_t kIdescS = umma_idesc_f8(128, kN, kCode, kE4m3, false, false);
      constexpr uint32_t kIdescO = umma_idesc_f8(128, 3 * kN, kCode, kE5m2, true, true);
      bool ok = true;
      int n = 0, queries = 0;
      const auto values = [&](int unit, bool first) {        // O += W V of a unit
        const int stage = unit % kStages;
        ok = ok && bounded_wait(&bar_p, unit & 1, gave_up);
        if (!ok) return;
        tc_fence_after();
        const uint32_t v = base + S::kRing + stage * 2 * kTileBytes + kTileBytes;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          umma_f8_ss(tmem_o, umma_desc_sw128(v + kk * 4096, 16, 1024), umma_desc_noswz_mn8(base + S::kP + kk * 512, 16 * kUnit),
                     kIdescO, !first || kk > 0);
        umma_commit(&s.empty[stage]);
        umma_commit(&bar_pv);
      };
      for (int item = 0; ok; ++item) {
        ok = bounded_wait(&s.item_full[item & 1], (item >> 1) & 1, gave_up);
        const int units = ok ? s.item[item & 1].units : -1;
        if (units < 0) break;
        mbar_arrive(&s.item_empty[item & 1]);
        if (units == 0) continue;
        ok = bounded_wait(&bar_q, queries++ & 1, gave_up);
        for (int i = 0; ok && i < units; ++i, ++n) {
          const int stage = n % kStages;
          ok = bounded_wait(&s.full[stage], (n / kStages) & 1, gave_up) && bounded_wait(&bar_sfree[n & 1], ((n >> 1) & 1) ^ 1, gave_up);
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
          if (i > 0) values(n - 1, i == 1);
        }
        values(n - 1, units == 1);
      }
      if (!ok) {
        umma_commit(&bar_drain);
        mbar_wait_drain(&bar_drain, 0);
      }
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- softmax
    // A wait that gave up makes the tile's results NaN, the CTA's tiles behind it are not written, and the status block says so.
    // Within an item every thread keeps to the same loops and barriers.
    const int quad = warp & 3, r = quad * 32 + lane;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const int stid = tid - 64;
    const int heads = p.heads_k * kGroup;

    // Query rows of an item: 8 threads per row, 16 values each.
    const auto write_query = [&](const Item& t) {
#pragma unroll
      for (int i = 0; i < kT; ++i) {
        const int col = i * 16 + (stid >> 3), c = stid & 7;
        uint4 x[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
        if (i < t.tokens) {
          const uint4* src = reinterpret_cast<const uint4*>(p.q + ((int64_t)(t.row + i) * heads + t.head * kGroup + (stid >> 3)) * kHeadDim + c * 16);
          x[0] = *src;
          x[1] = *(src + 1);
        }
        const float f = write_query16(x, smem + S::kQ + col * kHeadDim + ((c ^ (col & 7)) << 4), S::kQBytes, p.scale_log2);
        if (c == 0) s_c[col] = f;
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

    int n = 0;
    next_item(0);
    if (next.units > 0) write_query(next);
    for (int item = 0; next.units >= 0; ++item) {
      const Item t = next;
      // sums in registers; the columns' factors and references are read four at a time where they are used (in registers they
      // took two for every column, and what did not fit was spilled)
      float l[kN];
      named_sync<kSoftmax>();                      // s_c is written, the last item's s_fl and s_red are read
#pragma unroll
      for (int i = 0; i < kN; ++i) l[i] = 0.f;
      if (stid < kN) s_mu[stid] = kUnset;
      int e_ref[kE];                               // E
#pragma unroll
      for (int e = 0; e < kE; ++e) e_ref[e] = kNoScale;
#pragma unroll 1
      for (int i = 0; i < t.units; ++i, ++n) {
        const int stage = n % kStages;
        bounded_wait_warp(&s.full[stage], (n / kStages) & 1, gave_up);
        const Block* blk = &s.block[stage][r >> 6];
        const float k_scale = blk->k_scale;
        const int e_v = blk->e_v, valid = blk->valid & 0xFF;
        // E of this unit: none is chosen before a block has one (NaN values are taken to be at E, whatever it becomes)
        int e_new[kE];
#pragma unroll
        for (int e = 0; e < kE; ++e) {
          const int e_most = kE == kT ? blk->e_unit[e] : max(blk->e_unit[0], blk->e_unit[1]);
          e_new[e] = e_ref[e] != kNoScale && e_most - e_ref[e] <= kHighest ? e_ref[e] : e_most;
        }
        // which columns' tokens see the thread's key: the last token those below `valid`, the ones before it fewer if causal
        const int left = valid - (r & 63);         // > 0: a key
        uint32_t sees = left > 0 ? (1u << kT) - 1 : 0u;
        if (kT > 1 && left > 0) {
          const int in_reach = t.reach - (blk->pos + (r & 63));
          sees = kSelected ? blk->tokens : sees;
#pragma unroll
          for (int tok = 0; tok < kT; ++tok)
            if (p.causal && in_reach <= t.tokens - 1 - tok) sees &= ~(1u << tok);
        }
        const bool all = __all_sync(0xFFFFFFFFu, sees == (1u << kT) - 1);
        // eV - E; a NaN block's weights are NaN, those of a block far below the others' nothing
        int dv[kE];
        float v_ref[kE], v_scale[kE];
#pragma unroll
        for (int e = 0; e < kE; ++e) {
          // (a token that does not select the block has weights of 0, for which its exponent may be any)
          const bool any = e_v == kNanScale || (kE > 1 && !((blk->tokens >> e) & 1));
          dv[e] = any ? 0 : e_v - e_new[e];
          v_ref[e] = pow2i(max(dv[e], kDeepest));
          v_scale[e] = e_v == kNanScale ? NAN : dv[e] < kDeepest ? 0.f : v_ref[e];
        }
        bounded_wait_warp(&bar_s[n & 1], (n >> 1) & 1, gave_up);
        tc_fence_after();
        float w[kN];
        bool moves = false, settled = false;
        for (;;) {
          uint32_t x[kN];
          if constexpr (kN == 16) {
            tmem_ld16(tmem_s + (n & 1) * kN + lanes, x);
            tmem_wait_ld();
          } else {
            tmem_ld32_wait(tmem_s + (n & 1) * kN + lanes, x);
          }
          // (the two factors first: one may be 2^120 where the other is 2^-120)
          const uint64_t scale2 = pack_f32x2(k_scale, k_scale);
          if (moves && !settled) {
            // new references: the largest x + eV of each column, and E
#pragma unroll
            for (int j = 0; j < kN; ++j) {
              w[j] = fmaf(__uint_as_float(x[j]), q8::mul_exact(k_scale, s_c[j]), (float)max(dv[kE > 1 ? j / kGroup : 0], kDeepest));
              if (!((sees >> (j / kGroup)) & 1) || !(w[j] == w[j])) w[j] = -INFINITY;
            }
            const int first = reduce_columns<true, kN>(w, lane);
            s_red[quad][first] = w[0];             // (16 columns: two lanes, one value)
            // the largest part of the sums so far (of one number for all columns of an E: a number for each costs every call 0.7 us)
#pragma unroll
            for (int e = 0; e < kE; ++e) {
              float most = 0.f;
#pragma unroll
              for (int j = 0; j < kN / kE; ++j) most = fmaxf(most, l[e * (kN / kE) + j]);
              asm("redux.sync.max.f32 %0, %0, 0xFFFFFFFF;" : "+f"(most));
              if (lane == 0) s_most[quad][e] = most;
            }
            named_sync<kSoftmax>();
            if (stid < kN) {
              int delta = e_ref[0] == kNoScale ? 0 : e_new[0] - e_ref[0];
              if (kE > 1 && stid >= kGroup) delta = e_ref[kE - 1] == kNoScale ? 0 : e_new[kE - 1] - e_ref[kE - 1];
              const float top = fmaxf(fmaxf(s_red[0][stid], s_red[1][stid]), fmaxf(s_red[2][stid], s_red[3][stid]));
              const float was = s_mu[stid];
              float now = was, fl = 0.f, fo = 0.f;
              if (was == kUnset) {
                if (top > -INFINITY) now = top - kTop;
              } else {
                now = was - (float)delta;          // (M stays; further up where the sum, of blocks far below E, would leave fp32's range)
                if (top - now > kRoom) now = top - kTop;
                const int e = kE > 1 ? stid / kGroup : 0;
                const float most_l = fmaxf(fmaxf(s_most[0][e], s_most[1][e]), fmaxf(s_most[2][e], s_most[3][e]));
                if (delta > 0 && most_l > 0.f) now = fmaxf(now, was + lg2(most_l) - kMostSum);
                fl = ex2(0.5f * (was - now));      // (twice: l may hold 2^100 of blocks far below E, and their part in it counts)
                fo = ex2(was - now - (float)delta);
              }
              s_mu[stid] = now;
              s_fl[stid] = fl;
              s_fo[stid] = fo;
            }
            named_sync<kSoftmax>();
#pragma unroll
            for (int j = 0; j < kN; ++j) l[j] = l[j] > 0.f ? l[j] * s_fl[j] * s_fl[j] : l[j];
            if (i > 0) {                           // what is in O so far
              bounded_wait_warp(&bar_pv, (n - 1) & 1, gave_up);
              tc_fence_after();
#pragma unroll 1
              for (int c0 = 0; c0 < 3 * kN; c0 += 16) {
                uint32_t o[16];
                tmem_ld16(tmem_o + lanes + c0, o);
                tmem_wait_ld();
#pragma unroll
                for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * s_fo[(kT == 1 ? 0 : c0 & 16) + j]);
                tmem_st16(tmem_o + lanes + c0, o);
              }
              tmem_wait_st();
            }
            settled = true;
            continue;                              // (the scores are fetched again: 16 kT registers less until here)
          }
#pragma unroll
          for (int j = 0; j < kN; j += 4) {
            const float4 c = *reinterpret_cast<const float4*>(s_c + j), mu = *reinterpret_cast<const float4*>(s_mu + j);
            float y[4];
            unpack_f32x2(fma_f32x2(pack_f32x2(x[j], x[j + 1]), q8::mul_exact2(pack_f32x2(c.x, c.y), scale2), pack_f32x2(-mu.x, -mu.y)), y[0], y[1]);
            unpack_f32x2(fma_f32x2(pack_f32x2(x[j + 2], x[j + 3]), q8::mul_exact2(pack_f32x2(c.z, c.w), scale2), pack_f32x2(-mu.z, -mu.w)), y[2], y[3]);
#pragma unroll
            for (int e = 0; e < 4; ++e) w[j + e] = ex2(y[e]);
          }
          if (!all) {
#pragma unroll
            for (int j = 0; j < kN; ++j)
              if (!((sees >> (j / kGroup)) & 1)) w[j] = 0.f;
          }
          if (settled) break;
          bool far = false;
#pragma unroll
          for (int e = 0; e < kE; ++e) {
            constexpr int kOf = kN / kE;           // columns of an E
            float most = w[e * kOf];
#pragma unroll
            for (int j = 1; j < kOf; j += 2) most = fmaxf(fmaxf(most, w[e * kOf + j]), w[e * kOf + (j + 1 < kOf ? j + 1 : j)]);
            far |= e_new[e] != e_ref[e] || most * v_ref[e] > 32768.f;
          }
          // (one vote decides for all warps, whatever each has read: a wait that gave up must not part them)
          moves = named_any<kSoftmax>(far);
          if (!moves) break;
        }
        tc_fence_before();
        mbar_arrive_warp(&bar_sfree[n & 1]);
#pragma unroll
        for (int e = 0; e < kE; ++e) e_ref[e] = e_new[e];
        // the one buffer of weights is free again when the product before has been made
        if (n > 0) bounded_wait_warp(&bar_pv, (n - 1) & 1, gave_up);
#pragma unroll
        for (int j = 0; j < kN; ++j) l[j] += w[j];
        if (!all && !(v_scale[0] == v_scale[0])) {       // (only the columns that see the key are NaN)
#pragma unroll
          for (int j = 0; j < kN; ++j)
            if ((sees >> (j / kGroup)) & 1) w[j] = NAN;
        } else {
#pragma unroll
          for (int j = 0; j < kN; ++j) w[j] *= v_scale[kE > 1 ? j / kGroup : 0];
        }
#pragma unroll
        for (int tok = 0; tok < kT; ++tok) {
          uint32_t out[3][4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            split4(w[tok * 16 + 4 * j], w[tok * 16 + 4 * j + 1], w[tok * 16 + 4 * j + 2], w[tok * 16 + 4 * j + 3], out[0][j], out[1][j], out[2][j]);
#pragma unroll
          for (int k = 0; k < 3; ++k)
            *reinterpret_cast<uint4*>(smem + S::kP + k * S::kPBytes + tok * 16 * kUnit + r * 16) =
                make_uint4(out[k][0], out[k][1], out[k][2], out[k][3]);
        }
        // a value row that is no key, or of a page that is not there (another one is read in its place), may hold anything: 0 x NaN
        if (left <= 0 || s.block[stage][r >> 6].e_v == kNanScale) {
          uint4* row = reinterpret_cast<uint4*>(smem + S::kRing + stage * 2 * kTileBytes + kTileBytes + r * kHeadDim);
#pragma unroll
          for (int j = 0; j < 8; ++j) row[j] = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        tc_fence_before();
        mbar_arrive_warp(&bar_p);
      }
      // the next item's query, while the last product runs (every S of this item has been read)
      next_item(item + 1);
      if (next.units > 0) write_query(next);

      // ---- the item's results
      const int first = reduce_columns<false, kN>(l, lane);
      s_red[quad][first] = l[0];                   // (16 columns: two lanes, one value)
      named_sync<kSoftmax>();
      if (stid < kN) {
        const float sum = s_red[0][stid] + s_red[1][stid] + s_red[2][stid] + s_red[3][stid];
        const bool none = sum == 0.f;
        const float lse2 = *gave_up ? NAN : none ? -INFINITY : s_mu[stid] + lg2(sum);
        s_fl[stid] = none ? 0.f : rcp(sum);
        const int tok = stid / kGroup;
        if (t.piece >= 0) p.part_lse[(int64_t)t.piece * kN + stid] = lse2;
        else if (p.lse && tok < t.tokens)
          p.lse[(int64_t)(t.row + tok) * heads + t.head * kGroup + stid % kGroup] = lse2 == -INFINITY ? INFINITY : lse2 * kLn2;
      }
      if (t.units > 0) bounded_wait_warp(&bar_pv, (n - 1) & 1, gave_up);
      tc_fence_after();
      named_sync<kSoftmax>();
      const bool lost = *gave_up;
#pragma unroll
      for (int tok = 0; tok < kT; ++tok) {
        if (tok >= t.tokens) continue;
        // 2^E; a block's smallest exponent is -127
        const int e = e_ref[kE > 1 ? tok : 0];
        const float e_scale = lost ? NAN : e == -127 ? __uint_as_float(1u << 22) : pow2i(e > kNoScale ? e : 0);
        uint32_t o[3][16];
        if (t.units > 0) {
#pragma unroll
          for (int k = 0; k < 3; ++k) tmem_ld16(tmem_o + lanes + k * kN + tok * kGroup, o[k]);
          tmem_wait_ld();
        }
        float y[16];
#pragma unroll
        for (int c0 = 0; c0 < 16; c0 += 4) {
          const float4 f4 = *reinterpret_cast<const float4*>(s_fl + tok * kGroup + c0);
          const float f[4] = {f4.x, f4.y, f4.z, f4.w};
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int i = c0 + c;
            y[i] = q8::mul_exact((__uint_as_float(o[0][i]) + __uint_as_float(o[1][i]) + __uint_as_float(o[2][i])) * f[c], e_scale);
            if (f[c] == 0.f && !lost) y[i] = 0.f;  // (no key: O may be anything)
          }
        }
        if (t.piece < 0) {
          __nv_bfloat16* out = p.out + ((int64_t)(t.row + tok) * heads + t.head * kGroup) * kHeadDim + r;
#pragma unroll
          for (int c = 0; c < 16; ++c) out[c * kHeadDim] = __float2bfloat16(y[c]);
        } else {
          float* part = p.part_o + ((int64_t)t.piece * kN + tok * kGroup) * kHeadDim + r;
#pragma unroll
          for (int c = 0; c < 16; ++c) part[c * kHeadDim] = y[c];
        }
      }
      tc_fence_before();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && s.gave_up) atomicCAS(p.status + 1, 0, 101);
  if (warp == 1) tmem_dealloc(s.tmem, S::kTmem);
}

template <int kT, int kCode, bool kSelected>
int launch(const CUtensorMap& k_map, const CUtensorMap& v_map, const AttnParams& p, cudaStream_t stream) {
  constexpr int smem = Shape<kT>::kSmem;
  static std::atomic<uint64_t> allowed{0};
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(b8_few_kernel<kT, kCode, kSelected>), smem, allowed);
  if (e == cudaSuccess) e = launch_beside(b8_few_kernel<kT, kCode, kSelected>, dim3(kB8FewGrid), kThreads, smem, stream, k_map, v_map, p);
  if (e != cudaSuccess) return set_error((int)e, "b8_attn: %s", cudaGetErrorString(e));
  return check_launch("b8_attn");
}

template <int kT, int kCode>
int launch_with(const CUtensorMap& k_map, const CUtensorMap& v_map, const AttnParams& p, cudaStream_t stream) {
  return p.mask != nullptr || p.lists != nullptr ? launch<kT, kCode, true>(k_map, v_map, p, stream)
                                                 : launch<kT, kCode, false>(k_map, v_map, p, stream);
}

}  // namespace

int b8_launch_few(const CUtensorMap& k_map, const CUtensorMap& v_map, const AttnParams& p, int tokens, int code, cudaStream_t stream) {
  if (tokens == 1) return code == kE4m3 ? launch_with<1, kE4m3>(k_map, v_map, p, stream) : launch_with<1, kE5m2>(k_map, v_map, p, stream);
  return code == kE4m3 ? launch_with<2, kE4m3>(k_map, v_map, p, stream) : launch_with<2, kE5m2>(k_map, v_map, p, stream);
}

}  // namespace ifv2
