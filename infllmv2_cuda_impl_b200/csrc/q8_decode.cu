// One new token per sequence over a key-value cache in 8 bits (formulas of the codes: q8.cuh).
//
//   s_t = scale * q . K_t * 2^eK(t),  m = max s,  l = sum exp(s_t - m),  out = sum exp(s_t - m) 2^eV(t) V_t / l
//
// over the positions of the sequence, or those of the 64-key blocks that its mask row selects.  The keys are shared
// by 16 query heads, split over CTAs, and the partial (m, l, M, O) of the splits are joined by a second kernel.
//
// O is a sum over codes, O = sum 2^(z_t - M) V_t with z_t = log2(e) s_t + eV(t) and M = max z: the exponents of the
// values take part in the weights, next to the scores, so no weight is above 1, the largest is 1 whatever the values'
// sizes are, and out = O 2^(M - m) / l.  (m and M differ by at most 127, the range of the exponents.)
//
// Launches: [prepare: block lists, append] -> split -> combine.
#include "rotary.cuh"
#include "q8.cuh"

namespace ifv2 {
namespace {

using namespace q8;

constexpr int kThreads = 128;
constexpr int kUnit = 32;                        // keys handled at once
constexpr int kMaxSplits = 16;
constexpr int kPartialFloats = kHeadDim + 4;     // O row, m (log2 units), l, M, pad
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct Q8DecodeParams {
  const __nv_bfloat16* q;          // (batch, heads_q, 128)
  const uint8_t* k_codes;
  const uint8_t* v_codes;
  const uint8_t* k_scale;
  const uint8_t* v_scale;
  const unsigned long long* mask;  // (batch, heads_k, mask_words) or null = all positions
  int mask_words;
  const int32_t* cache_seqlens;
  Place place;
  int64_t capacity;
  int batch, heads_k, new_tokens, splits, rotate;
  RotaryParams rotary;
  float scale_log2;
  float* partial;                  // (batch, heads_k, splits, 16, kPartialFloats)
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

// Four consecutive features (4 lane ..) of row `src`, rotated for token t.
__device__ __forceinline__ void load_rotated(float (&x)[4], const __nv_bfloat16* src, const RotaryParams& r, bool rotate,
                                             int64_t t, int lane) {
  auto at = [&](int i) { return __bfloat162float(ldg16(src + i)); };
  const int half = r.dim / 2;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int f = 4 * lane + i;
    x[i] = at(f);
    if (!rotate || f >= r.dim) continue;
    const int pair = r.interleaved ? f / 2 : f % half;
    const bool second = r.interleaved ? f & 1 : f >= half;
    const int other = r.interleaved ? f ^ 1 : second ? f - half : f + half;
    float x0 = second ? at(other) : x[i], x1 = second ? x[i] : at(other);
    const int64_t e = r.table_row(t, pair) * half + pair;
    rotate2(x0, x1, __ldg(r.cos_t + e), __ldg(r.sin_t + e));
    x[i] = second ? x1 : x0;
  }
}

// One CTA per (sequence, KV head): block lists -> mask row; the new key (rotated) and value -> their row.
template <int kCode>
__global__ void __launch_bounds__(kThreads) q8_prepare_kernel(const Q8PrepareParams a, const Q8DecodeParams p) {
  extern __shared__ unsigned long long row_words[];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
  const int64_t pair = (int64_t)b * p.heads_k + h;
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
      float x[4];
      load_rotated(x, (is_v ? a.v_new : a.k_new) + pair * kHeadDim, p.rotary, p.rotate && !is_v, b, lane);
      store_row<kCode>(x, (is_v ? a.v_codes : a.k_codes) + row * kHeadDim, (is_v ? a.v_scale : a.k_scale) + row, lane);
    }
  }
  if (a.topk_idx != nullptr) {
    __syncthreads();
    for (int w = tid; w < a.words; w += kThreads) a.mask[pair * a.words + w] = row_words[w];
  }
}

// One split of one (sequence, KV head): eight threads per query head.
template <int kCode>
__global__ void __launch_bounds__(kThreads) q8_split_kernel(const Q8DecodeParams p) {
  __shared__ float qs[kGroup][kHeadDim], ks[kUnit][kHeadDim + 1], vs[kUnit][kHeadDim], ps[kGroup][kUnit], ek[kUnit], ev[kUnit];
  const int split = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = tid / 8, c = tid % 8;
  const int64_t pair = (int64_t)b * p.heads_k + h;
  const int len = keys_of(p, b);
  const int n_blocks = (len + kBlockN - 1) / kBlockN;
  for (int i = warp; i < kGroup; i += kThreads / 32) {
    float x[4];
    load_rotated(x, p.q + (pair * kGroup + i) * kHeadDim, p.rotary, p.rotate, b, lane);
#pragma unroll
    for (int j = 0; j < 4; ++j) qs[i][4 * lane + j] = x[j];
  }
  float o[16], m = -INFINITY, mv = -INFINITY, l = 0.f;
#pragma unroll
  for (int j = 0; j < 16; ++j) o[j] = 0.f;
  for (int blk = split; blk < n_blocks; blk += p.splits) {
    if (p.mask != nullptr && (blk / 64 >= p.mask_words || !((p.mask[pair * p.mask_words + blk / 64] >> (blk & 63)) & 1ull)))
      continue;
    for (int key0 = blk * kBlockN; key0 < min(len, (blk + 1) * kBlockN); key0 += kUnit) {
      __syncthreads();
      for (int i = warp; i < kUnit; i += kThreads / 32) {
        const bool in = key0 + i < len;
        const int64_t row0 = in ? p.place.row0(b, key0 + i) : -1;
        float xk[4] = {0.f, 0.f, 0.f, 0.f}, xv[4] = {0.f, 0.f, 0.f, 0.f};
        int bk = in ? kNanByte : 0, bv = bk;     // (a page that the cache does not have: the result is NaN)
        if (row0 >= 0) {
          const int64_t row = p.place.row(row0, h);
          bk = p.k_scale[row];
          bv = p.v_scale[row];
          decode4<kCode>(xk, reinterpret_cast<const uint32_t*>(p.k_codes + row * kHeadDim)[lane]);
          decode4<kCode>(xv, reinterpret_cast<const uint32_t*>(p.v_codes + row * kHeadDim)[lane]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          ks[i][4 * lane + j] = xk[j];
          vs[i][4 * lane + j] = xv[j];
        }
        if (lane == 0) {
          ek[i] = scale_value(bk);
          ev[i] = bv == kNanByte ? scale_value(bv) : (float)(bv - 127);
        }
      }
      __syncthreads();
      float s[4], z[4], mx = m, mz = mv;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int t = c + 8 * u;
        float acc = 0.f;
        for (int j = 0; j < kHeadDim; ++j) acc = fmaf(qs[r][j], ks[t][j], acc);
        const bool in = key0 + t < len;
        s[u] = in ? mul_exact(acc, ek[t]) * p.scale_log2 : -INFINITY;
        z[u] = in ? s[u] + ev[t] : -INFINITY;
        mx = fmaxf(mx, s[u]);
        mz = fmaxf(mz, z[u]);
      }
#pragma unroll
      for (int d = 1; d < 8; d <<= 1) {
        mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, d));
        mz = fmaxf(mz, __shfl_xor_sync(0xFFFFFFFFu, mz, d));
      }
      const float f = mx == -INFINITY ? 1.f : exp2f(m - mx), sub = mx == -INFINITY ? 0.f : mx;
      const float fv = mz == -INFINITY ? 1.f : exp2f(mv - mz), subv = mz == -INFINITY ? 0.f : mz;
      m = mx;
      mv = mz;
      l *= f;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        l += exp2f(s[u] - sub);
        ps[r][c + 8 * u] = exp2f(z[u] - subv);
      }
      __syncwarp();
#pragma unroll
      for (int j = 0; j < 16; ++j) o[j] *= fv;
      for (int t = 0; t < kUnit; ++t) {
        const float e = ps[r][t];
#pragma unroll
        for (int j = 0; j < 16; ++j) o[j] = fmaf(e, vs[t][c + 8 * j], o[j]);
      }
    }
  }
#pragma unroll
  for (int d = 1; d < 8; d <<= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, d);
  float* dst = p.partial + ((pair * p.splits + split) * kGroup + r) * kPartialFloats;
#pragma unroll
  for (int j = 0; j < 16; ++j) dst[c + 8 * j] = o[j];
  if (c == 0) {
    dst[kHeadDim] = m;
    dst[kHeadDim + 1] = l;
    dst[kHeadDim + 2] = mv;
  }
}

// A partial sum in units of 2^m as one in units of 2^top.  Without a finite m it is 0, or NaN and stays so.
__device__ __forceinline__ float join(float m, float top, float x) { return m == -INFINITY ? x : x * exp2f(m - top); }

// x 2^d, |d| <= 127, in two steps so that neither factor leaves the normal numbers.
__device__ __forceinline__ float times_exp2(float x, float d) {
  const float f = exp2f(0.5f * d);
  return mul_exact(mul_exact(x, f), f);
}

// Joins the splits: one CTA per (sequence, KV head), one thread per feature.
__global__ void __launch_bounds__(kThreads) q8_combine_kernel(const Q8DecodeParams p) {
  const int h = blockIdx.x, b = blockIdx.y, d = threadIdx.x;
  const int64_t pair = (int64_t)b * p.heads_k + h;
  for (int r = 0; r < kGroup; ++r) {
    const float* src = p.partial + (pair * p.splits * kGroup + r) * kPartialFloats;
    float m = -INFINITY, mv = -INFINITY;
    for (int s = 0; s < p.splits; ++s) {
      m = fmaxf(m, src[(int64_t)s * kGroup * kPartialFloats + kHeadDim]);
      mv = fmaxf(mv, src[(int64_t)s * kGroup * kPartialFloats + kHeadDim + 2]);
    }
    float acc = 0.f, l = 0.f;
    for (int s = 0; s < p.splits; ++s) {
      const float* part = src + (int64_t)s * kGroup * kPartialFloats;
      l += join(part[kHeadDim], m, part[kHeadDim + 1]);
      acc += join(part[kHeadDim + 2], mv, part[d]);
    }
    const bool none = l == 0.f;
    const int64_t row = pair * kGroup + r;
    p.out[row * kHeadDim + d] = __float2bfloat16_rn(none ? 0.f : times_exp2(acc / l, mv - m));
    if (p.lse != nullptr && d == 0) p.lse[row] = none ? INFINITY : (m + log2f(l)) * kLn2;
  }
}

}  // namespace
}  // namespace ifv2

using namespace ifv2;

extern "C" int64_t ifv2_q8_decode_workspace_bytes(int batch, int heads_q, int head_dim) {
  if (batch < 0 || heads_q < 0 || head_dim != kHeadDim) return 0;
  return (int64_t)batch * heads_q * kMaxSplits * kPartialFloats * 4 + 256;
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
  IFV2_REQUIRE(topk_idx == nullptr || (mask != nullptr && topk >= 0), IFV2_ERR_INVALID_ARG, "q8_decode: block lists need a mask buffer");
  IFV2_REQUIRE(mask == nullptr || mask_words >= 1, IFV2_ERR_INVALID_ARG, "q8_decode: mask_words < 1");
  IFV2_REQUIRE(topk_idx == nullptr || mask_words <= 4096, IFV2_ERR_TOO_LARGE, "q8_decode: more than 4096 mask words");
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
  IFV2_REQUIRE(batch <= 65535 && heads_k <= 65535, IFV2_ERR_TOO_LARGE, "q8_decode: batch or heads_k > 65535");
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
  p.k_codes = static_cast<const uint8_t*>(k_cache);
  p.v_codes = static_cast<const uint8_t*>(v_cache);
  p.k_scale = static_cast<const uint8_t*>(k_scale);
  p.v_scale = static_cast<const uint8_t*>(v_scale);
  p.mask = reinterpret_cast<const unsigned long long*>(mask);
  p.mask_words = mask_words;
  p.cache_seqlens = cache_seqlens;
  p.place = Place{block_table, cache_batch_idx, block_table_stride, heads_k, (int)length, (int)slots};
  p.capacity = capacity;
  p.batch = batch;
  p.heads_k = heads_k;
  p.new_tokens = k_new != nullptr;
  p.scale_log2 = softmax_scale * kLog2e;
  p.partial = static_cast<float*>(workspace);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.lse = lse;
  p.splits = kMaxSplits;
  cudaStream_t st = (cudaStream_t)stream;
  if (k_new != nullptr || topk_idx != nullptr) {
    const Q8PrepareParams a{static_cast<const __nv_bfloat16*>(k_new), static_cast<const __nv_bfloat16*>(v_new),
                            static_cast<uint8_t*>(k_cache), static_cast<uint8_t*>(v_cache), static_cast<uint8_t*>(k_scale),
                            static_cast<uint8_t*>(v_scale), topk_idx, reinterpret_cast<unsigned long long*>(mask), topk, mask_words};
    const size_t smem = topk_idx ? (size_t)mask_words * 8 : 0;
    if (code == kE4m3) q8_prepare_kernel<kE4m3><<<dim3(heads_k, batch), kThreads, smem, st>>>(a, p);
    else q8_prepare_kernel<kInt8><<<dim3(heads_k, batch), kThreads, smem, st>>>(a, p);
    int rc = check_launch("q8_prepare");
    if (rc) return rc;
  }
  if (code == kE4m3) q8_split_kernel<kE4m3><<<dim3(p.splits, heads_k, batch), kThreads, 0, st>>>(p);
  else q8_split_kernel<kInt8><<<dim3(p.splits, heads_k, batch), kThreads, 0, st>>>(p);
  int rc = check_launch("q8_split");
  if (rc) return rc;
  q8_combine_kernel<<<dim3(heads_k, batch), kThreads, 0, st>>>(p);
  return check_launch("q8_combine");
}
