// Attention of new tokens over a cache in 8 bits with block scales (b8.cuh).
#include "b8.cuh"

namespace ifv2 {
namespace {

using namespace b8;

constexpr int kThreads = 128;

struct B8AttnParams {
  const __nv_bfloat16* q;
  const uint8_t *k_cache, *v_cache, *k_scale, *v_scale;
  __nv_bfloat16* out;
  float* lse;
  const int32_t *cu_q, *seqlens, *block_table;
  const unsigned long long* mask;
  int bt_stride, words, batch, heads_k, length, causal;
  int64_t total_q, pages;
  float scale;
};

template <int kCode>
__global__ void __launch_bounds__(kThreads) b8_attn_simple_kernel(const B8AttnParams p) {
  __shared__ float s_q[kGroup][kHeadDim], s_p[kGroup][kThreads];
  __shared__ float s_m[kGroup], s_l[kGroup], s_f[kGroup];
  const int64_t t = blockIdx.x;
  const int h = blockIdx.y, tid = threadIdx.x;
  const int heads = p.heads_k * kGroup;
  __nv_bfloat16* out = p.out + (t * heads + h * kGroup) * kHeadDim;
  int keys = 0, b = 0;
  if (t < p.cu_q[p.batch]) {
    b = find_sequence(p.cu_q, p.batch, (int)t);
    const int64_t cap = p.block_table ? (int64_t)p.bt_stride * p.length : p.length;
    const int len = (int)min((int64_t)max(p.seqlens[b], 0), cap);
    keys = p.causal ? len - (p.cu_q[b + 1] - (int)t) + 1 : len;
  }
  for (int g = 0; g < kGroup; ++g) s_q[g][tid] = __bfloat162float(p.q[(t * heads + h * kGroup + g) * kHeadDim + tid]) * p.scale;
  if (tid < kGroup) s_m[tid] = -INFINITY, s_l[tid] = 0.f;
  float acc[kGroup];
  for (int g = 0; g < kGroup; ++g) acc[g] = 0.f;
  __syncthreads();
  const unsigned long long* mask = p.mask ? p.mask + ((int64_t)h * p.total_q + t) * p.words : nullptr;
  for (int k0 = 0; k0 < keys; k0 += kBlockN) {
    const int blk = k0 / kBlockN;
    if (mask && !((mask[blk >> 6] >> (blk & 63)) & 1)) continue;
    const int64_t page = p.block_table ? p.block_table[(int64_t)b * p.bt_stride + k0 / p.length] : b;
    const bool bad = page < 0 || page >= p.pages;
    const int place = p.block_table ? k0 % p.length : k0;
    const int64_t row = bad ? 0 : (page * p.heads_k + h) * (int64_t)p.length + place;
    const float ks = bad ? NAN : q8::scale_value(p.k_scale[row / kBlockN]), vs = bad ? NAN : q8::scale_value(p.v_scale[row / kBlockN]);
    const int n = min(kBlockN, keys - k0);
    if (tid < kBlockN) {
      float x[kGroup];
      for (int g = 0; g < kGroup; ++g) x[g] = 0.f;
      if (tid < n) {
        const uint32_t* code = reinterpret_cast<const uint32_t*>(p.k_cache + (row + tid) * kHeadDim);
        for (int c = 0; c < kHeadDim / 4; ++c) {
          float y[4];
          decode4<kCode>(y, code[c]);
          for (int g = 0; g < kGroup; ++g)
            for (int j = 0; j < 4; ++j) x[g] += s_q[g][4 * c + j] * (y[j] * ks);
        }
      }
      for (int g = 0; g < kGroup; ++g) s_p[g][tid] = tid < n ? x[g] : -INFINITY;
    }
    __syncthreads();
    if (tid < kGroup) {
      float m = s_m[tid];
      for (int j = 0; j < n; ++j) m = fmaxf(m, s_p[tid][j]);
      const float f = __expf(s_m[tid] - m);
      float l = s_l[tid] * f;
      for (int j = 0; j < n; ++j) {
        const float e = __expf(s_p[tid][j] - m);
        s_p[tid][j] = e;
        l += e;
      }
      s_m[tid] = m, s_l[tid] = l, s_f[tid] = f;
    }
    __syncthreads();
    for (int g = 0; g < kGroup; ++g) acc[g] *= s_f[g];
    for (int j = 0; j < n; ++j) {
      const uint8_t c = p.v_cache[(row + j) * kHeadDim + tid];
      const float y = __half2float(__half(__nv_cvt_fp8_to_halfraw(c, kCode == kE4m3 ? __NV_E4M3 : __NV_E5M2))) * vs;
      for (int g = 0; g < kGroup; ++g) acc[g] += s_p[g][j] * y;
    }
    __syncthreads();
  }
  for (int g = 0; g < kGroup; ++g) {
    const bool none = s_l[g] == 0.f;
    out[g * kHeadDim + tid] = __float2bfloat16(none ? 0.f : acc[g] / s_l[g]);
    if (p.lse && tid == 0) p.lse[t * heads + h * kGroup + g] = none ? INFINITY : s_m[g] + logf(s_l[g]);
  }
}

}  // namespace
}  // namespace ifv2

using namespace ifv2;

extern "C" int64_t ifv2_b8_attn_workspace_bytes(int64_t total_q, int batch, int heads_q, int head_dim, int max_seqlen_q) {
  return 16;
}

extern "C" int ifv2_b8_attn(const void* q, const void* k_cache, const void* v_cache, const void* k_scale, const void* v_scale,
                            void* out, float* lse, const int32_t* cu_seqlens_q, const int32_t* cache_seqlens,
                            const int32_t* block_table, int block_table_stride, const int64_t* mask, int mask_words, int batch,
                            int64_t total_q, int max_seqlen_q, int64_t num_pages, int64_t length, int code, int heads_q, int heads_k,
                            int head_dim, float softmax_scale, int causal, void* workspace, int64_t workspace_bytes, void* stream) {
  IFV2_REQUIRE(head_dim == kHeadDim && heads_q == heads_k * kGroup, IFV2_ERR_UNSUPPORTED,
               "b8_attn: head_dim must be %d, with %d query heads per KV head", kHeadDim, kGroup);
  if (total_q == 0) return IFV2_OK;
  B8AttnParams p{static_cast<const __nv_bfloat16*>(q), static_cast<const uint8_t*>(k_cache), static_cast<const uint8_t*>(v_cache),
                 static_cast<const uint8_t*>(k_scale), static_cast<const uint8_t*>(v_scale), static_cast<__nv_bfloat16*>(out), lse,
                 cu_seqlens_q, cache_seqlens, block_table, reinterpret_cast<const unsigned long long*>(mask), block_table_stride,
                 mask_words, batch, heads_k, (int)length, causal, total_q, num_pages, softmax_scale};
  const dim3 grid((unsigned)total_q, heads_k);
  if (code == kE4m3) b8_attn_simple_kernel<kE4m3><<<grid, kThreads, 0, (cudaStream_t)stream>>>(p);
  else b8_attn_simple_kernel<kE5m2><<<grid, kThreads, 0, (cudaStream_t)stream>>>(p);
  return check_launch("b8_attn");
}
