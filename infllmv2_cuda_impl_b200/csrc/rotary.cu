// Rotary positions over several axes (time, height, width of images and video) for packed queries and keys,
// forward and backward (formulas: rotary.cuh).  The gradient of a rotation is the rotation by minus the angle.
//
// Bound by HBM: every row is read and written once (512 B); a token's angles are read once for all of its rows.
#include "rotary.cuh"

namespace ifv2 {

int make_rotary(RotaryParams* r, const char* what, const float* cos_t, const float* sin_t, const int32_t* positions,
                int64_t axis_stride, const uint8_t* pair_axis, int axes, int dim, int64_t rows, int interleaved) {
  IFV2_REQUIRE(dim >= 16 && dim <= kHeadDim && dim % 16 == 0, IFV2_ERR_INVALID_ARG,
               "%s: rotary_dim must be a positive multiple of 16 and <= head_dim", what);
  IFV2_REQUIRE(axes >= 1 && axes <= kMaxAxes, IFV2_ERR_INVALID_ARG, "%s: 1 to %d axes", what, kMaxAxes);
  IFV2_REQUIRE(rows >= 1 && rows <= INT32_MAX, IFV2_ERR_INVALID_ARG, "%s: the tables hold no position, or too many", what);
  IFV2_REQUIRE(cos_t && sin_t && positions, IFV2_ERR_INVALID_ARG, "%s: null pointer", what);
  IFV2_REQUIRE((reinterpret_cast<uintptr_t>(cos_t) | reinterpret_cast<uintptr_t>(sin_t)) % 16 == 0, IFV2_ERR_INVALID_ARG,
               "%s: tables must be 16-byte aligned", what);
  *r = RotaryParams{cos_t, sin_t, positions, axis_stride, dim, (int)rows, interleaved ? 1 : 0, {0u, 0u, 0u, 0u}};
  for (int i = 0; pair_axis != nullptr && i < dim / 2; ++i) {
    IFV2_REQUIRE(pair_axis[i] < axes, IFV2_ERR_INVALID_ARG, "%s: pair %d names axis %d of %d", what, i, (int)pair_axis[i], axes);
    r->axis_map[i >> 4] |= (uint32_t)pair_axis[i] << (2 * (i & 15));
  }
  return IFV2_OK;
}

namespace {

constexpr int kThreads = 256;
constexpr int kLanes = 8;                       // threads of a row, 8 pairs (16 features) each
constexpr int kRows = 32 / kLanes;              // rows that a warp turns at once

struct RotaryKernelParams {
  RotaryParams r;
  const uint4* src[2];           // queries, keys
  uint4* dst[2];                 // (tokens, heads, 128), dense
  int64_t token_stride[2], head_stride[2];      // of src, in 16-byte vectors
  int heads[2];
  int64_t tokens;
  int chunks, chunk;             // a token's rows are shared by `chunks` warps, `chunk` rows each
  int back;
};

// A warp takes up to 36 rows of one token, four at a time.  Four CTAs per SM with one row per thread under way: two or
// three rows loaded ahead cost the registers of a CTA and were slower (32768 tokens of 34 heads: 98 us, 92 % of the copy
// bandwidth; 110 with two rows, 127 with three, 103 with five CTAs, whose registers spill, 108 with 18 rows per warp).
template <bool kInterleaved>
__global__ void __launch_bounds__(kThreads, 4) rotary_axes_kernel(const RotaryKernelParams p) {
  const int64_t w = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 5;
  const int64_t t = w / p.chunks;
  if (t >= p.tokens) return;
  const int first = (int)(w - t * p.chunks) * p.chunk, last = min(first + p.chunk, p.heads[0] + p.heads[1]);
  const int lane = threadIdx.x & 31, l = lane % kLanes;
  const bool turn = 8 * l < p.r.dim / 2;
  // vectors of the thread's 16 features: a neighbouring pair of vectors, or one in each half
  const int a = !turn || kInterleaved ? 2 * l : l, b = !turn || kInterleaved ? 2 * l + 1 : l + p.r.dim / 16;
  const uint4 *src_q = p.src[0] + t * p.token_stride[0], *src_k = p.src[1] + t * p.token_stride[1];
  uint4 *dst_q = p.dst[0] + t * p.heads[0] * (kHeadDim / 8), *dst_k = p.dst[1] + t * p.heads[1] * (kHeadDim / 8);
  auto load = [&](int row, uint4& va, uint4& vb) {
    const int h = row - p.heads[0];
    const uint4* s = h < 0 ? src_q + row * p.head_stride[0] : src_k + h * p.head_stride[1];
    va = __ldg(s + a);
    vb = __ldg(s + b);
  };
  // the first row's loads and the angles, which wait for the positions, travel together
  int row = first + lane / kLanes;
  uint4 va, vb;
  if (row < last) load(row, va, vb);
  float c[8], s[8];
  if (turn) {
    const uint32_t axes = (p.r.axis_map[l >> 1] >> (16 * (l & 1))) & 0xFFFFu;
    if (axes == (axes & 3) * 0x5555u) {          // all eight pairs on one axis: they are neighbours in the tables
      const int64_t at = p.r.table_row(t, 8 * l) * (p.r.dim / 2) + 8 * l;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 fc = __ldg(reinterpret_cast<const float4*>(p.r.cos_t + at) + i);
        const float4 fs = __ldg(reinterpret_cast<const float4*>(p.r.sin_t + at) + i);
        c[4 * i] = fc.x; c[4 * i + 1] = fc.y; c[4 * i + 2] = fc.z; c[4 * i + 3] = fc.w;
        s[4 * i] = fs.x; s[4 * i + 1] = fs.y; s[4 * i + 2] = fs.z; s[4 * i + 3] = fs.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int64_t at = p.r.table_row(t, 8 * l + i) * (p.r.dim / 2) + 8 * l + i;
        c[i] = __ldg(p.r.cos_t + at);
        s[i] = __ldg(p.r.sin_t + at);
      }
    }
    if (p.back) {
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] = -s[i];
    }
  }
  while (row < last) {
    uint4* d = row < p.heads[0] ? dst_q + row * (kHeadDim / 8) : dst_k + (row - p.heads[0]) * (kHeadDim / 8);
    if (turn) {
      uint32_t x[8] = {va.x, va.y, va.z, va.w, vb.x, vb.y, vb.z, vb.w};
      float lo[8], hi[8];                        // first and second feature of pairs 0 .. 7
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float f0 = __uint_as_float(x[j] << 16), f1 = __uint_as_float(x[j] & 0xFFFF0000u);
        if (kInterleaved) {
          lo[j] = f0;
          hi[j] = f1;
        } else {                                 // words 0 .. 3: first features of pairs 2j, 2j + 1
          (j < 4 ? lo : hi)[2 * (j & 3)] = f0;
          (j < 4 ? lo : hi)[2 * (j & 3) + 1] = f1;
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) rotate2(lo[j], hi[j], c[j], s[j]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const __nv_bfloat162 v = kInterleaved ? __floats2bfloat162_rn(lo[j], hi[j])
                                 : j < 4      ? __floats2bfloat162_rn(lo[2 * (j & 3)], lo[2 * (j & 3) + 1])
                                              : __floats2bfloat162_rn(hi[2 * (j & 3)], hi[2 * (j & 3) + 1]);
        x[j] = *reinterpret_cast<const uint32_t*>(&v);
      }
      va = make_uint4(x[0], x[1], x[2], x[3]);
      vb = make_uint4(x[4], x[5], x[6], x[7]);
    }
    d[a] = va;
    d[b] = vb;
    row += kRows;
    if (row < last) load(row, va, vb);
  }
}

}  // namespace
}  // namespace ifv2

using namespace ifv2;

extern "C" int ifv2_rotary_axes(const void* q, const void* k, void* q_out, void* k_out, const float* rotary_cos,
                                const float* rotary_sin, const int32_t* positions, int64_t axis_stride,
                                const uint8_t* pair_axis, int axes, int64_t tokens, int heads_q, int heads_k, int head_dim,
                                int64_t q_token_stride, int64_t q_head_stride, int64_t k_token_stride,
                                int64_t k_head_stride, int rotary_dim, int64_t table_rows, int interleaved, int backward,
                                void* stream) {
  IFV2_REQUIRE(head_dim == kHeadDim, IFV2_ERR_UNSUPPORTED, "rotary_axes: head_dim %d not supported (only 128)", head_dim);
  IFV2_REQUIRE(tokens >= 0 && heads_q >= 0 && heads_k >= 0 && heads_q <= 65535 && heads_k <= 65535, IFV2_ERR_INVALID_ARG,
               "rotary_axes: bad size");
  RotaryKernelParams p{};
  if (tokens == 0 || heads_q + heads_k == 0) return IFV2_OK;
  int rc = make_rotary(&p.r, "rotary_axes", rotary_cos, rotary_sin, positions, axis_stride, pair_axis, axes, rotary_dim,
                       table_rows, interleaved);
  if (rc) return rc;
  IFV2_REQUIRE((heads_q == 0 || (q && q_out)) && (heads_k == 0 || (k && k_out)), IFV2_ERR_INVALID_ARG, "rotary_axes: null pointer");
  for (const void* ptr : {q, k, (const void*)q_out, (const void*)k_out})
    IFV2_REQUIRE(reinterpret_cast<uintptr_t>(ptr) % 16 == 0, IFV2_ERR_INVALID_ARG, "rotary_axes: tensors must be 16-byte aligned");
  IFV2_REQUIRE((q_token_stride | q_head_stride | k_token_stride | k_head_stride) % 8 == 0, IFV2_ERR_INVALID_ARG,
               "rotary_axes: rows must be 16-byte aligned");
  p.src[0] = static_cast<const uint4*>(q);
  p.src[1] = static_cast<const uint4*>(k);
  p.dst[0] = static_cast<uint4*>(q_out);
  p.dst[1] = static_cast<uint4*>(k_out);
  p.token_stride[0] = q_token_stride / 8;
  p.token_stride[1] = k_token_stride / 8;
  p.head_stride[0] = q_head_stride / 8;
  p.head_stride[1] = k_head_stride / 8;
  p.heads[0] = heads_q;
  p.heads[1] = heads_k;
  p.tokens = tokens;
  // rows per warp: many where there are many tokens, so that a token's angles are fetched by few warps; few where there
  // are few, so that all SMs have work (64 tokens of 34 heads in a graph: 2.3 us with 4 rows, 2.7 with 12)
  const int rows = heads_q + heads_k;
  p.chunks = ceil_div(rows, tokens >= kNumSMs * 16 ? 36 : tokens >= kNumSMs ? 12 : 4);
  p.chunk = ceil_div(rows, p.chunks);
  p.back = backward ? 1 : 0;
  const int64_t blocks = ceil_div64(tokens * p.chunks, kThreads / 32);
  IFV2_REQUIRE(blocks <= INT32_MAX, IFV2_ERR_TOO_LARGE, "rotary_axes: too many tokens x heads");
  if (interleaved) rotary_axes_kernel<true><<<(unsigned)blocks, kThreads, 0, (cudaStream_t)stream>>>(p);
  else rotary_axes_kernel<false><<<(unsigned)blocks, kThreads, 0, (cudaStream_t)stream>>>(p);
  return check_launch("rotary_axes");
}
