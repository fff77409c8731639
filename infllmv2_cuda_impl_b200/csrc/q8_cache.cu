// Writing packed keys and values into an 8-bit cache, and reading rows of it back (formulas: q8.cuh).
//
// Bound by HBM: 256 B of bf16 and 129 B of code and scale per row, each touched once.
#include "q8.cuh"

namespace ifv2 {
namespace {

using namespace q8;

constexpr int kThreads = 256;
constexpr int kLanes = 8;                       // threads of a row, 16 values each
constexpr int kTile = kThreads / kLanes;        // tokens of a CTA

struct MoveParams {
  const uint4* src[2];           // packed keys, values (read: null)
  int64_t token_stride[2], head_stride[2];      // of the packed tensors, in 16-byte vectors
  uint4* dst[2];                 // packed keys, values (write: null)
  uint8_t* codes[2];
  uint8_t* scales[2];
  const int32_t* cu;             // (batch + 1)
  const int32_t* start;          // (batch) position of each sequence's first token, or null = 0
  int32_t* seqlens_out;          // (batch) or null
  Place place;
  int batch;
  int64_t total, capacity;
};

// Row of head 0 for packed token t; -1: nowhere, -2: not a token of any sequence.
__device__ __forceinline__ int64_t token_row(const MoveParams& p, int64_t t) {
  if (t >= p.total || t >= p.cu[p.batch]) return -2;
  const int b = find_sequence(p.cu, p.batch, (int)t);
  const int64_t at = t - p.cu[b];
  return at < 0 ? -2 : p.place.row0(b, at + (p.start ? p.start[b] : 0));
}

__device__ __forceinline__ void to_float(float (&x)[16], const uint4& a, const uint4& b) {
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}

// A CTA writes one head of kTile tokens, keys and values: eight threads per row, whose vectors l and l + 8 leave
// as two 8-byte stores.  Bound by HBM: 131072 tokens of 8 heads 123 us, the copy bandwidth (128 with the rows asked for
// after their places).  In a long run the power cap takes clocks away, and instructions then count: packed maxima, packed
// products and rounding by addition keep it at 122.5 us where one value at a time took 132 (int8; at 1.7 GHz).  8430 tokens of two heads in pages take 4.4 us, mostly a launch and two trips to memory.
template <int kCode>
__global__ void __launch_bounds__(kThreads) q8_fill_kernel(const MoveParams p) {
  const int h = blockIdx.y, l = threadIdx.x % kLanes;
  const int64_t t = (int64_t)blockIdx.x * kTile + threadIdx.x / kLanes;
  if (p.seqlens_out != nullptr && h == 0)
    for (int64_t b = (int64_t)blockIdx.x * kThreads + threadIdx.x; b < p.batch; b += (int64_t)gridDim.x * kThreads)
      p.seqlens_out[b] = (int32_t)min(max((int64_t)p.cu[b + 1] - p.cu[b] + (p.start ? p.start[b] : 0), (int64_t)0), p.capacity);
  uint4 raw[2][2];                               // (on their way while the row's place is looked up)
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint4* src = p.src[i] + t * p.token_stride[i] + h * p.head_stride[i] + l;
    raw[i][0] = t < p.total ? __ldg(src) : make_uint4(0u, 0u, 0u, 0u);
    raw[i][1] = t < p.total ? __ldg(src + kLanes) : make_uint4(0u, 0u, 0u, 0u);
  }
  const int64_t row0 = token_row(p, t);
  const bool on = row0 >= 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    // the largest of the even and of the odd features (bf16 magnitudes are ordered as their bits are)
    const uint4 &r0 = raw[i][0], &r1 = raw[i][1];
    constexpr uint32_t kAbs = 0x7FFF7FFFu;
    uint32_t top = __vimax3_u16x2(r0.x & kAbs, r0.y & kAbs, r0.z & kAbs);
    top = __vimax3_u16x2(top, r0.w & kAbs, r1.x & kAbs);
    top = __vimax3_u16x2(top, r1.y & kAbs, r1.z & kAbs);
    top = __vmaxu2(top, r1.w & kAbs);
#pragma unroll
    for (int d = 1; d < kLanes; d <<= 1) top = __vmaxu2(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
    if (!on) continue;
    const int byte = scale_byte<kCode>(max(top << 16, top & 0xFFFF0000u));
    float x[16];
    to_float(x, r0, r1);
    const int64_t row = p.place.row(row0, h);
    uint32_t c[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float y[4] = {x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]};
      c[j] = encode4<kCode>(y, byte);
    }
    uint2* out = reinterpret_cast<uint2*>(p.codes[i] + row * kHeadDim) + l;
    out[0] = make_uint2(c[0], c[1]);
    out[kLanes] = make_uint2(c[2], c[3]);
    if (l == 0) p.scales[i][row] = (uint8_t)byte;
  }
}

// The way back: one head of kTile tokens, eight threads per row; two 8-byte loads leave as vectors l and l + 8, whole
// sectors per store (65536 tokens of 8 heads 68 us, 91 % of the copy bandwidth, against 75 with 16 values in a row per
// thread; 7500 tokens of two heads in pages of 16 4.1 us).  A row that the cache does not have reads as NaN; rows behind
// the last sequence are zeros.
template <int kCode>
__global__ void __launch_bounds__(kThreads) q8_read_kernel(const MoveParams p) {
  const int h = blockIdx.y, l = threadIdx.x % kLanes;
  const int64_t t = (int64_t)blockIdx.x * kTile + threadIdx.x / kLanes;
  if (t >= p.total) return;
  const int64_t row0 = token_row(p, t);
  const int64_t row = row0 >= 0 ? p.place.row(row0, h) : 0;
  uint2 raw[2][2];
  int byte[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    raw[i][0] = raw[i][1] = make_uint2(0u, 0u);
    byte[i] = row0 == -2 ? 0 : kNanByte;
    if (row0 >= 0) {
      const uint2* src = reinterpret_cast<const uint2*>(p.codes[i] + row * kHeadDim) + l;
      raw[i][0] = __ldg(src);
      raw[i][1] = __ldg(src + kLanes);
      byte[i] = __ldg(p.scales[i] + row);
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float s = scale_value(byte[i]);
    uint4* out = p.dst[i] + (t * p.place.heads + h) * (kHeadDim / 8) + l;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      float x[8];
      uint32_t w[4];
      decode4<kCode>(*reinterpret_cast<float(*)[4]>(x), raw[i][v].x);
      decode4<kCode>(*reinterpret_cast<float(*)[4]>(x + 4), raw[i][v].y);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(mul_exact(x[2 * u], s), mul_exact(x[2 * u + 1], s));
        w[u] = *reinterpret_cast<const uint32_t*>(&b);
      }
      out[v * kLanes] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

struct AppendQ8Params {
  const __nv_bfloat16* src[2];   // (batch, heads, 128) new keys, values
  uint8_t* codes[2];
  uint8_t* scales[2];
  __nv_bfloat16* comp[2];        // (batch, comp_cap, heads, 128) compressed keys, or null
  int32_t* n_comp[2];            // (batch) or null
  int kernel[2], stride[2];
  int64_t comp_cap[2];
  int32_t* seqlens;              // (batch) in: lengths before the append, out: after it
  int32_t* positions;            // (batch) or null
  Place place;
};

// Mean of the last `kernel` keys of the sequence as the cache holds them, in token order; four features per thread.
template <int kCode>
__device__ __forceinline__ void window_mean(const AppendQ8Params& p, int b, int len, int kernel, __nv_bfloat16* dst) {
  for (int i = threadIdx.x; i < p.place.heads * (kHeadDim / 4); i += kThreads) {
    const int h = i / (kHeadDim / 4), f = i % (kHeadDim / 4);
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int t = 0; t < kernel; ++t) {
      const int64_t row = p.place.row(p.place.row0(b, len - kernel + t), h);
      float x[4];
      // (ordinary loads: the newest of these rows was written by this CTA)
      decode4<kCode>(x, reinterpret_cast<const uint32_t*>(p.codes[0] + row * kHeadDim)[f]);
      const float s = scale_value(p.scales[0][row]);
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] += mul_exact(x[j], s);
    }
    const float n = (float)kernel;
    __nv_bfloat162 lo = __floats2bfloat162_rn(__fdiv_rn(acc[0], n), __fdiv_rn(acc[1], n));
    __nv_bfloat162 hi = __floats2bfloat162_rn(__fdiv_rn(acc[2], n), __fdiv_rn(acc[3], n));
    *reinterpret_cast<uint2*>(dst + h * kHeadDim + 4 * f) =
        make_uint2(*reinterpret_cast<uint32_t*>(&lo), *reinterpret_cast<uint32_t*>(&hi));
  }
}

// One decode step of bookkeeping for one sequence per CTA (slots only): append, compression windows that the new
// token completes, lengths.  Every thread that reads the sequence's length sits in the CTA that later writes it.  Bound by
// latency: the length, the row and the window's rows, one after the other.  In a graph, with a window of 32 every 16 tokens:
// one sequence 2.8 us; 64 sequences of two heads, some of which complete a window at every step, 11.2 (the bf16 cache's kernel: 3.5).
template <int kCode>
__global__ void __launch_bounds__(kThreads) q8_append_kernel(const AppendQ8Params p) {
  const int b = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int old_len = p.seqlens[b];
  __syncthreads();
  const bool room = old_len >= 0 && old_len < p.place.length;      // a full cache is left untouched
  const int len = room ? old_len + 1 : old_len;
  if (room) {
    const int64_t row0 = p.place.row0(b, old_len);
    for (int i = warp; i < 2 * p.place.heads; i += kThreads / 32) {
      const int h = i >> 1, kind = i & 1;
      const int64_t row = p.place.row(row0, h);
      const uint2 raw = __ldg(reinterpret_cast<const uint2*>(p.src[kind] + ((int64_t)b * p.place.heads + h) * kHeadDim) + lane);
      const float x[4] = {__uint_as_float(raw.x << 16), __uint_as_float(raw.x & 0xFFFF0000u), __uint_as_float(raw.y << 16),
                          __uint_as_float(raw.y & 0xFFFF0000u)};
      store_row<kCode>(x, p.codes[kind] + row * kHeadDim, p.scales[kind] + row, lane);
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 2; ++c)
      if (p.comp[c] != nullptr && len >= p.kernel[c] && (len - p.kernel[c]) % p.stride[c] == 0 &&
          (len - p.kernel[c]) / p.stride[c] < p.comp_cap[c])
        window_mean<kCode>(p, b, len, p.kernel[c],
                           p.comp[c] + ((int64_t)b * p.comp_cap[c] + (len - p.kernel[c]) / p.stride[c]) * p.place.heads * kHeadDim);
  }
  if (threadIdx.x == 0) {
    p.seqlens[b] = len;
    if (p.positions != nullptr) p.positions[b] = old_len;
#pragma unroll
    for (int c = 0; c < 2; ++c)
      if (p.n_comp[c] != nullptr)
        p.n_comp[c][b] = (int32_t)min((int64_t)(len >= p.kernel[c] ? (len - p.kernel[c]) / p.stride[c] + 1 : 0), p.comp_cap[c]);
  }
}

}  // namespace
}  // namespace ifv2

using namespace ifv2;

// Whether na and nb numbers from a and b on share memory (null: they do not).
static bool overlap(const int32_t* a, int64_t na, const int32_t* b, int64_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return a != nullptr && b != nullptr && x < y + 4 * (uintptr_t)nb && y < x + 4 * (uintptr_t)na;
}

static int move_common(MoveParams& p, const char* what, void* k_cache, void* v_cache, void* k_scale, void* v_scale,
                       const int32_t* cu_seqlens, const int32_t* start, const int32_t* block_table, int block_table_stride,
                       int64_t slots, int64_t length, int code, int batch, int64_t total, int heads_k, int head_dim) {
  IFV2_REQUIRE(head_dim == kHeadDim, IFV2_ERR_UNSUPPORTED, "%s: head_dim %d not supported (only 128)", what, head_dim);
  IFV2_REQUIRE(code == kE4m3 || code == kInt8, IFV2_ERR_INVALID_ARG, "%s: code must be 0 (e4m3) or 1 (int8)", what);
  IFV2_REQUIRE(batch >= 1 && total >= 0 && heads_k >= 1 && slots >= 1 && length >= 1, IFV2_ERR_INVALID_ARG, "%s: bad size", what);
  IFV2_REQUIRE(k_cache && v_cache && k_scale && v_scale && cu_seqlens, IFV2_ERR_INVALID_ARG, "%s: null pointer", what);
  IFV2_REQUIRE(block_table == nullptr || block_table_stride >= 1, IFV2_ERR_INVALID_ARG, "%s: empty block table", what);
  IFV2_REQUIRE(block_table != nullptr || slots >= batch, IFV2_ERR_INVALID_ARG, "%s: fewer slots than sequences", what);
  IFV2_REQUIRE((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) % 16 == 0, IFV2_ERR_INVALID_ARG,
               "%s: tensors must be 16-byte aligned", what);
  IFV2_REQUIRE(total <= INT32_MAX && length <= INT32_MAX && slots <= INT32_MAX && heads_k <= 65535 &&
                   (block_table == nullptr || block_table_stride <= INT32_MAX / length),
               IFV2_ERR_TOO_LARGE, "%s: a size is too large", what);
  p.codes[0] = static_cast<uint8_t*>(k_cache);
  p.codes[1] = static_cast<uint8_t*>(v_cache);
  p.scales[0] = static_cast<uint8_t*>(k_scale);
  p.scales[1] = static_cast<uint8_t*>(v_scale);
  p.cu = cu_seqlens;
  p.start = start;
  p.place = q8::Place{block_table, nullptr, block_table_stride, heads_k, (int)length, (int)slots};
  p.batch = batch;
  p.total = total;
  p.capacity = block_table != nullptr ? (int64_t)block_table_stride * length : length;
  return IFV2_OK;
}

extern "C" int ifv2_q8_fill(const void* k, const void* v, int64_t k_token_stride, int64_t k_head_stride,
                            int64_t v_token_stride, int64_t v_head_stride, void* k_cache, void* v_cache, void* k_scale,
                            void* v_scale, const int32_t* cu_seqlens, const int32_t* start, const int32_t* block_table,
                            int block_table_stride, int32_t* seqlens_out, int64_t slots, int64_t length, int code, int batch,
                            int64_t total, int heads_k, int head_dim, void* stream) {
  MoveParams p{};
  int rc = move_common(p, "q8_fill", k_cache, v_cache, k_scale, v_scale, cu_seqlens, start, block_table, block_table_stride,
                       slots, length, code, batch, total, heads_k, head_dim);
  if (rc) return rc;
  IFV2_REQUIRE((k && v) || total == 0, IFV2_ERR_INVALID_ARG, "q8_fill: null pointer");
  IFV2_REQUIRE((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 16 == 0 &&
                   (k_token_stride | k_head_stride | v_token_stride | v_head_stride) % 8 == 0,
               IFV2_ERR_INVALID_ARG, "q8_fill: rows must be 16-byte aligned");
  IFV2_REQUIRE(!overlap(seqlens_out, batch, start, batch) && !overlap(seqlens_out, batch, cu_seqlens, (int64_t)batch + 1),
               IFV2_ERR_INVALID_ARG, "q8_fill: seqlens_out must not overlap start or cu_seqlens");
  p.src[0] = static_cast<const uint4*>(k);
  p.src[1] = static_cast<const uint4*>(v);
  p.token_stride[0] = k_token_stride / 8;
  p.head_stride[0] = k_head_stride / 8;
  p.token_stride[1] = v_token_stride / 8;
  p.head_stride[1] = v_head_stride / 8;
  p.seqlens_out = seqlens_out;
  int64_t blocks = ceil_div64(total, kTile);
  if (blocks < 1) blocks = 1;                   // (the lengths are written in any case)
  const dim3 grid((unsigned)blocks, heads_k);
  if (code == kE4m3) q8_fill_kernel<kE4m3><<<grid, kThreads, 0, (cudaStream_t)stream>>>(p);
  else q8_fill_kernel<kInt8><<<grid, kThreads, 0, (cudaStream_t)stream>>>(p);
  return check_launch("q8_fill");
}

extern "C" int ifv2_q8_read(const void* k_cache, const void* v_cache, const void* k_scale, const void* v_scale, void* k,
                            void* v, const int32_t* cu_seqlens, const int32_t* start, const int32_t* block_table,
                            int block_table_stride, int64_t slots, int64_t length, int code, int batch, int64_t total,
                            int heads_k, int head_dim, void* stream) {
  MoveParams p{};
  int rc = move_common(p, "q8_read", const_cast<void*>(k_cache), const_cast<void*>(v_cache), const_cast<void*>(k_scale),
                       const_cast<void*>(v_scale), cu_seqlens, start, block_table, block_table_stride, slots, length, code, batch,
                       total, heads_k, head_dim);
  if (rc) return rc;
  if (total == 0) return IFV2_OK;
  IFV2_REQUIRE(k && v, IFV2_ERR_INVALID_ARG, "q8_read: null pointer");
  IFV2_REQUIRE((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 16 == 0, IFV2_ERR_INVALID_ARG,
               "q8_read: tensors must be 16-byte aligned");
  p.dst[0] = static_cast<uint4*>(k);
  p.dst[1] = static_cast<uint4*>(v);
  const dim3 grid((unsigned)ceil_div64(total, kTile), heads_k);
  if (code == kE4m3) q8_read_kernel<kE4m3><<<grid, kThreads, 0, (cudaStream_t)stream>>>(p);
  else q8_read_kernel<kInt8><<<grid, kThreads, 0, (cudaStream_t)stream>>>(p);
  return check_launch("q8_read");
}

extern "C" int ifv2_q8_append(const void* k_new, const void* v_new, void* k_cache, void* v_cache, void* k_scale, void* v_scale,
                              void* kc_cache, void* kc2_cache, int32_t* cache_seqlens, int32_t* positions, int32_t* n_comp,
                              int32_t* n_comp2, int code, int batch, int64_t slots, int64_t capacity, int64_t c_capacity,
                              int64_t c2_capacity, int heads_k, int head_dim, int kernel_size, int kernel_stride,
                              int kernel2_size, int kernel2_stride, void* stream) {
  IFV2_REQUIRE(head_dim == kHeadDim, IFV2_ERR_UNSUPPORTED, "q8_append: head_dim %d not supported (only 128)", head_dim);
  IFV2_REQUIRE(code == kE4m3 || code == kInt8, IFV2_ERR_INVALID_ARG, "q8_append: code must be 0 (e4m3) or 1 (int8)");
  IFV2_REQUIRE(batch >= 1 && slots >= batch && heads_k >= 1 && capacity >= 1, IFV2_ERR_INVALID_ARG, "q8_append: bad size");
  IFV2_REQUIRE(k_new && v_new && k_cache && v_cache && k_scale && v_scale && cache_seqlens, IFV2_ERR_INVALID_ARG,
               "q8_append: null pointer");
  const int32_t* written[4] = {cache_seqlens, positions, n_comp, n_comp2};
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < i; ++j)
      IFV2_REQUIRE(!overlap(written[i], batch, written[j], batch), IFV2_ERR_INVALID_ARG,
                   "q8_append: cache_seqlens, positions and the counts must not overlap");
  IFV2_REQUIRE(kc_cache == nullptr || (c_capacity >= 1 && kernel_size >= 1 && kernel_stride >= 1), IFV2_ERR_INVALID_ARG,
               "q8_append: bad compression arguments");
  IFV2_REQUIRE(kc2_cache == nullptr || (c2_capacity >= 1 && kernel2_size >= 1 && kernel2_stride >= 1), IFV2_ERR_INVALID_ARG,
               "q8_append: bad second compression arguments");
  IFV2_REQUIRE((n_comp == nullptr || kc_cache != nullptr) && (n_comp2 == nullptr || kc2_cache != nullptr), IFV2_ERR_INVALID_ARG,
               "q8_append: a count output needs its compressed cache");
  for (const void* ptr : {k_new, v_new, (const void*)k_cache, (const void*)v_cache, (const void*)kc_cache, (const void*)kc2_cache})
    IFV2_REQUIRE(reinterpret_cast<uintptr_t>(ptr) % 16 == 0, IFV2_ERR_INVALID_ARG, "q8_append: tensors must be 16-byte aligned");
  IFV2_REQUIRE(batch <= 1 << 30 && slots <= INT32_MAX && capacity <= INT32_MAX - 1, IFV2_ERR_TOO_LARGE, "q8_append: a size is too large");
  const AppendQ8Params p{{static_cast<const __nv_bfloat16*>(k_new), static_cast<const __nv_bfloat16*>(v_new)},
                         {static_cast<uint8_t*>(k_cache), static_cast<uint8_t*>(v_cache)},
                         {static_cast<uint8_t*>(k_scale), static_cast<uint8_t*>(v_scale)},
                         {static_cast<__nv_bfloat16*>(kc_cache), static_cast<__nv_bfloat16*>(kc2_cache)},
                         {n_comp, n_comp2},
                         {kc_cache ? kernel_size : 1, kc2_cache ? kernel2_size : 1},
                         {kc_cache ? kernel_stride : 1, kc2_cache ? kernel2_stride : 1},
                         {c_capacity, c2_capacity},
                         cache_seqlens,
                         positions,
                         Place{nullptr, nullptr, 0, heads_k, (int)capacity, (int)slots}};
  if (code == kE4m3) q8_append_kernel<kE4m3><<<batch, kThreads, 0, (cudaStream_t)stream>>>(p);
  else q8_append_kernel<kInt8><<<batch, kThreads, 0, (cudaStream_t)stream>>>(p);
  return check_launch("q8_append");
}
