// Rows written by slot into a cache in 8 bits with block scales (b8.cuh).
//
// Consecutive tokens of the call whose slots follow one another within a block are a run: at most 64 rows, which
// get one scale.  A run that begins a block decides its scale; one that begins inside a block may only raise it, and
// where it does, the block's earlier codes are rounded to the new scale.  (Powers of two make that harmless for these
// types: a code only changes where it becomes one of the type's subnormal numbers.)
//
// One CTA looks through a segment of kSeg tokens for the runs that begin there, for one head of the keys or values.
// Runs of more than 16 rows are taken by the whole CTA, shorter ones by a warp each; the rows stay in registers
// between the maximum and the codes, so that they are read once.  What bounds it is memory where tokens are many (131072
// tokens of 8 heads: 131 us for 806 MB, 94 % of the copy bandwidth; its arithmetic alone keeps the schedulers 70 % busy), and
// the way from slot to row to scale to code where they are few (64 tokens: 2.8 us, of which 2.3 are a launch).  Sixteen lanes
// with eight values for a row, two rows a step, eight CTAs per SM: with a lane for four values 183 us, with four CTAs 156.
#include "b8.cuh"
#include "beside.cuh"

namespace ifv2 {
namespace {

using namespace b8;

constexpr int kThreads = 128, kWarps = kThreads / 32;
constexpr int kBlock = kBlockN;                  // tokens of a block
constexpr int kRowsPerWarp = 16, kSteps = kRowsPerWarp / 2;

struct B8WriteParams {
  const uint4 *k, *v;
  int64_t k_token, k_head, v_token, v_head;      // strides in pieces of eight values
  uint8_t *k_cache, *v_cache, *k_scale, *v_scale;
  const int64_t* slots;
  int64_t total, limit;                          // tokens; slots of the cache
  int heads, page_size, segment;
};

__device__ __forceinline__ uint32_t amax_of(const uint4& x, uint32_t amax) {
  // bf16 magnitudes are ordered as their bits
  amax = __vmaxu2(__vmaxu2(x.x & 0x7FFF7FFFu, x.y & 0x7FFF7FFFu), amax);
  return __vmaxu2(__vmaxu2(x.z & 0x7FFF7FFFu, x.w & 0x7FFF7FFFu), amax);
}
template <int kCode>
__device__ __forceinline__ uint32_t encode_pairs(uint32_t a, uint32_t b, float inv) {
  const float y[4] = {__uint_as_float(a << 16), __uint_as_float(a & 0xFFFF0000u), __uint_as_float(b << 16), __uint_as_float(b & 0xFFFF0000u)};
  return encode4<kCode>(y, inv);
}

// kAll: the CTA's warps share the run; otherwise one warp has it to itself.  `n` rows from token t0 on.  A warp takes two rows
// at a time, 16 lanes each with 8 values.
template <int kCode, bool kAll>
__device__ __forceinline__ void write_run(const B8WriteParams& p, int64_t t0, int n, int64_t slot, int head, bool val, uint32_t* s_max) {
  const int lane = threadIdx.x & 31, warp = kAll ? threadIdx.x >> 5 : 0, piece = lane & 15;
  constexpr int kStep = 2 * (kAll ? kWarps : 1);
  const int r0 = 2 * warp + (lane >> 4);
  const int64_t token = val ? p.v_token : p.k_token;
  const uint4* src = (val ? p.v : p.k) + (t0 + r0) * token + (int64_t)head * (val ? p.v_head : p.k_head) + piece;
  uint4 x[kSteps];
#pragma unroll
  for (int i = 0; i < kSteps; ++i, src += kStep * token) x[i] = r0 + i * kStep < n ? __ldcs(src) : make_uint4(0u, 0u, 0u, 0u);
  const int64_t page = slot / p.page_size;
  const int place = (int)(slot - page * p.page_size), off = place & (kBlock - 1);
  uint8_t* scale = (val ? p.v_scale : p.k_scale) + (page * p.heads + head) * (p.page_size / kBlock) + place / kBlock;
  const int before = off > 0 ? *scale : 0;
  uint32_t m2 = 0;
#pragma unroll
  for (int i = 0; i < kSteps; ++i) m2 = amax_of(x[i], m2);
  uint32_t amax = __reduce_max_sync(0xFFFFFFFFu, max(m2 & 0xFFFFu, m2 >> 16));
  if (kAll) {
    if (lane == 0) s_max[warp] = amax;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) amax = max(amax, s_max[w]);
  }
  const int byte = max(scale_byte<kCode>(amax << 16), before);
  uint8_t* rows = (val ? p.v_cache : p.k_cache) + ((page * p.heads + head) * (int64_t)p.page_size + place) * kHeadDim + piece * 8;
  if (byte > before && off > 0 && byte != kNanByte) {            // earlier rows of the block: to the new scale
    const float down = __uint_as_float((uint32_t)(127 - min(byte - before, 64)) << 23);
    for (int r = r0 - off; r < 0; r += kStep) {
      uint2* at = reinterpret_cast<uint2*>(rows + (int64_t)r * kHeadDim);
      const uint2 c = *at;
      float a[4], b[4];
      decode4<kCode>(a, c.x);
      decode4<kCode>(b, c.y);
      *at = make_uint2(encode4<kCode>(a, down), encode4<kCode>(b, down));
    }
  }
  uint8_t* to = rows + r0 * kHeadDim;
  if (byte == kNanByte) {
#pragma unroll
    for (int i = 0; i < kSteps; ++i) x[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  const float inv = q8::inverse_scale(byte);
#pragma unroll
  for (int i = 0; i < kSteps; ++i)
    if (r0 + i * kStep < n)
      *reinterpret_cast<uint2*>(to + i * kStep * kHeadDim) = make_uint2(encode_pairs<kCode>(x[i].x, x[i].y, inv), encode_pairs<kCode>(x[i].z, x[i].w, inv));
  if (kAll) __syncthreads();                     // s_max is free again; `before` has been read by every warp
  else __syncwarp();
  if (warp == 0 && lane == 0) *scale = (uint8_t)byte;
}

template <int kCode>
__global__ void __launch_bounds__(kThreads, 8) b8_write_kernel(const B8WriteParams p) {
  __shared__ int64_t s_slot[2 * kBlock + 1];     // of the token before the segment, the segment's, and 63 behind it
  __shared__ uint64_t s_start;                   // tokens of the segment that begin a run
  __shared__ uint64_t s_end[2];                  // tokens (from the segment's first on) that do not continue one
  __shared__ uint32_t s_max[kWarps];
  allow_next();
  wait_previous();
  const int64_t t0 = (int64_t)blockIdx.x * p.segment;
  const int head = blockIdx.y >> 1;
  const bool val = blockIdx.y & 1;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid < 2) s_end[tid] = 0;
  if (tid == 2) s_start = 0;
  for (int i = tid; i < 2 * kBlock + 1; i += kThreads) {
    const int64_t t = t0 - 1 + i;
    const int64_t s = t >= 0 && t < p.total ? p.slots[t] : -1;
    s_slot[i] = s >= 0 && s < p.limit ? s : -1;
  }
  __syncthreads();
  {
    const int64_t s = s_slot[tid + 1], prev = s_slot[tid];
    const bool more = s >= 0 && s == prev + 1 && (s & (kBlock - 1)) != 0;       // (pages are whole blocks)
    const uint32_t ends = __ballot_sync(0xFFFFFFFFu, !more), starts = __ballot_sync(0xFFFFFFFFu, !more && s >= 0 && tid < p.segment);
    if (lane == 0) {
      reinterpret_cast<uint32_t*>(s_end)[warp] = ends;
      if (warp < 2) reinterpret_cast<uint32_t*>(&s_start)[warp] = starts;
    }
  }
  __syncthreads();
  const uint64_t e0 = s_end[0], e1 = s_end[1];
  int turn = 0;
  // runs of one warp first: they need no barrier
  for (uint64_t left = s_start; left != 0; left &= left - 1) {
    const int i = __ffsll((long long)left) - 1;
    const uint64_t behind = i == 63 ? e1 : (e0 >> (i + 1)) | (e1 << (63 - i));
    const int n = behind ? __ffsll((long long)behind) : kBlock;
    if (n <= kRowsPerWarp && (turn++ & (kWarps - 1)) == warp) write_run<kCode, false>(p, t0 + i, n, s_slot[i + 1], head, val, s_max);
  }
  for (uint64_t left = s_start; left != 0; left &= left - 1) {
    const int i = __ffsll((long long)left) - 1;
    const uint64_t behind = i == 63 ? e1 : (e0 >> (i + 1)) | (e1 << (63 - i));
    const int n = behind ? __ffsll((long long)behind) : kBlock;
    if (n > kRowsPerWarp) write_run<kCode, true>(p, t0 + i, n, s_slot[i + 1], head, val, s_max);
  }
}

}  // namespace
}  // namespace ifv2

using namespace ifv2;

extern "C" int ifv2_b8_write(const void* k, const void* v, int64_t k_token, int64_t k_head, int64_t v_token, int64_t v_head,
                             void* k_cache, void* v_cache, void* k_scale, void* v_scale, const int64_t* slots, int64_t num_pages,
                             int page_size, int code, int64_t total, int heads_k, int head_dim, void* stream) {
  IFV2_REQUIRE(head_dim == kHeadDim, IFV2_ERR_UNSUPPORTED, "b8_write: head_dim must be %d", kHeadDim);
  IFV2_REQUIRE(code == kE4m3 || code == kE5m2, IFV2_ERR_INVALID_ARG, "b8_write: code must be 0 (e4m3) or 1 (e5m2)");
  IFV2_REQUIRE(num_pages >= 0 && page_size >= kBlockN && page_size % kBlockN == 0 && total >= 0 && heads_k >= 1, IFV2_ERR_INVALID_ARG,
               "b8_write: pages must be a positive multiple of %d positions", kBlockN);
  IFV2_REQUIRE(heads_k <= 32767 && total < (1ll << 31), IFV2_ERR_TOO_LARGE, "b8_write: at most 32767 heads and 2^31 - 1 tokens");
  if (total == 0 || num_pages == 0) return IFV2_OK;
  IFV2_REQUIRE(k && v && k_cache && v_cache && k_scale && v_scale && slots, IFV2_ERR_INVALID_ARG, "b8_write: null pointer");
  IFV2_REQUIRE(((k_token | k_head | v_token | v_head) & 7) == 0 &&
               ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0 &&
               ((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 7) == 0,
               IFV2_ERR_INVALID_ARG, "b8_write: rows of k and v must begin at multiples of 16 bytes, caches at multiples of 8");
  // The longest segment that still gives every SM a few CTAs: with short ones many CTAs find that no run begins in
  // theirs, with long ones the runs of a decode step queue up in few.
  int segment = kBlockN;
  while (segment > 1 && ceil_div64(total, segment) * heads_k * 2 < 4 * kNumSMs) segment /= 4;
  B8WriteParams p{static_cast<const uint4*>(k), static_cast<const uint4*>(v), k_token / 8, k_head / 8, v_token / 8, v_head / 8,
                  static_cast<uint8_t*>(k_cache), static_cast<uint8_t*>(v_cache), static_cast<uint8_t*>(k_scale),
                  static_cast<uint8_t*>(v_scale), slots, total, num_pages * page_size, heads_k, page_size, segment};
  const dim3 grid((unsigned)ceil_div64(total, segment), 2 * heads_k);
  const cudaError_t e = launch_beside(code == kE4m3 ? b8_write_kernel<kE4m3> : b8_write_kernel<kE5m2>, grid, kThreads, 0,
                                      (cudaStream_t)stream, p);
  if (e != cudaSuccess) return set_error((int)e, "b8_write: %s", cudaGetErrorString(e));
  return check_launch("b8_write");
}
