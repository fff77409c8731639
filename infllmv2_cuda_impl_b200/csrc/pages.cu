// Pages of a cache: the block tables and slots of a step, and bf16 rows written by slot.
//
// A request of n tokens has ceil(n / page_size) pages, whose numbers stand in its row of the block table.  Pages that
// nobody has stand in a ring: `count` of them from `first` on.  A step takes pages from the front of the ring, in
// the order of the requests, and puts those of requests that became shorter behind its end.  The two stretches do not
// meet (pages in the ring and in the table are at most the ring's size), and what is read (lengths, first and count) is
// never written, so CTAs need not wait for one another and a call that is made twice gives the same twice.
//
// What bounds it is latency: lengths, their sums, a page's number, its slot follow one another.  Every CTA adds up all
// requests by itself (a second launch or a wait for another CTA would cost more than the 1-2 us of a few thousand).
// Measured on the device: a decode step of 64 requests 4.6 us (2.3 of them an empty launch), 131072 new tokens among 256
// requests 9.6 us.
#include "beside.cuh"

namespace ifv2 {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxBatch = 16384;                 // 12 bytes of shared memory each

struct ResizeParams {
  const int32_t *seqlens, *targets;
  int32_t* table;
  int64_t table_stride;
  int32_t* ring;
  const int32_t* range;                          // (first, count)
  int32_t *seqlens_out, *range_out, *cu, *positions;
  int64_t* slots;
  int batch, width, num_pages, page_size;
  int64_t total;
};

// Inclusive sums of three numbers over the CTA.
__device__ __forceinline__ void block_scan3(int64_t (&v)[3], int64_t* scratch) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int k = 0; k < 3; ++k)
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t o = __shfl_up_sync(0xFFFFFFFFu, v[k], d);
      if (lane >= d) v[k] += o;
    }
  if (lane == 31)
    for (int k = 0; k < 3; ++k) scratch[k * 8 + warp] = v[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 3; ++k)
    for (int w = 0; w < warp; ++w) v[k] += scratch[k * 8 + w];
  __syncthreads();
}

// Place `off` behind `first` in a ring; neither is above its size.  (A 64-bit remainder takes some 100 instructions.)
__device__ __forceinline__ int ring_at(int first, int off, int ring) {
  const uint32_t x = (uint32_t)first + (uint32_t)off;
  return (int)(x >= (uint32_t)ring ? x - (uint32_t)ring : x);
}

__device__ __forceinline__ int pages_of(int tokens, int page_size) {
  return (int)(((uint32_t)tokens + (uint32_t)page_size - 1) / (uint32_t)page_size);
}

__device__ __forceinline__ int sat32(int64_t x) { return (int)min(x, (int64_t)0x7FFFFFFF); }

__global__ void __launch_bounds__(kThreads) pages_resize_kernel(const ResizeParams p) {
  extern __shared__ int32_t smem[];
  int32_t* s_cu = smem;                          // (batch + 1) first row of each request's new tokens
  int32_t* s_old = smem + p.batch + 1;           // (batch)
  int32_t* s_take = s_old + p.batch;             // (batch) pages that requests before it take; -1: refused
  __shared__ int64_t scratch[24];
  __shared__ int64_t s_back[kThreads];           // of the chunk's requests: pages given back up to it, pages before and after
  __shared__ int s_had[kThreads], s_want[kThreads];
  __shared__ int64_t s_sum[2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  allow_next();
  wait_previous();
  const int ring = p.num_pages;
  const int place = p.range[0] % ring, first = place < 0 ? place + ring : place;
  const int count = min(max(p.range[1], 0), ring);
  const int64_t reach = (int64_t)p.width * p.page_size;

  int64_t before[3] = {0, 0, 0};                 // new tokens, pages asked for, pages given back by earlier chunks
  int64_t taken = 0;                             // pages that granted requests take
  for (int base = 0; base < p.batch; base += kThreads) {
    const int b = base + tid;
    int64_t v[3] = {0, 0, 0};
    int old = 0, target = 0, had = 0, want = 0;
    if (b < p.batch) {
      old = (int)min((int64_t)max(p.seqlens[b], 0), reach);
      target = max(p.targets[b], 0);
      had = pages_of(old, p.page_size);
      want = pages_of(target, p.page_size);
      v[0] = max(target - old, 0);
      if (want <= p.width) v[1] = max(want - had, 0);
      v[2] = max(had - want, 0);
    }
    const int64_t mine[3] = {v[0], v[1], v[2]};
    block_scan3(v, scratch);
    s_back[tid] = before[2] + v[2];
    s_had[tid] = had, s_want[tid] = want;
    if (tid == kThreads - 1) s_sum[0] = before[0] + v[0], s_sum[1] = before[1] + v[1];
    const bool granted = want <= p.width && (mine[1] == 0 || before[1] + v[1] <= count);
    if (b < p.batch) {
      s_cu[b] = sat32(before[0] + v[0] - mine[0]);
      s_old[b] = old;
      s_take[b] = granted ? (int)min(before[1] + v[1] - mine[1], (int64_t)count) : -1;
      if (blockIdx.x == 0) {
        p.cu[b] = s_cu[b];
        p.seqlens_out[b] = granted ? target : old;
      }
    }
    // the last sum of pages that fits is what all granted requests take: sums only grow
    {
      const int64_t upto = before[1] + v[1];
      const int fits = (b < p.batch && upto <= count) ? (int)upto : 0;
      const int most = __reduce_max_sync(0xFFFFFFFFu, fits);
      if (lane == 0) scratch[warp] = most;
      __syncthreads();
      for (int w = 0; w < kThreads / 32; ++w) taken = max(taken, scratch[w]);
      __syncthreads();
    }
    // the table's rows and the ring, a warp per request
    const int here = min(kThreads, p.batch - base);
    for (int r = warp; r < here; r += kThreads / 32) {
      const int req = base + r;
      if (req % gridDim.x != blockIdx.x) continue;
      const int take = s_take[req];
      if (take < 0) continue;
      const int had_r = s_had[r], want_r = s_want[r];
      int32_t* row = p.table + (int64_t)req * p.table_stride;
      for (int i = had_r + lane; i < want_r; i += 32)
        row[i] = p.ring[ring_at(first, take + i - had_r, ring)];
      const int64_t behind = s_back[r] - max(had_r - want_r, 0);             // pages given back by earlier requests
      for (int i = want_r + lane; i < had_r; i += 32)
        p.ring[(int)(((int64_t)first + count + behind + i - want_r) % ring)] = row[i];
    }
    before[0] = s_sum[0], before[1] = s_sum[1], before[2] = s_back[kThreads - 1];
    __syncthreads();
  }
  if (tid == 0) {
    s_cu[p.batch] = sat32(before[0]);
    if (blockIdx.x == 0) {
      p.cu[p.batch] = sat32(before[0]);
      p.range_out[0] = (int)((first + taken) % ring);
      p.range_out[1] = (int)min(count - taken + before[2], (int64_t)ring);
    }
  }
  __syncthreads();

  const int64_t rows = min(p.total, before[0]);
  for (int64_t t = (int64_t)blockIdx.x * kThreads + tid; t < p.total; t += (int64_t)gridDim.x * kThreads) {
    int pos = 0;
    int64_t slot = -1;
    if (t < rows) {
      const int b = find_sequence(s_cu, p.batch, (int)t);
      pos = s_old[b] + (int)(t - s_cu[b]);
      const int take = s_take[b];
      if (take >= 0) {
        const int i = pos / p.page_size, had = pages_of(s_old[b], p.page_size);
        // (a page of this step may not stand in the table yet: it is looked up where the table's row gets it from)
        const int page = i < had ? p.table[(int64_t)b * p.table_stride + i]
                                 : p.ring[ring_at(first, take + i - had, ring)];
        if (page >= 0) slot = (int64_t)page * p.page_size + (pos - i * p.page_size);
      }
    }
    p.positions[t] = pos;
    p.slots[t] = slot;
  }
}

// ---------------------------------------------------------------------------- rows by slot --
// Copies of 16 bytes.  A CTA takes kTokens tokens, whose slots it looks up once; a thread has four copies under way.  Bound by
// memory: 65536 tokens of 8 heads 85 us for 537 MB, 96 % of the copy bandwidth; 8432 tokens of 2 heads 3.8 us, of which 2.3 are a launch.
constexpr int kTokens = 8;

struct WriteParams {
  const uint4 *k, *v;
  int64_t k_token, k_head, v_token, v_head;      // strides in 16-byte pieces
  uint4 *k_cache, *v_cache;
  const int64_t* slots;
  int64_t total, rows;                           // rows of the cache: pages * page_size
  int heads;
};

__global__ void __launch_bounds__(kThreads) cache_write_kernel(const WriteParams p) {
  __shared__ int64_t s_slot[kTokens];
  allow_next();
  wait_previous();
  const int64_t t0 = (int64_t)blockIdx.x * kTokens;
  const int tokens = (int)min((int64_t)kTokens, p.total - t0);
  if (threadIdx.x < tokens) {
    const int64_t s = p.slots[t0 + threadIdx.x];
    s_slot[threadIdx.x] = s >= 0 && s < p.rows ? s : -1;
  }
  __syncthreads();
  const int per = p.heads * 16, all = tokens * per * 2;       // 16-byte pieces of a token's keys, of the CTA
  for (int i0 = threadIdx.x; i0 < all; i0 += 4 * kThreads) {
    uint4 x[4];
    uint4* to[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + u * kThreads;
      to[u] = nullptr;
      if (i < all) {
        const int t = i / (2 * per), j = i - t * 2 * per;
        const bool val = j >= per;
        const int h = (val ? j - per : j) >> 4, c = j & 15;
        const int64_t slot = s_slot[t];
        if (slot >= 0) {
          const uint4* from = val ? p.v + (t0 + t) * p.v_token + h * p.v_head : p.k + (t0 + t) * p.k_token + h * p.k_head;
          x[u] = __ldcs(from + c);
          to[u] = (val ? p.v_cache : p.k_cache) + (slot * p.heads + h) * 16 + c;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (to[u]) *to[u] = x[u];
  }
}

}  // namespace
}  // namespace ifv2

using namespace ifv2;

extern "C" int ifv2_pages_resize(const int32_t* seqlens, const int32_t* targets, int32_t* block_table, int64_t table_stride,
                                 int width, int32_t* free_pages, int num_pages, const int32_t* free_range,
                                 int32_t* seqlens_out, int32_t* free_range_out, int32_t* cu_seqlens, int32_t* positions,
                                 int64_t* slots, int batch, int page_size, int64_t total, void* stream) {
  IFV2_REQUIRE(batch >= 1 && width >= 1 && num_pages >= 1 && page_size >= 1 && total >= 0, IFV2_ERR_INVALID_ARG,
               "pages_resize: sizes must be positive");
  IFV2_REQUIRE(batch <= kMaxBatch, IFV2_ERR_TOO_LARGE, "pages_resize: at most %d requests", kMaxBatch);
  IFV2_REQUIRE((int64_t)width * page_size < (1ll << 31) && total < (1ll << 31), IFV2_ERR_TOO_LARGE,
               "pages_resize: a request's positions and the new tokens must be below 2^31");
  IFV2_REQUIRE(table_stride >= width || batch == 1, IFV2_ERR_INVALID_ARG, "pages_resize: rows of the block table overlap");
  IFV2_REQUIRE(seqlens && targets && block_table && free_pages && free_range && seqlens_out && free_range_out && cu_seqlens &&
               ((positions && slots) || total == 0), IFV2_ERR_INVALID_ARG, "pages_resize: null pointer");
  ResizeParams p{seqlens, targets, block_table, table_stride, free_pages, free_range, seqlens_out, free_range_out,
                 cu_seqlens, positions, slots, batch, width, num_pages, page_size, total};
  const int smem = 4 * (3 * batch + 1);
  if (smem > 40 * 1024) {                          // (beside the static part; for all sizes at once, as calls may be made by several threads)
    const cudaError_t e = cudaFuncSetAttribute(pages_resize_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 4 * (3 * kMaxBatch + 1));
    if (e != cudaSuccess) return set_error((int)e, "pages_resize: %s", cudaGetErrorString(e));
  }
  // a CTA per 256 tokens or 8 requests, up to two per SM (131072 new tokens: 10.3 us with one, 9.6 with two, 11.2 with four)
  const int64_t want = max(ceil_div64(total, 256), (int64_t)ceil_div(batch, 8));
  const int most = smem <= 100 * 1024 ? 2 * kNumSMs : kNumSMs;
  const int grid = (int)min(max(want, (int64_t)1), (int64_t)most);
  const cudaError_t e = launch_beside(pages_resize_kernel, dim3(grid), kThreads, smem, (cudaStream_t)stream, p);
  if (e != cudaSuccess) return set_error((int)e, "pages_resize: %s", cudaGetErrorString(e));
  return check_launch("pages_resize");
}

extern "C" int ifv2_cache_write(const void* k, const void* v, int64_t k_token, int64_t k_head, int64_t v_token, int64_t v_head,
                                void* k_cache, void* v_cache, const int64_t* slots, int64_t num_pages, int page_size,
                                int64_t total, int heads_k, int head_dim, void* stream) {
  IFV2_REQUIRE(head_dim == kHeadDim, IFV2_ERR_UNSUPPORTED, "cache_write: head_dim must be %d", kHeadDim);
  IFV2_REQUIRE(num_pages >= 0 && page_size >= 1 && total >= 0 && heads_k >= 1 && heads_k <= 4096, IFV2_ERR_INVALID_ARG,
               "cache_write: bad sizes");
  if (total == 0 || num_pages == 0) return IFV2_OK;
  IFV2_REQUIRE(total < (1ll << 31), IFV2_ERR_TOO_LARGE, "cache_write: at most 2^31 - 1 tokens");
  IFV2_REQUIRE(k && v && k_cache && v_cache && slots, IFV2_ERR_INVALID_ARG, "cache_write: null pointer");
  IFV2_REQUIRE(((k_token | k_head | v_token | v_head) & 7) == 0 &&
               ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(k_cache) |
                 reinterpret_cast<uintptr_t>(v_cache)) & 15) == 0,
               IFV2_ERR_INVALID_ARG, "cache_write: rows must begin at multiples of 16 bytes");
  WriteParams p{static_cast<const uint4*>(k), static_cast<const uint4*>(v), k_token / 8, k_head / 8, v_token / 8, v_head / 8,
                static_cast<uint4*>(k_cache), static_cast<uint4*>(v_cache), slots, total, num_pages * page_size, heads_k};
  const cudaError_t e = launch_beside(cache_write_kernel, dim3((unsigned)ceil_div64(total, kTokens)), kThreads, 0, (cudaStream_t)stream, p);
  if (e != cudaSuccess) return set_error((int)e, "cache_write: %s", cudaGetErrorString(e));
  return check_launch("cache_write");
}
