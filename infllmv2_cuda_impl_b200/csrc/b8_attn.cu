// Attention over 8-bit blocks: the list of tiles of a call with long sequences, the join of tiles that shares cut, and
// the C entry (formulas and shares: b8_attn.cuh).
#include "b8_attn.cuh"

namespace ifv2 {
namespace {

using namespace b8;

constexpr int kPlanThreads = 1024, kJoinThreads = 128;
// Blocks that a token's mask row is taken to select: how many CTAs get a share follows from it.  A count would be a pass over the
// masks in front.  Where sequences are many it matters little (64 sequences of 32768 tokens, 16 / 64 / 256 / 512 blocks each: 21.4 / 36.3 /
// 95.0 / 177 us, as lists, whose length is known, 15.7 / 34.3 / 99.0 / 180); one token alone walks masks of more blocks in few CTAs (131072
// tokens, 64 / 256 / 512 / 2048 blocks: 13.5 / 23.8 / 37.3 / 118 us, as lists 12.0 / 15.8 / 18.1 / 57.6, without a selection 30).
constexpr int kUsualBlocks = 64;
constexpr int kTokensPerTile = 8;                // of listed tiles

__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* scratch) {      // inclusive, over kPlanThreads
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t o = __shfl_up_sync(0xFFFFFFFFu, v, d);
    if (lane >= d) v += o;
  }
  if (lane == 31) scratch[warp] = v;
  __syncthreads();
  if (warp == 0) {
    int64_t w = scratch[lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t o = __shfl_up_sync(0xFFFFFFFFu, w, d);
      if (lane >= d) w += o;
    }
    scratch[lane] = w;
  }
  __syncthreads();
  if (warp > 0) v += scratch[warp - 1];
  return v;
}

// One CTA: chunks of eight tokens per sequence, tiles and their costs, and the tile that each CTA begins with.
__global__ void __launch_bounds__(kPlanThreads) b8_plan_kernel(const AttnParams p, int grid_most) {
  constexpr int kT = kTokensPerTile;
  __shared__ int64_t scratch[32], s_total;
  const int tid = threadIdx.x;
  allow_next();
  wait_inputs();
  int64_t before = 0;
  for (int base = 0; base < p.batch; base += kPlanThreads) {
    const int b = base + tid;
    int row0;
    const int64_t n = b < p.batch ? ceil_div(tokens_of(p, b, row0), kT) : 0;
    const int64_t upto = before + block_scan(n, scratch);
    if (b < p.batch) p.first_chunk[b] = (int)min(upto - n, (int64_t)p.most_chunks);
    if (tid == kPlanThreads - 1) s_total = upto;
    __syncthreads();
    before = s_total;
    __syncthreads();
  }
  const int chunks = (int)min(before, (int64_t)p.most_chunks);
  if (tid == 0) p.first_chunk[p.batch] = chunks;
  __syncthreads();
  const int tiles = chunks * p.heads_k;
  before = 0;
  for (int base = 0; base < tiles; base += kPlanThreads) {
    const int i = base + tid;
    int64_t cost = 0;
    if (i < tiles) {
      const int chunk = i / p.heads_k, head = i - chunk * p.heads_k;
      int b = 0, row0;                           // largest b with first_chunk[b] <= chunk
      for (int hi = p.batch; hi - b > 1;) {
        const int mid = (b + hi) >> 1;
        if (p.first_chunk[mid] <= chunk) b = mid; else hi = mid;
      }
      const int n = tokens_of(p, b, row0), t0 = (chunk - p.first_chunk[b]) * kT, tokens = max(min(kT, n - t0), 0);
      const int len = keys_of(p, b), reach = max(p.causal ? len - n + t0 + tokens : len, 0);
      p.tiles[i] = make_int4(b, row0 + t0, reach, tokens << 16 | head);
      int units = ceil_div(reach, kUnit);
      if (p.mask || p.lists) units = min(units, ceil_div(p.usual * (3 + tokens), 8));
      cost = kStart + units;
    }
    const int64_t upto = before + block_scan(cost, scratch);
    if (i < tiles) p.start[i] = upto - cost;
    if (tid == kPlanThreads - 1) s_total = upto;
    __syncthreads();
    before = s_total;
    __syncthreads();
  }
  if (tid == 0) {
    p.start[tiles] = before;
    p.first_tile[grid_most] = tiles;
  }
  __syncthreads();
  Shares<int64_t> shares;
  shares.deal(max(before, (int64_t)1), grid_most, p.least_share);
  for (int g = tid; g < grid_most; g += kPlanThreads) {
    const int64_t at = shares.begin(min(g, shares.grid - 1));
    int lo = 0, hi = tiles;                        // start[lo] <= at < start[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (p.start[mid] <= at) lo = mid; else hi = mid;
    }
    p.first_tile[g] = lo;
  }
}

// The pieces of a tile that shares cut: CTA x has tile x (where tiles are few), or the tile that share x begins inside if no
// earlier share does; join[x] says whether there is one.
// Piece results are normal outputs with the log2 of their sums.  A warp has a head; where tiles are few and pieces many (one
// sequence of 12001 tokens, two heads: 32 pieces a tile), the four warps of a CTA share a head's pieces.  Also: rows behind
// the last sequence.
// What bounds it is latency: trips to memory of 0.7 us, here two.  (A warp stops at the first instruction that wants a number
// that is not there yet, so what does not depend on it is asked for before.)
template <bool kShared>
__global__ void __launch_bounds__(kJoinThreads) b8_join_kernel(const AttnParams p, int tokens_per_tile, int shares) {
  __shared__ float4 s_acc[4][32];
  __shared__ float s_sum[4];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, heads = p.heads_k * kGroup, columns = kGroup * tokens_per_tile;
  allow_next();
  wait_inputs();
  const int4 cut = p.join[blockIdx.x];
  const int rows = p.cu_q[p.batch];
  int row0 = 0, some = 1;
  if (p.by_tile) some = tokens_of(p, blockIdx.x / p.heads_k, row0);        // (a sequence without tokens has no tile)
  if (rows < p.total_q) {
    const int64_t me = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * kJoinThreads + tid, all = (int64_t)gridDim.x * gridDim.y * kJoinThreads;
    uint4* out = reinterpret_cast<uint4*>(p.out);
    for (int64_t i = (int64_t)max(rows, 0) * heads * 16 + me; i < p.total_q * heads * 16; i += all) out[i] = make_uint4(0, 0, 0, 0);
    if (p.lse)
      for (int64_t i = (int64_t)max(rows, 0) * heads + me; i < p.total_q * heads; i += all) p.lse[i] = INFINITY;
  }
  const int column = kShared ? blockIdx.y : blockIdx.y * 4 + warp, tok = column / kGroup;
  if (some == 0 || cut.z >= cut.w || tok >= cut.y >> 16) return;
  // (what stands here after a CTA gave up may be anything)
  if (cut.z < 0 || cut.w >= shares || cut.x < 0 || cut.x + (int64_t)tok >= p.total_q || (cut.y & 0xFFFF) >= p.heads_k) return;
  // pieces: the second of the first share, the first of those behind it
  const int pieces = cut.w - cut.z + 1;
  const auto piece = [&](int i) { return (2 * (cut.z + i) + (i == 0)) * columns + column; };
  constexpr int kStep = kShared ? 4 : 1, kAtOnce = kShared ? 8 : 4;
  float4 o[kAtOnce];
  const auto load = [&](int i) {                   // (a piece that is not there: the last one, which gets no weight)
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u)
      o[u] = reinterpret_cast<const float4*>(p.part_o + (int64_t)piece(min(i + u * kStep, pieces - 1)) * kHeadDim)[lane];
  };
  int i = kShared ? warp : 0;
  load(i);
  float most = -INFINITY;
  for (int j = lane; j < pieces; j += 32) most = fmaxf(most, p.part_lse[piece(j)]);
  asm("redux.sync.max.f32 %0, %0, 0xFFFFFFFF;" : "+f"(most));
  const float ref = most == -INFINITY ? 0.f : most;
  float sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
  for (; i < pieces; i += kAtOnce * kStep) {
    float w[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) w[u] = p.part_lse[piece(min(i + u * kStep, pieces - 1))];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      // its square root, so that a small part of large values is not lost below 2^-126 (NaN: the sum is, and all that it divides)
      const float f = i + u * kStep < pieces ? ex2(0.5f * (w[u] - ref)) : 0.f;
      sum += f * f;
      acc.x += f * (f * o[u].x), acc.y += f * (f * o[u].y), acc.z += f * (f * o[u].z), acc.w += f * (f * o[u].w);
    }
    if (i + kAtOnce * kStep < pieces) load(i + kAtOnce * kStep);
  }
  if (kShared) {
    s_acc[warp][lane] = acc;
    if (lane == 0) s_sum[warp] = sum;
    __syncthreads();
    if (warp != 0) return;
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      const float4 a = s_acc[w][lane];
      sum += s_sum[w];
      acc.x += a.x, acc.y += a.y, acc.z += a.z, acc.w += a.w;
    }
  }
  const float inv = sum == 0.f ? 0.f : rcp(sum);   // (to 1 ulp; a sum is 0 or between 1 and the number of pieces)
  const int64_t row = (int64_t)(cut.x + tok) * heads + (cut.y & 0xFFFF) * kGroup + column % kGroup;
  reinterpret_cast<uint2*>(p.out + row * kHeadDim)[lane] = make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
  if (p.lse && lane == 0) p.lse[row] = sum == 0.f ? INFINITY : (most + lg2(sum)) * kLn2;
}

// ------------------------------------------------------------------------------- host --
struct Layout {
  int tokens, grid;                                // of a tile; CTAs
  bool listed;
  int64_t chunks, lse_at, o_at, tiles_at, start_at, chunk_at, first_at, bytes;
  Layout(int64_t total_q, int batch, int heads_k, int max_seqlen_q, int64_t capacity) {
    const auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
    // (CTAs that find their share themselves add up costs in 32 bits)
    listed = max_seqlen_q > kTokensPerTile || (int64_t)batch * heads_k * (capacity / kUnit + 1 + kStart) >= (1ll << 30);
    tokens = listed ? kTokensPerTile : max_seqlen_q <= 1 ? 1 : max_seqlen_q == 2 ? 2 : kTokensPerTile;
    grid = tokens <= 2 ? kB8FewGrid : kB8ChunkGrid;
    chunks = listed ? ceil_div64(total_q, kTokensPerTile) + batch : 0;
    lse_at = up(16 * grid);
    o_at = up(lse_at + 4ll * 2 * grid * kGroup * tokens);
    tiles_at = up(o_at + 4ll * 2 * grid * kGroup * tokens * kHeadDim);
    start_at = up(tiles_at + 16 * chunks * heads_k);
    chunk_at = up(start_at + 8 * (chunks * heads_k + 1));
    first_at = up(chunk_at + 4 * ((int64_t)batch + 1));
    bytes = first_at + 4 * (grid + 1);
    if (!listed) bytes = tiles_at;
  }
};

}  // namespace
}  // namespace ifv2

using namespace ifv2;

extern "C" int64_t ifv2_b8_attn_workspace_bytes(int64_t total_q, int batch, int heads_q, int head_dim, int max_seqlen_q,
                                                int64_t capacity) {
  if (total_q < 0 || batch < 0 || heads_q < 0 || head_dim != kHeadDim || capacity < 0) return 0;
  return Layout(total_q, batch, heads_q / kGroup, max_seqlen_q, capacity).bytes;
}

extern "C" int ifv2_b8_attn(const void* q, const void* k_cache, const void* v_cache, const void* k_scale, const void* v_scale,
                            void* out, float* lse, const int32_t* cu_seqlens_q, const int32_t* cache_seqlens,
                            const int32_t* block_table, int block_table_stride, const int32_t* topk_idx, int topk, const int64_t* mask,
                            int mask_words, int batch, int64_t total_q, int max_seqlen_q, int64_t num_pages, int64_t length, int code,
                            int heads_q, int heads_k, int head_dim, float softmax_scale, int causal, void* workspace,
                            int64_t workspace_bytes, int32_t* status, void* stream) {
  IFV2_REQUIRE(head_dim == kHeadDim && heads_k >= 1 && heads_q == heads_k * kGroup, IFV2_ERR_UNSUPPORTED,
               "b8_attn: head_dim must be %d, with %d query heads per KV head", kHeadDim, kGroup);
  IFV2_REQUIRE(code == kE4m3 || code == kE5m2, IFV2_ERR_INVALID_ARG, "b8_attn: code must be 0 (e4m3) or 1 (e5m2)");
  IFV2_REQUIRE(batch >= 0 && total_q >= 0 && max_seqlen_q >= 0 && num_pages >= 0 && length >= kBlockN && length % kBlockN == 0 &&
               mask_words >= 0 && topk >= 0 && topk < (1 << 30) && (block_table == nullptr || block_table_stride >= 1), IFV2_ERR_INVALID_ARG,
               "b8_attn: bad sizes");
  IFV2_REQUIRE(mask == nullptr || topk_idx == nullptr, IFV2_ERR_INVALID_ARG, "b8_attn: block lists and a mask exclude one another");
  if (total_q == 0) return IFV2_OK;
  IFV2_REQUIRE(batch >= 1 && q && out && cu_seqlens_q && cache_seqlens && workspace && status, IFV2_ERR_INVALID_ARG, "b8_attn: null pointer");
  IFV2_REQUIRE(num_pages >= 1 && (block_table || num_pages >= batch) && k_cache && v_cache && k_scale && v_scale, IFV2_ERR_INVALID_ARG,
               "b8_attn: the cache has too few pages");
  const int64_t cap = block_table ? (int64_t)block_table_stride * length : length;
  IFV2_REQUIRE(heads_k < 32768 && total_q < (1ll << 31) && cap < (1ll << 31) && num_pages * length * heads_k < (1ll << 31),
               IFV2_ERR_TOO_LARGE, "b8_attn: rows of the queries, of a sequence and of the cache must be below 2^31");
  IFV2_REQUIRE(mask == nullptr || mask_words == ceil_div64(cap, 64 * kBlockN), IFV2_ERR_INVALID_ARG,
               "b8_attn: mask rows must have a word per 64 blocks of the capacity");
  IFV2_REQUIRE((mask == nullptr && topk_idx == nullptr) || cap <= kMaxMaskWords * 64 * kBlockN, IFV2_ERR_TOO_LARGE,
               "b8_attn: blocks are selected among at most %d keys", kMaxMaskWords * 64 * kBlockN);
  const Layout at(total_q, batch, heads_k, max_seqlen_q, cap);
  IFV2_REQUIRE(at.chunks * heads_k < (1ll << 31), IFV2_ERR_TOO_LARGE, "b8_attn: too many tiles");
  IFV2_REQUIRE(workspace_bytes >= at.bytes, IFV2_ERR_INVALID_ARG, "b8_attn: the workspace is too small");
  IFV2_REQUIRE(((reinterpret_cast<uintptr_t>(workspace) | reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) == 0,
               IFV2_ERR_INVALID_ARG, "b8_attn: q, out and the workspace must begin at multiples of 16 bytes");
  CUtensorMap k_map, v_map;
  const uint64_t rows = (uint64_t)num_pages * heads_k * length;
  int rc = make_tensor_map_rows128(&k_map, k_cache, rows, kBlockN);
  if (rc == IFV2_OK) rc = make_tensor_map_rows128(&v_map, v_cache, rows, kBlockN);
  if (rc != IFV2_OK) return rc;
  AttnParams p{};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.k_scale = static_cast<const uint8_t*>(k_scale);
  p.v_scale = static_cast<const uint8_t*>(v_scale);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.lse = lse;
  p.cu_q = cu_seqlens_q;
  p.seqlens = cache_seqlens;
  p.block_table = block_table;
  p.mask = reinterpret_cast<const unsigned long long*>(mask);
  p.lists = topk_idx;
  p.bt_stride = block_table_stride;
  p.words = mask_words;
  p.topk = topk;
  p.batch = batch;
  p.heads_k = heads_k;
  p.length = (int)length;
  p.causal = causal;
  p.usual = topk_idx ? min(max(topk, 1), kMaxMaskWords * 64) : kUsualBlocks;
  p.total_q = total_q;
  p.capacity = cap;
  p.pages = (int)num_pages;                        // (below 2^31 / 64, as the cache's rows are)
  p.scale_log2 = softmax_scale * kLog2e;
  // block / n for n blocks per page: umulhi(2 block, ceil(2^(31 + shift) / n)) >> shift with 2^shift < n <= 2^(shift + 1) (or
  // n = 1, shift 0); exact while block n < 2^(31 + shift), and blocks are below 2^25
  const uint32_t n = (uint32_t)(length / kBlockN);
  while ((2u << p.page_shift) < n) ++p.page_shift;
  p.page_mul = (uint32_t)(((1ull << (31 + p.page_shift)) + n - 1) / n);
  p.least_share = 3;
  p.status = status;
  char* ws = static_cast<char*>(workspace);
  p.join = reinterpret_cast<int4*>(ws);
  p.by_tile = !at.listed && (int64_t)batch * heads_k <= at.grid;
  p.part_lse = reinterpret_cast<float*>(ws + at.lse_at);
  p.part_o = reinterpret_cast<float*>(ws + at.o_at);
  p.most_chunks = (int)at.chunks;
  p.tiles = reinterpret_cast<int4*>(ws + at.tiles_at);
  p.start = reinterpret_cast<int64_t*>(ws + at.start_at);
  p.first_chunk = reinterpret_cast<int32_t*>(ws + at.chunk_at);
  p.first_tile = reinterpret_cast<int32_t*>(ws + at.first_at);
  cudaStream_t s = (cudaStream_t)stream;
  if (at.listed) {
    const cudaError_t e = launch_beside(b8_plan_kernel, dim3(1), kPlanThreads, 0, s, p, at.grid);
    if (e != cudaSuccess) return set_error((int)e, "b8_attn (plan): %s", cudaGetErrorString(e));
    if ((rc = check_launch("b8_attn (plan)"))) return rc;
  }
  rc = at.tokens <= 2 ? b8_launch_few(k_map, v_map, p, at.tokens, code, s) : b8_launch_chunk(k_map, v_map, p, at.listed, code, s);
  if (rc) return rc;
  const unsigned cuts = p.by_tile ? batch * heads_k : at.grid;
  const bool shared = at.tokens == 1 && cuts < 64;
  const cudaError_t e = shared ? launch_beside(b8_join_kernel<true>, dim3(cuts, kGroup), kJoinThreads, 0, s, p, at.tokens, at.grid)
                                       : launch_beside(b8_join_kernel<false>, dim3(cuts, 4 * at.tokens), kJoinThreads, 0, s, p, at.tokens, at.grid);
  if (e != cudaSuccess) return set_error((int)e, "b8_attn (join): %s", cudaGetErrorString(e));
  return check_launch("b8_attn (join)");
}
