// Look-up of the blocks that a mask row of a decode step selects.
#pragma once
#include "common.cuh"

namespace ifv2 {

// The selected blocks of one (sequence, KV head), lowest first, looked up by a whole warp that takes
// every kStride-th of them: lane l fetches mask word 32 c + l of a chunk of words, a warp scan gives
// the selected blocks before it, and lane i of the warp finds the i-th next block of the warp by two
// short bisections, so that 32 look-ups cost one trip to memory.  (One thread walking the words paid a
// chain of a load per word, 33 of them at 131072 tokens, for the count and again for every block.)
// Every lane must make the calls and gets the same answers.
// kWritten: the words may be written while the kernel lives already, by one beside which it starts and for which it
// waits before the first call; a read-only load (__ldg) is not for them, and may be moved in front of the wait.
template <int kStride, bool kWritten = false>
struct BlockList {
  const unsigned long long* words;   // null = every block below nblk
  int nwords, nblk;
  int cached;                        // lane i: block of look-up 32 n + i
  __device__ unsigned long long word(int w) const {
    if (w >= nwords) return 0ull;
    unsigned long long x = kWritten ? words[w] : __ldg(words + w);
    const int first = w * 64;
    if (nblk - first < 64) x &= (nblk > first) ? ((1ull << (nblk - first)) - 1ull) : 0ull;
    return x;
  }
  __device__ int count(int lane) const {
    if (words == nullptr) return nblk;
    int n = 0;
    for (int w = lane; w < nwords; w += 32) n += __popcll(word(w));
    return __reduce_add_sync(0xFFFFFFFFu, n);
  }
  // blocks number j, j + kStride, ... (0-based), one per lane; -1 past the end of the mask
  __device__ void refill(int j, int lane) {
    const int target = j + lane * kStride;
    cached = -1;
    int before = 0;
    for (int c = 0; c * 32 < nwords && before <= j + 31 * kStride; ++c) {
      const unsigned long long mine = word(c * 32 + lane);
      const int cnt = __popcll(mine);
      int incl = cnt;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int up = __shfl_up_sync(0xFFFFFFFFu, incl, d);
        if (lane >= d) incl += up;
      }
      const int excl = incl - cnt, total = __shfl_sync(0xFFFFFFFFu, incl, 31);
      const bool here = target >= before && target < before + total;
      const int r = here ? target - before : 0;
      int src = 0;                               // last word that starts at or below block r
#pragma unroll
      for (int d = 16; d >= 1; d >>= 1)
        if (__shfl_sync(0xFFFFFFFFu, excl, src + d) <= r) src += d;
      unsigned long long x = __shfl_sync(0xFFFFFFFFu, mine, src);
      int rank = r - __shfl_sync(0xFFFFFFFFu, excl, src), pos = 0;
#pragma unroll
      for (int d = 32; d >= 1; d >>= 1) {        // position of the set bit with `rank` set bits below it
        const int low = __popcll(x & ((1ull << d) - 1ull));
        if (rank >= low) { rank -= low; pos += d; x >>= d; }
      }
      if (here) cached = (c * 32 + src) * 64 + pos;
      before += total;
    }
  }
  // the warp's look-up number i, of block j = first + i * kStride; look-ups come in order
  __device__ int nth(int i, int j, int lane) {
    if (words == nullptr) return j;
    if ((i & 31) == 0) refill(j, lane);
    return __shfl_sync(0xFFFFFFFFu, cached, i & 31);
  }
};

}  // namespace ifv2
