// Rotary positions over several axes: what the kernels that rotate rows share.
//
// Pair i of R/2 turns by the angle that the tables hold for position pos[axis(i)]:
//   y0 = x0 c - x1 s,  y1 = x0 s + x1 c,   c = cos[pos[axis(i)]][i], s = sin[...][i]
// Pairs are neighbours (2i, 2i + 1) or halves (i, i + R/2); features from R on pass through.  The products are
// rounded one by one (no fused multiply-add), so a row comes out the same here, in the decode step and from fp32
// tensor arithmetic.  Positions outside the tables take their first or last row.
#pragma once
#include "common.cuh"

namespace ifv2 {

constexpr int kMaxAxes = 4;

struct RotaryParams {
  const float* cos_t;            // (rows, dim / 2)
  const float* sin_t;
  const int32_t* positions;      // (axes, n), or (n) positions that all axes share (stride 0)
  int64_t axis_stride;
  int dim, rows, interleaved;
  uint32_t axis_map[4];          // two bits for each of up to 64 pairs
  __device__ __forceinline__ int axis(int pair) const { return (axis_map[pair >> 4] >> (2 * (pair & 15))) & 3; }
  __device__ __forceinline__ int64_t table_row(int64_t t, int pair) const {
    return min(max(__ldg(positions + axis(pair) * axis_stride + t), 0), rows - 1);
  }
};

__device__ __forceinline__ void rotate2(float& x0, float& x1, float c, float s) {
  const float y0 = __fsub_rn(__fmul_rn(x0, c), __fmul_rn(x1, s));
  x1 = __fadd_rn(__fmul_rn(x0, s), __fmul_rn(x1, c));
  x0 = y0;
}

// Checks the arguments every rotating entry shares and fills `r` (host).  pair_axis: HOST array of dim / 2 axis
// numbers, or null = axis 0.
int make_rotary(RotaryParams* r, const char* what, const float* cos_t, const float* sin_t, const int32_t* positions,
                int64_t axis_stride, const uint8_t* pair_axis, int axes, int dim, int64_t rows, int interleaved);

}  // namespace ifv2
