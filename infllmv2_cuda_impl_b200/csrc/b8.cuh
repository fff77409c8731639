// A key-value cache in 8 bits whose scales belong to blocks: 64 tokens of one head share one power of two.
//
// Codes are e4m3 or e5m2, the two 8-bit numbers that the tensor cores multiply as they are, so that a code is never
// converted on its way through the attention.  For a block with amax = max |x| the exponent e is the smallest integer
// >= -127 with amax 2^-e <= T (448 or 57344); code = round-to-nearest-even(x 2^-e), scale byte = e + 127 (e8m0).  Both
// types have a relative spacing, so a power of two costs nothing against amax / T, and it makes every step but
// the code's own rounding exact.  A block with an infinity or a NaN gets scale byte 255 (NaN).
#pragma once
#include "q8.cuh"

namespace ifv2 {
namespace b8 {

constexpr int kE4m3 = 0, kE5m2 = 1;
constexpr int kNanByte = q8::kNanByte;

template <int kCode>
__device__ __forceinline__ int scale_byte(uint32_t amax) {
  if (amax >= 0x7F800000u) return kNanByte;
  // amax = 1.f 2^(k - 127); T = 1.75 2^8 or 1.75 2^15
  const int k = (int)(amax >> 23), over = (amax & 0x7FFFFFu) > 0x600000u;
  return max(k - (kCode == kE4m3 ? 8 : 15) + over, 0);
}

// Four numbers times a power of two to four codes, the first in the low byte.
template <int kCode>
__device__ __forceinline__ uint32_t encode4(const float (&x)[4], float inv) {
  constexpr __nv_fp8_interpretation_t kind = kCode == kE4m3 ? __NV_E4M3 : __NV_E5M2;
  const uint64_t inv2 = tc::pack_f32x2(inv, inv);
  const uint64_t pa = q8::mul_exact2(tc::pack_f32x2(x[0], x[1]), inv2), pb = q8::mul_exact2(tc::pack_f32x2(x[2], x[3]), inv2);
  float2 a, b;
  tc::unpack_f32x2(pa, a.x, a.y);
  tc::unpack_f32x2(pb, b.x, b.y);
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(a, __NV_SATFINITE, kind), hi = __nv_cvt_float2_to_fp8x2(b, __NV_SATFINITE, kind);
  return lo | hi << 16;
}

// Four codes to numbers (without the scale); exact.
template <int kCode>
__device__ __forceinline__ void decode4(float (&x)[4], uint32_t c) {
  constexpr __nv_fp8_interpretation_t kind = kCode == kE4m3 ? __NV_E4M3 : __NV_E5M2;
  const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c & 0xFFFFu), kind);
  const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c >> 16), kind);
  const float2 fa = __half22float2(__half2(a)), fb = __half22float2(__half2(b));
  x[0] = fa.x; x[1] = fa.y; x[2] = fb.x; x[3] = fb.y;
}

}  // namespace b8
}  // namespace ifv2
