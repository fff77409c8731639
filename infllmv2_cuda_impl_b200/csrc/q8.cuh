// Rows of a key-value cache in 8 bits: 128 codes (e4m3 or int8) and one power-of-two scale.
//
// For a row x with amax = max |x| the exponent e is the smallest integer >= -127 with amax 2^-e <= T, where T is
// the type's largest code (448 or 127); code = round-to-nearest-even(x 2^-e), scale byte = e + 127 (e8m0).  With a
// power of two the product is exact and so is code 2^e on the way back: a value is rounded once, its place in the
// code alone decides how, and what is read back is a bf16 number that no further rounding touches.  For e4m3,
// whose spacing is relative, the power of two costs nothing against amax / 448; int8 loses up to one bit.
// A row that holds an infinity or a NaN gets scale byte 255 (NaN) and codes 0: it reads back as NaN.
#pragma once
#include <cuda_fp8.h>
#include "common.cuh"
#include "tc05.cuh"

namespace ifv2 {
namespace q8 {

constexpr int kE4m3 = 0, kInt8 = 1;
constexpr int kNanByte = 255;

// A product that keeps subnormal inputs and results (the build flushes them otherwise): a row whose largest
// value is below 2^-118 has scale 2^-127 and elements that are subnormal numbers.
__device__ __forceinline__ float mul_exact(float a, float b) {
  float r;
  asm("mul.rn.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ uint64_t mul_exact2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ uint64_t fma_exact2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// Scale byte of a row whose largest |x| has the bit pattern `amax`.
template <int kCode>
__device__ __forceinline__ int scale_byte(uint32_t amax) {
  if (amax >= 0x7F800000u) return kNanByte;
  // amax = 1.f 2^(k - 127); 448 = 1.75 2^8, 127 = 1.984375 2^6
  const int k = (int)(amax >> 23), over = (amax & 0x7FFFFFu) > (kCode == kE4m3 ? 0x600000u : 0x7E0000u);
  return max(k - (kCode == kE4m3 ? 8 : 6) + over, 0);
}
// 2^-e; a NaN row is multiplied by 0 ... its codes are set to 0 by encode4.
__device__ __forceinline__ float inverse_scale(int byte) { return __uint_as_float((uint32_t)(254 - min(byte, 253)) << 23); }
// 2^e, or NaN
__device__ __forceinline__ float scale_value(int byte) {
  return __uint_as_float(byte == kNanByte ? 0x7FC00000u : byte == 0 ? 0x00400000u : (uint32_t)byte << 23);
}

// Four values (times 2^-e) to four codes, the first in the low byte.
template <int kCode>
__device__ __forceinline__ uint32_t encode4(const float (&x)[4], int byte) {
  if (byte == kNanByte) return 0u;
  const float inv = inverse_scale(byte);
  const uint64_t inv2 = tc::pack_f32x2(inv, inv);
  float2 a, b;
  if (kCode == kE4m3) {
    const uint64_t pa = mul_exact2(tc::pack_f32x2(x[0], x[1]), inv2), pb = mul_exact2(tc::pack_f32x2(x[2], x[3]), inv2);
    tc::unpack_f32x2(pa, a.x, a.y);
    tc::unpack_f32x2(pb, b.x, b.y);
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(a, __NV_SATFINITE, __NV_E4M3), hi = __nv_cvt_float2_to_fp8x2(b, __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
  }
  // 1.5 2^23 + y has steps of 1, so that the sum is rounded to the integer, whose low byte is the number's
  const uint64_t one = tc::pack_f32x2(0x1.8p23f, 0x1.8p23f);
  const uint64_t pa = fma_exact2(tc::pack_f32x2(x[0], x[1]), inv2, one), pb = fma_exact2(tc::pack_f32x2(x[2], x[3]), inv2, one);
  const uint32_t lo = __byte_perm((uint32_t)pa, (uint32_t)(pa >> 32), 0x0040), hi = __byte_perm((uint32_t)pb, (uint32_t)(pb >> 32), 0x0040);
  return __byte_perm(lo, hi, 0x5410);
}

// Four codes to numbers (without the scale); exact.
template <int kCode>
__device__ __forceinline__ void decode4(float (&x)[4], uint32_t c) {
  if (kCode == kE4m3) {
    const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c & 0xFFFFu), __NV_E4M3);
    const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c >> 16), __NV_E4M3);
    const float2 fa = __half22float2(__half2(a)), fb = __half22float2(__half2(b));
    x[0] = fa.x; x[1] = fa.y; x[2] = fb.x; x[3] = fb.y;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(c >> (8 * i));
  }
}

// Four codes as two fp16 pairs, codes (0, 1) and (2, 3); exact.  Integers go through 1024 + (code + 128), whose
// fp16 numbers are 0x6400 + (code + 128).
template <int kCode>
__device__ __forceinline__ void decode_h2(uint32_t& lo, uint32_t& hi, uint32_t c, uint32_t lo_bytes = 0x4140, uint32_t hi_bytes = 0x4342) {
  if (kCode == kE4m3) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi) : "r"(c));
  } else {
    c ^= 0x80808080u;
    const uint32_t a = __byte_perm(c, 0x64646464u, lo_bytes), b = __byte_perm(c, 0x64646464u, hi_bytes);
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(a), "r"(0x64806480u));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(b), "r"(0x64806480u));
  }
}
// The same for codes (0, 2) and (1, 3): a transposed 16-bit load holds two tokens' codes of two features.
template <int kCode>
__device__ __forceinline__ void decode_h2_even_odd(uint32_t& even, uint32_t& odd, uint32_t c) {
  if (kCode == kE4m3) decode_h2<kCode>(even, odd, __byte_perm(c, 0u, 0x3120));
  else decode_h2<kCode>(even, odd, c, 0x4240, 0x4341);
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

// A row of 128 values, four per lane, quantised by one warp.
template <int kCode>
__device__ __forceinline__ void store_row(const float (&x)[4], uint8_t* codes, uint8_t* scale, int lane) {
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) amax = max(amax, abs_bits(x[i]));
  amax = __reduce_max_sync(0xFFFFFFFFu, amax);
  const int byte = scale_byte<kCode>(amax);
  reinterpret_cast<uint32_t*>(codes)[lane] = encode4<kCode>(x, byte);
  if (lane == 0) *scale = (uint8_t)byte;
}

// Where position `pos` of sequence b lives: row ((slot * heads + h) * length + off) of the (rows, 128) codes and of
// the (rows) scales.  A slot is a sequence (or the one that batch_idx names) or a page of the block table.
struct Place {
  const int32_t* block_table;    // (batch, bt_stride) or null
  const int32_t* batch_idx;      // (batch) or null
  int bt_stride, heads, length, slots;
  // row of head 0, or -1 where there is no such row: a page or a slot that the cache does not have, a position
  // past the table or below 0
  __device__ __forceinline__ int64_t row0(int b, int64_t pos) const {
    int slot, off;
    if (pos < 0) return -1;
    if (block_table != nullptr) {
      if (pos >= (int64_t)bt_stride * length) return -1;
      const uint32_t page = (uint32_t)pos / (uint32_t)length;      // (the host keeps positions below 2^31)
      slot = __ldg(block_table + (int64_t)b * bt_stride + page);
      off = (int)((uint32_t)pos - page * (uint32_t)length);
    } else {
      if (pos >= length) return -1;
      slot = batch_idx ? __ldg(batch_idx + b) : b;
      off = (int)pos;
    }
    if (slot < 0 || slot >= slots) return -1;
    return (int64_t)slot * heads * length + off;
  }
  __device__ __forceinline__ int64_t row(int64_t row0, int h) const { return row0 + (int64_t)h * length; }
};

}  // namespace q8
}  // namespace ifv2
