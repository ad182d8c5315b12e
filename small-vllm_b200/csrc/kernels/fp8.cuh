// Device-side pieces of the 8-bit KV cache: e4m3 codes with one power-of-two scale per row.
//
// A row x of head_dim values is held as codes c_i = e4m3(x_i * 2^-e) and the scale 2^e, where e is
// the least integer with max |x_i| <= 448 * 2^e (448 is e4m3's largest number), clamped to
// [kScaleMin, kScaleMax]. e4m3 is a floating-point type, so a power of two costs no precision
// against max / 448 (the codes keep four significant bits wherever in its binade the maximum
// lies), and it makes the scaling exact: a value is rounded once, c * 2^e is a bf16 value, and
// the scale takes one byte, e + 127, the e8m0 encoding. The clamp keeps 2^e, its inverse and the
// product of the two ends of the range inside fp32: magnitudes above 448 * 2^60 = 5.2e20 saturate,
// rows all below 2^-70 become zero. (Softmax weights times 2^e are kept inside fp32 by the attention
// itself, whose maximum is that of their products.)
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace svllm::k {

constexpr int kScaleMin = -60;
constexpr int kScaleMax = 60;
constexpr int kScaleBias = 127;

// The exponent e of a row whose largest magnitude has the given fp32 bits (finite, non-negative).
// 448 = 1.75 * 2^8, so with max = m * 2^x, m in [1, 2): e = x - 8, one more where m > 1.75.
__device__ __forceinline__ int scale_exponent(uint32_t amax_bits) {
  const int e = static_cast<int>(amax_bits >> 23) - (127 + 8) +
                ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, kScaleMin), kScaleMax);
}

// 2^e for an exponent in [-126, 127].
__device__ __forceinline__ float exp2_int(int e) {
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

// 2^(b - 127) of an e8m0 byte b in [1, 254].
__device__ __forceinline__ float scale_value(uint32_t b) { return __uint_as_float(b << 23); }

// A scale byte as it is used: the nearest of those that the writer leaves. Further out, 2^e or what is
// multiplied with it would leave fp32, and 255 is e8m0's NaN.
__device__ __forceinline__ uint32_t scale_in_range(uint32_t b) {
  return min(max(b, static_cast<uint32_t>(kScaleMin + kScaleBias)),
             static_cast<uint32_t>(kScaleMax + kScaleBias));
}

// Two values rounded to nearest even and saturated to e4m3 codes, lo in the low byte (a NaN
// becomes 0x7f).
__device__ __forceinline__ uint32_t pack_e4m3x2(float lo, float hi) {
  uint16_t d;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(hi), "f"(lo));
  return d;
}

// The codes in the low and in the high half of a word as two packed f16 values each (exact: every
// e4m3 number is an f16 number).
__device__ __forceinline__ uint32_t e4m3_to_f16x2_lo(uint32_t w) {
  uint32_t d;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}"
      : "=r"(d)
      : "r"(w));
  return d;
}

__device__ __forceinline__ uint32_t e4m3_to_f16x2_hi(uint32_t w) {
  uint32_t d;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}"
      : "=r"(d)
      : "r"(w));
  return d;
}

// Two fp32 values rounded to nearest even into one f16x2 word (lo in the low half).
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}

// d += a * b on the tensor cores: A 16x16 f16 (row), B 16x8 f16 (col), fp32 accumulators.
__device__ __forceinline__ void mma_16816_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                              uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

}  // namespace svllm::k
