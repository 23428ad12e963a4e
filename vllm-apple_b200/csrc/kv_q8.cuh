// e4m3 rows with one power-of-two scale: device helpers of the 8-bit KV cache.
//
// A row is the head_size values of one token and one kv head.  With a = the largest
// finite |x| of the row, its exponent is e = ceil(log2(a / 448)) clamped to [-14, 7]
// (-14 for a row of zeros): the smallest e in that range with a <= 448 * 2^e.  The row
// is stored as the e4m3 codes of x * 2^-e and one byte e + 127.
//
// Why a power of two: x * 2^-e is exact in fp32, so the code is x rounded ONCE, to the
// nearest e4m3 (half a step, 2^-4 relative).  Why that range: a code is a multiple of
// 2^-9 up to 448, so code * 2^e is a multiple of 2^-23 up to 57344, an fp16 value for
// every e -- reading back is exact, and the attention kernels feed the tensor cores
// code * 2^e in fp16 without a second rounding.  Values past 57344 (and infinities)
// saturate; NaN stays NaN.
#pragma once

#include "common.cuh"

namespace va {

constexpr int kQ8ExpBias = 127;

// Largest |x| of a packed fp16 pair, as fp16 bits per half, folded into `m` (magnitudes of
// one sign order like their bits; infinities and NaN come out at 0x7c00 and above) ...
VA_DEVINL uint32_t q8_absmax2(uint32_t m, uint32_t w) { return __vmaxu2(m, w & 0x7fff7fffu); }
// ... and of the finite ones alone, for the rare row that holds others.
VA_DEVINL uint32_t q8_absmax2_finite(uint32_t m, uint32_t w) {
  const uint32_t a = w & 0x7fff7fffu;
  return __vmaxu2(m, a & __vcmpltu2(a, 0x7c007c00u));
}

// Exponent of a row whose largest finite magnitude has the fp16 bits `amax`.
VA_DEVINL int q8_exponent(uint32_t amax) {
  const uint32_t b = __float_as_uint(__half2float(__ushort_as_half((unsigned short)amax)));
  // a = f * 2^E, 1 <= f < 2; 448 = 1.75 * 2^8
  const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, -14), 7);
}

// fp16 bits of 2^e, from the stored byte e + 127 (e in [-14, 7]), in both halves.
VA_DEVINL uint32_t q8_scale_h2(uint32_t byte) { return ((byte - 112u) << 10 & 0xffffu) * 0x10001u; }

// fp16 bits of 2^-e, in both halves.
VA_DEVINL uint32_t q8_inv_h2(int e) { return (uint32_t)(15 - e) << 10 | (uint32_t)(15 - e) << 26; }

// Four fp16 values times inv (2^-e from q8_inv_h2), as four e4m3 codes.  The product in
// fp16 is exact wherever it matters: it is at most 512, and what falls below fp16's normal
// range (2^-14) is below half the smallest code (2^-10) in any case.
VA_DEVINL uint32_t q8_encode4(uint32_t a, uint32_t b, uint32_t inv) {
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\t.reg .b32 x, y;\n\t"
      "mul.rn.f16x2 x, %1, %3;\n\t"
      "mul.rn.f16x2 y, %2, %3;\n\t"
      "cvt.rn.satfinite.e4m3x2.f16x2 l, x;\n\t"
      "cvt.rn.satfinite.e4m3x2.f16x2 h, y;\n\t"
      "mov.b32 %0, {l, h};\n\t}"
      : "=r"(r)
      : "r"(a), "r"(b), "r"(inv));
  return r;
}

// Four e4m3 codes as two fp16 pairs.
VA_DEVINL void q8_decode4(uint32_t c, uint32_t &lo, uint32_t &hi) {
  asm("{\n\t.reg .b16 l, h;\n\t"
      "mov.b32 {l, h}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, l;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(c));
}

VA_DEVINL uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

}  // namespace va
