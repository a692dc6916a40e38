// 8-bit linear layer (fp8_quant.hip, fp8_gemm.hip): e4m3 values with one power-of-two scale
// for each block of 128.
//
//   scale of a block = 2^e, e the least integer with amax <= 448 * 2^e, clamped to
//     [-126, 120]; e = 0 for a block of zeros; amax over the finite elements
//   q = x * 2^-e rounded to nearest even e4m3 (448 is its largest value); a non-finite x
//     becomes NaN
// A power of two makes x * 2^-e exact, so q depends on no rounding but its own, and is what
// the matrix instruction's block scale takes (a biased exponent, one byte).
//
// A quantised matrix [R][C], contracted along C: q [R][CP], CP = C rounded up to 128 with
// zeros behind C, and scale bytes s [R][SP], byte j for columns [128 j, 128 j + 128),
// SP = CP / 128 rounded up to 4 (one dword holds 4 blocks; the padding is 127 = 2^0). Blocks
// are 1 x 128 or, for weights, 128 x 128 with the byte repeated in each of their rows, so a
// transposed weight has the same values.
#pragma once
#include "common.h"

#define FP8_ONE 127u

ACC_DEV unsigned fp8_finite_bits(float v) {
  const unsigned b = __float_as_uint(v) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}
// biased scale exponent (e + 127) from the bits of amax: amax = 1.f * 2^(E-127), 448 =
// 1.75 * 2^8, so e = E - 127 - 8, one more where the fraction exceeds .75
ACC_DEV int fp8_scale_byte(unsigned amax) {
  const int e = (int)(amax >> 23) - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
  return amax == 0u ? (int)FP8_ONE : min(max(e, 1), 247);
}
// 2^-e as a float: biased exponent 254 - byte
ACC_DEV float fp8_inverse(int byte) { return __uint_as_float((unsigned)(254 - byte) << 23); }

ACC_DEV unsigned fp8_pack4(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
  return (unsigned)r;
}

static inline long fp8_pad(long c) { return (c + 127) / 128 * 128; }
static inline long fp8_scale_pitch(long c) { return ((c + 127) / 128 + 3) / 4 * 4; }
