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

typedef unsigned fp8_u4 __attribute__((ext_vector_type(4), aligned(2)));
// 8 neighbouring elements as loaded
template <typename T>
struct Fp8Raw {
  fp8_u4 w[sizeof(T) / 2];
  ACC_DEV float get(int u) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[u >> 2][u & 3]);
    else return u & 1 ? bfhi(w[0][u >> 1]) : bflo(w[0][u >> 1]);
  }
};
// n elements at p, zeros behind them; 16-byte loads, which the card takes at any address
template <typename T>
ACC_DEV Fp8Raw<T> fp8_load8(const T* p, int n) {
  Fp8Raw<T> r;
  if (n >= 8) {
#pragma unroll
    for (int k = 0; k < (int)sizeof(T) / 2; ++k)
      r.w[k] = *reinterpret_cast<const fp8_u4*>(p + 4 * k * (4 / sizeof(T)));
  } else {
#pragma unroll
    for (int k = 0; k < (int)sizeof(T) / 2; ++k) r.w[k] = (fp8_u4){0u, 0u, 0u, 0u};
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (u < n) {
        if constexpr (sizeof(T) == 4) r.w[u >> 2][u & 3] = __float_as_uint(p[u]);
        else r.w[0][u >> 1] |= (unsigned)p[u] << (16 * (u & 1));
      }
  }
  return r;
}

typedef int v8i __attribute__((ext_vector_type(8)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v2b __attribute__((ext_vector_type(2)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));

// 8 e4m3 bytes as bf16, times a power of two
ACC_DEV v8b fp8_widen(int lo, int hi, float scale) {
  const v2b a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)lo, scale, false);
  const v2b b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)lo, scale, true);
  const v2b c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)hi, scale, false);
  const v2b d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)hi, scale, true);
  return (v8b){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

static inline long fp8_pad(long c) { return (c + 127) / 128 * 128; }
static inline long fp8_scale_pitch(long c) { return ((c + 127) / 128 + 3) / 4 * 4; }

// internal entry points (fp8_quant.hip, fp8_gemm.hip, fp8_token.hip)
#define FP8_MAX_DIM (1L << 22)  // features: K, N
static inline int fp8_check(long M, long K, long N, int dt) {
  if (M <= 0 || K <= 0 || N <= 0 || K > FP8_MAX_DIM || N > FP8_MAX_DIM || M > (1L << 30))
    return ACC_EBADSHAPE;
  return dt == ACC_F32 || dt == ACC_BF16 ? ACC_OK : ACC_EBADARG;
}
// q, s and / or qt, st of x [R][C]; sum: column sums through ws (fp8_sum_elems fp32)
size_t fp8_sum_elems(long R, int C);
void fp8_quantize(const void* x, int dt, bool square, unsigned char* q, unsigned char* s,
                  unsigned char* qt, unsigned char* st, float* sum, float* ws, long R, int C,
                  hipStream_t str);
// c [M][N] = A B^T (+ bias); ws: fp8_gemm_elems fp32
size_t fp8_gemm_elems(long M, long N, long K);
void fp8_gemm(const unsigned char* a, const unsigned char* sa, const unsigned char* b,
              const unsigned char* sb, const float* bias, void* c, int cdt, float* ws, long M,
              long N, long K, hipStream_t st);
// up to 16 tokens: x is quantised where it is used
#define FP8_TOKENS 16
void fp8_token(const void* x, const unsigned char* w, const unsigned char* sw, const float* bias,
               void* y, int dt, int M, int N, int K, hipStream_t st);
