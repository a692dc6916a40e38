// The 8-bit linear layer for up to 16 tokens (formats in fp8.h): y [M][N] = Q(x) W^T (+ bias),
// W quantised, x quantised on the way. Bound by the weight's bytes and by latency: one launch,
// the weight read once.
//
// A block has 16 output features; its waves share the k-tiles. A lane loads 32 bytes of its
// feature's row and 32 elements of its token's row for each k-tile (tokens past M as zeros);
// four lanes hold a token's block of 128, so two lane swaps give the block's largest element
// and the scale. Every block quantises x again: a few hundred instructions for each 2 KB of
// weights, less than these take to arrive. The waves' sums are added in LDS in a fixed order.
#include "fp8.h"

#define FP8_TW 8  // waves a block

template <typename T, bool WIDE>
__global__ void __launch_bounds__(64 * FP8_TW)
fp8_token_kernel(const T* __restrict__ x, const unsigned char* __restrict__ w,
                 const unsigned char* __restrict__ sw, const float* __restrict__ bias,
                 T* __restrict__ y, int M, int N, int K, int KP, int SP) {
  constexpr int FP8_TU = sizeof(T) == 4 ? 2 : 4;  // k-tiles a wave has in flight
  __shared__ float4 red[FP8_TW][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int l15 = lane & 15, kg = lane >> 4;
  const int n0 = blockIdx.x * 16, nr = min(n0 + l15, N - 1);
  const unsigned char* wr = w + (long)nr * KP + kg * 32;
  const unsigned char* sr = sw + (long)nr * SP;
  const T* xr = x + (long)min(l15, M - 1) * K + kg * 32;
  const int tiles = KP / 128;
  v4f acc = (v4f){0.f, 0.f, 0.f, 0.f};
  for (int k0 = wave; k0 < tiles; k0 += FP8_TW * FP8_TU) {
    v8i fw[FP8_TU];
    int bw[FP8_TU];
    Fp8Raw<T> rx[FP8_TU][4];
#pragma unroll
    for (int u = 0; u < FP8_TU; ++u) {
      const int kt = min(k0 + u * FP8_TW, tiles - 1);
      const v4i lo = *reinterpret_cast<const v4i*>(wr + (long)kt * 128);
      const v4i hi = *reinterpret_cast<const v4i*>(wr + (long)kt * 128 + 16);
      fw[u] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      bw[u] = sr[kt];
      const int left = l15 < M ? K - (kt * 128 + kg * 32) : 0;
#pragma unroll
      for (int q = 0; q < 4; ++q) rx[u][q] = fp8_load8(xr + kt * 128 + q * 8, left - q * 8);
    }
#pragma unroll
    for (int u = 0; u < FP8_TU; ++u) {
      const int kt = k0 + u * FP8_TW;
      if (kt >= tiles) break;  // the same for the wave
      float v[4][8];
      unsigned m = 0u;
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[q][e] = rx[u][q].get(e);
          m = max(m, fp8_finite_bits(v[q][e]));
        }
      m = max(m, (unsigned)__shfl_xor((int)m, 16));
      m = max(m, (unsigned)__shfl_xor((int)m, 32));
      const int b = fp8_scale_byte(m);
      const float inv = fp8_inverse(b);
      v8i fx;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        fx[2 * q] = (int)fp8_pack4(v[q][0] * inv, v[q][1] * inv, v[q][2] * inv, v[q][3] * inv);
        fx[2 * q + 1] = (int)fp8_pack4(v[q][4] * inv, v[q][5] * inv, v[q][6] * inv, v[q][7] * inv);
      }
      if constexpr (WIDE) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              fp8_widen(fw[u][2 * q], fw[u][2 * q + 1], __uint_as_float((unsigned)bw[u] << 23)),
              fp8_widen(fx[2 * q], fx[2 * q + 1], __uint_as_float((unsigned)b << 23)), acc, 0, 0, 0);
      } else {
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fw[u], fx, acc, 0, 0, 0, bw[u], 0, b);
      }
    }
  }
  red[wave][lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
  __syncthreads();
  // lane: token l15, features n0 + 4 kg .. + 3
  if (wave == 0 && l15 < M) {
    float4 s = red[0][lane];
#pragma unroll
    for (int i = 1; i < FP8_TW; ++i) {
      const float4 p = red[i][lane];
      s.x += p.x; s.y += p.y; s.z += p.z; s.w += p.w;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int n = n0 + kg * 4 + e;
      if (n < N) st1(y + (long)l15 * N + n, f4get(s, e) + (bias ? bias[n] : 0.f));
    }
  }
}

void fp8_token(const void* x, const unsigned char* w, const unsigned char* sw, const float* bias,
               void* y, int dt, int M, int N, int K, hipStream_t st) {
  with_dt(dt, [&](auto tag) {
    using T = decltype(tag);
    hipLaunchKernelGGL((fp8_token_kernel<T, sizeof(T) == 4>), dim3((N + 15) / 16),
                       dim3(64 * FP8_TW), 0, st, (const T*)x, w, sw, bias, (T*)y, M, N, K,
                       (int)fp8_pad(K), (int)fp8_scale_pitch(K));
  });
}
