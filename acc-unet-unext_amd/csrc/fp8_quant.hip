// Quantisers of the 8-bit linear layer; formats in fp8.h. Bound by memory: the input is
// read once, whatever is made of it (rows, transposed rows, column sums), one byte an
// element is written for each form.
#include "fp8.h"

// Rows only: 16 threads a block of 128, 8 elements each. A thread past the scale pitch's
// last block leaves; one in the padding writes the padding.
template <typename T>
__global__ void __launch_bounds__(256)
fp8_rows_kernel(const T* __restrict__ x, unsigned char* __restrict__ q,
                unsigned char* __restrict__ s, long R, int C, int CP, int SP) {
  const int per = SP * 16;  // threads a row
  const long g = blockIdx.x * 256L + threadIdx.x;
  const long row = g / per;
  if (row >= R) return;
  const int t = (int)(g - row * per);
  const int c = t * 8;
  const Fp8Raw<T> raw = fp8_load8(x + row * C + c, C - c);
  float v[8];
  unsigned m = 0u;
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    v[u] = raw.get(u);
    m = max(m, fp8_finite_bits(v[u]));
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, o));
  const int e = fp8_scale_byte(m);
  const float inv = fp8_inverse(e);
  if (c < CP) {
    uint2 w;
    w.x = fp8_pack4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
    w.y = fp8_pack4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
    *reinterpret_cast<uint2*>(q + row * CP + c) = w;
  }
  if ((t & 15) == 0) s[row * SP + (t >> 4)] = (unsigned char)e;
}

// A 128 x 128 tile: thread t holds columns 8 (t % 16) .. + 7 of rows 8 (t / 16) .. + 7.
//   q, s     blocks 1 x 128 along the rows          (square: the tile is one block)
//   qt, st   the transposed matrix [C][RP], blocks 1 x 128 along the rows of x
//   sum      [tiles of rows][C] column sums
// The transposed bytes go through LDS: [column][row], the 8 rows of a column as two dwords; a
// column's 128 bytes are padded to 132, which spreads a wave's dwords evenly over the banks.
#define FP8_TP 132
template <typename T>
__global__ void __launch_bounds__(256)
fp8_tile_kernel(const T* __restrict__ x, unsigned char* __restrict__ q,
                unsigned char* __restrict__ s, unsigned char* __restrict__ qt,
                unsigned char* __restrict__ st, float* __restrict__ sum, long R, int C, int CP,
                int SP, long RP, int SPT, int square) {
  __shared__ __attribute__((aligned(16))) unsigned char tile[128 * FP8_TP];
  __shared__ unsigned cmax[16][128];
  __shared__ unsigned wmax[4];
  __shared__ unsigned char cb[128];
  float (*csum)[128] = reinterpret_cast<float (*)[128]>(tile);
  const int t = threadIdx.x, cg = t & 15, rg = t >> 4;
  const long r0 = (long)blockIdx.x * 128;
  const int c0 = blockIdx.y * 128, c = c0 + cg * 8;
  // kept as loaded: 32 registers for bf16, and twice the blocks a CU
  Fp8Raw<T> raw[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const long r = r0 + rg * 8 + i;
    raw[i] = fp8_load8(x + r * C + c, r < R ? C - c : 0);
  }
  int e[8];
  unsigned all = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    unsigned m = 0u;
#pragma unroll
    for (int u = 0; u < 8; ++u) m = max(m, fp8_finite_bits(raw[i].get(u)));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, o));
    e[i] = fp8_scale_byte(m);
    all = max(all, m);
  }
  if (square) {
    all = max(all, (unsigned)__shfl_xor((int)all, 16));
    all = max(all, (unsigned)__shfl_xor((int)all, 32));
    if ((t & 63) == 0) wmax[t >> 6] = all;
    __syncthreads();
    const int eb = fp8_scale_byte(max(max(wmax[0], wmax[1]), max(wmax[2], wmax[3])));
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = eb;
  }
  if (q) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const long r = r0 + rg * 8 + i;
      if (r >= R) continue;
      const float inv = fp8_inverse(e[i]);
      uint2 w;
      w.x = fp8_pack4(raw[i].get(0) * inv, raw[i].get(1) * inv, raw[i].get(2) * inv, raw[i].get(3) * inv);
      w.y = fp8_pack4(raw[i].get(4) * inv, raw[i].get(5) * inv, raw[i].get(6) * inv, raw[i].get(7) * inv);
      *reinterpret_cast<uint2*>(q + r * CP + c) = w;
      if (cg == 0) s[r * SP + blockIdx.y] = (unsigned char)e[i];
      // the scale row's padding, written once
      if (cg == 0 && (int)blockIdx.y == CP / 128 - 1)
        for (int b = CP / 128; b < SP; ++b) s[r * SP + b] = (unsigned char)FP8_ONE;
    }
  }
  if (qt) {
    float inv[8];
    if (square) {
      const float iv = fp8_inverse(e[0]);
#pragma unroll
      for (int u = 0; u < 8; ++u) inv[u] = iv;
      if (t < 128) cb[t] = (unsigned char)e[0];
    } else {
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        unsigned m = 0u;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, fp8_finite_bits(raw[i].get(u)));
        cmax[rg][cg * 8 + u] = m;
      }
      __syncthreads();
      if (t < 128) {
        unsigned m = 0u;
#pragma unroll
        for (int k = 0; k < 16; ++k) m = max(m, cmax[k][t]);
        cb[t] = (unsigned char)fp8_scale_byte(m);
      }
      __syncthreads();
#pragma unroll
      for (int u = 0; u < 8; ++u) inv[u] = fp8_inverse(cb[cg * 8 + u]);
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const float iv = inv[u];
      unsigned* dst = reinterpret_cast<unsigned*>(tile + (cg * 8 + u) * FP8_TP + rg * 8);
      dst[0] = fp8_pack4(raw[0].get(u) * iv, raw[1].get(u) * iv, raw[2].get(u) * iv, raw[3].get(u) * iv);
      dst[1] = fp8_pack4(raw[4].get(u) * iv, raw[5].get(u) * iv, raw[6].get(u) * iv, raw[7].get(u) * iv);
    }
    __syncthreads();
    // 8 threads a column, 16 bytes each
    for (int k = t; k < 128 * 8; k += 256) {
      const int cc = k >> 3, b = (k & 7) * 16;
      if (c0 + cc >= C) continue;
      const unsigned* src = reinterpret_cast<const unsigned*>(tile + cc * FP8_TP + b);
      *reinterpret_cast<uint4*>(qt + (long)(c0 + cc) * RP + r0 + b) =
          make_uint4(src[0], src[1], src[2], src[3]);
    }
    if (t < 128 && c0 + t < C) {
      unsigned char* so = st + (long)(c0 + t) * SPT;
      so[blockIdx.x] = cb[t];
      if ((long)blockIdx.x == RP / 128 - 1)
        for (int b = (int)(RP / 128); b < SPT; ++b) so[b] = (unsigned char)FP8_ONE;
    }
  }
  if (sum) {
    __syncthreads();  // tile is read above
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      float a = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) a += raw[i].get(u);
      csum[rg][cg * 8 + u] = a;
    }
    __syncthreads();
    if (t < 128 && c0 + t < C) {
      float a = 0.f;
#pragma unroll
      for (int k = 0; k < 16; ++k) a += csum[k][t];
      sum[(long)blockIdx.x * C + c0 + t] = a;
    }
  }
}

// out[c] = sum over n rows of part [n][C] in order
__global__ void __launch_bounds__(256)
fp8_colsum_kernel(const float* __restrict__ part, long n, int C, float* __restrict__ out) {
  __shared__ double red[4][64];
  const int cl = threadIdx.x & 63, g = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + cl;
  double v[1] = {0.0};
  if (c < C)
    ordered_strided_sum<4>(v, g, (int)n, 4, [&](int r, double (&o)[1]) { o[0] = part[(long)r * C + c]; });
  red[g][cl] = v[0];
  __syncthreads();
  if (g == 0 && c < C) out[c] = (float)(((red[0][cl] + red[1][cl]) + red[2][cl]) + red[3][cl]);
}

size_t fp8_sum_elems(long R, int C) { return (size_t)((R + 127) / 128) * C; }

void fp8_quantize(const void* x, int dt, bool square, unsigned char* q, unsigned char* s,
                  unsigned char* qt, unsigned char* st, float* sum, float* ws, long R, int C,
                  hipStream_t str) {
  const int CP = (int)fp8_pad(C), SP = (int)fp8_scale_pitch(C);
  const long RP = fp8_pad(R);
  const int SPT = (int)fp8_scale_pitch(R);
  with_dt(dt, [&](auto tag) {
    using T = decltype(tag);
    if (!square && !qt && !sum) {
      // a launch holds fewer than 2^32 threads
      const long most = (1L << 31) / (SP * 16);
      for (long r = 0; r < R; r += most) {
        const long rows = min(most, R - r);
        hipLaunchKernelGGL(fp8_rows_kernel<T>, dim3((unsigned)((rows * SP * 16 + 255) / 256)),
                           dim3(256), 0, str, (const T*)x + r * C, q + r * CP, s + r * SP, rows, C,
                           CP, SP);
      }
      return;
    }
    hipLaunchKernelGGL(fp8_tile_kernel<T>, dim3((unsigned)(RP / 128), CP / 128), dim3(256), 0, str,
                       (const T*)x, q, s, qt, st, sum ? ws : nullptr, R, C, CP, SP, RP, SPT,
                       square ? 1 : 0);
    if (sum)
      hipLaunchKernelGGL(fp8_colsum_kernel, dim3(ceil_div(C, 64)), dim3(256), 0, str, ws, RP / 128,
                         C, sum);
  });
}

extern "C" int accunet_fp8_quantize(const void* x, int square, void* q, void* s, void* qt, void* st,
                                    long R, int C, int dt, void* stream) {
  const int rc = fp8_check(R, C, 1, dt);
  if (rc != ACC_OK) return rc;
  if (!x || !q || !s || (qt != nullptr) != (st != nullptr)) return ACC_EBADARG;
  fp8_quantize(x, dt, square != 0, (unsigned char*)q, (unsigned char*)s, (unsigned char*)qt,
               (unsigned char*)st, nullptr, nullptr, R, C, (hipStream_t)stream);
  return hipGetLastError() == hipSuccess ? ACC_OK : ACC_ELAUNCH;
}
