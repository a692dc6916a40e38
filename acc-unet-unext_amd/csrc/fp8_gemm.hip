// The 8-bit linear layer's product: C[m][n] = sum_k A[m][k] B[n][k] (+ bias[n]) over two
// quantised matrices contracted along their rows (formats in fp8.h).
//
// Two forms of the inner product:
//   bf16 outputs: v_mfma_scale_f32_16x16x128_f8f6f4 contracts one 128-block of 16 rows of
//     each side, the block scales (one exponent byte a row) applied by the instruction, so a
//     k-tile is one scale block. Measured on the card: the instruction aligns groups of 8
//     products and keeps 13 bits below the largest of a group (groups and accumulator join in
//     fp32). The loss, about 2e-5 of a random sum's size, is a hundredth of bf16's rounding.
//   fp32 outputs (WIDE): the bytes become bf16 in registers, scale included, which is exact,
//     and v_mfma_f32_16x16x32_bf16 sums in fp32 (its products were exact to 2^-23 in the same
//     measurement). Half the matrix rate; a value times its scale must stay a normal fp32.
// The first operand is B: a lane then holds 4 neighbouring n of one m and
// stores them at once. Tiles go global -> LDS by 16-byte DMA without registers; a tile row's
// eight 16-byte chunks are permuted by (row >> 1) & 7 through the source address, so 16 rows
// of one chunk, which a fragment read takes at once, cover all 64 banks. The scale dwords of
// four k-tiles ride along every fourth tile. Rows past the end read the last row; what they
// yield is not stored.
#include "fp8.h"

// Lane i copies 16 (4) bytes from its `src` to lds + 16 i (4 i), lds the same for the wave.
// From inline asm: the compiler would otherwise wait for every copy before any LDS read of
// the array. The wave waits for its copies itself, before the barrier that publishes them.
ACC_DEV unsigned fp8_lds_addr(const void* p) {
  return __builtin_amdgcn_readfirstlane(
      (unsigned)(size_t)(__attribute__((address_space(3))) const void*)p);
}
ACC_DEV void fp8_dma16(const void* src, unsigned lds) {
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\t"
               "global_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
               : "=&s"(keep) : "v"(src), "s"(lds) : "memory");
}
ACC_DEV void fp8_dma4(const void* src, unsigned lds) {
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\t"
               "global_load_lds_dword %1, off\n\ts_mov_b32 m0, %0"
               : "=&s"(keep) : "v"(src), "s"(lds) : "memory");
}

struct Fp8GemmArgs {
  const unsigned char *a, *sa, *b, *sb;
  void* c;
  const float* bias;
  float* slab;  // split: [splits][M][N] partial sums
  long M, N;
  int KP, SP, kt_per;  // k-tiles per split (a multiple of 4)
  int tiles_m, tiles_n, vec;
};

// Tile of a block. Blocks go to the 8 XCDs in turn, each with an L2 of its own: XCD x takes
// the x-th eighth of the tiles, in groups of 8 rows of tiles walked column by column, so
// that what runs together on an XCD shares its operands. false past the last tile.
ACC_DEV bool fp8_tile(const Fp8GemmArgs& g, int& mt, int& nt) {
  const int total = g.tiles_m * g.tiles_n, per = (total + 7) / 8;
  const int t = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if (t >= total || (int)(blockIdx.x >> 3) >= per) return false;
  const int group = t / (8 * g.tiles_n), rows = min(8, g.tiles_m - group * 8);
  const int in = t - group * 8 * g.tiles_n;
  mt = group * 8 + in % rows;
  nt = in / rows;
  return true;
}

template <typename T>
ACC_DEV void fp8_store4(T* p, const float (&v)[4], int n, bool vec) {
  if (vec && n >= 4) {
    stq(p, make_float4(v[0], v[1], v[2], v[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) st1(p + i, v[i]);
  }
}

// WM x WN waves, TM x TN fragments of 16 x 16 each. 128 x 128 tiles (2 x 2 waves of 4 x 4)
// read 64 KB of fragments a k-tile from LDS for 512 cycles of matrix work, which is more than
// LDS delivers beside the copies; 256 x 256 tiles (2 x 4 waves of 8 x 4) read 192 KB for
// 2048 cycles, one block a CU. Kernel traces on two cards, medians, normal data, with
// 128 x 128 and 256 x 256: 16384 x 4096 x 4096 bf16 318-325 and 288-295 us (1.9 PFLOP/s), fp32
// outputs 505-529 and 440-463 us (1.2); bf16 4096 x 4096 x 16384 254-264 and 213-234 us
// (2.3-2.6), 4096 x 8192 x 8192 255-267 and 221-238 us (2.3-2.5).
template <typename T, bool SPLIT, bool WIDE, int WM, int WN, int TM, int TN>
__global__ void __launch_bounds__(64 * WM * WN, 2)
fp8_gemm_kernel(const Fp8GemmArgs g) {
  constexpr int BM = WM * TM * 16, BN = WN * TN * 16, NW = WM * WN;
  constexpr int IA = BM / 8 / NW, IB = BN / 8 / NW;  // copies of 8 rows a wave
  static_assert(BM + BN == 64 * NW && BM % 64 == 0, "one scale dword a thread");
  __shared__ __attribute__((aligned(1024))) unsigned char sA[2][BM * 128];
  __shared__ __attribute__((aligned(1024))) unsigned char sB[2][BN * 128];
  __shared__ __attribute__((aligned(1024))) unsigned sS[2][BM + BN];
  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wm = wave % WM, wn = wave / WM;
  int mt, nt;
  if (!fp8_tile(g, mt, nt)) return;
  const long m0 = (long)mt * BM, n0 = (long)nt * BN;
  const int kt0 = SPLIT ? blockIdx.z * g.kt_per : 0;
  const int kt1 = SPLIT ? min(g.KP / 128, kt0 + g.kt_per) : g.KP / 128;

  const unsigned char *pa[IA], *pb[IB];
#pragma unroll
  for (int i = 0; i < IA; ++i) {
    const int r = (wave * IA + i) * 8 + (lane >> 3);
    pa[i] = g.a + min(m0 + r, g.M - 1) * g.KP + ((lane & 7) ^ ((r >> 1) & 7)) * 16 + (long)kt0 * 128;
  }
#pragma unroll
  for (int i = 0; i < IB; ++i) {
    const int r = (wave * IB + i) * 8 + (lane >> 3);
    pb[i] = g.b + min(n0 + r, g.N - 1) * g.KP + ((lane & 7) ^ ((r >> 1) & 7)) * 16 + (long)kt0 * 128;
  }
  const unsigned char* ps = wave < BM / 64 ? g.sa + min(m0 + t, g.M - 1) * g.SP
                                           : g.sb + min(n0 + t - BM, g.N - 1) * g.SP;
  auto stage = [&](int kt) {
    const int buf = (kt - kt0) & 1;
#pragma unroll
    for (int i = 0; i < IA; ++i) {
      fp8_dma16(pa[i], fp8_lds_addr(&sA[buf][(wave * IA + i) * 1024]));
      pa[i] += 128;
    }
#pragma unroll
    for (int i = 0; i < IB; ++i) {
      fp8_dma16(pb[i], fp8_lds_addr(&sB[buf][(wave * IB + i) * 1024]));
      pb[i] += 128;
    }
    if (((kt - kt0) & 3) == 0) fp8_dma4(ps + kt, fp8_lds_addr(&sS[((kt - kt0) >> 2) & 1][wave * 64]));
  };

  v4f acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = (v4f){0.f, 0.f, 0.f, 0.f};
  unsigned sa[TM], sb[TN];
  const int l15 = lane & 15, kg = lane >> 4;
  const int ra = wm * TM * 16 + l15, rb = wn * TN * 16 + l15;
  auto frag = [&](const unsigned char* tile, int r) {
    const int sw = (r >> 1) & 7;
    const v4i lo = *reinterpret_cast<const v4i*>(tile + r * 128 + ((2 * kg) ^ sw) * 16);
    const v4i hi = *reinterpret_cast<const v4i*>(tile + r * 128 + ((2 * kg + 1) ^ sw) * 16);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };

  if (kt0 < kt1) stage(kt0);
  for (int kt = kt0; kt < kt1; ++kt) {
    // this wave's copies have landed and its reads of the other buffer are done; behind
    // the barrier both hold for every wave
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (kt + 1 < kt1) stage(kt + 1);
    const int buf = (kt - kt0) & 1, q = (kt - kt0) & 3;
    if (q == 0) {
      const unsigned* sc = sS[((kt - kt0) >> 2) & 1];
#pragma unroll
      for (int i = 0; i < TM; ++i) sa[i] = sc[ra + i * 16];
#pragma unroll
      for (int j = 0; j < TN; ++j) sb[j] = sc[BM + rb + j * 16];
    }
    v8i fb[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) fb[j] = frag(sB[buf], rb + j * 16);
    if constexpr (WIDE) {
      v8i fa[TM];
#pragma unroll
      for (int i = 0; i < TM; ++i) fa[i] = frag(sA[buf], ra + i * 16);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v8b wb[TN];
#pragma unroll
        for (int j = 0; j < TN; ++j)
          wb[j] = fp8_widen(fb[j][2 * k], fb[j][2 * k + 1], __uint_as_float((sb[j] & 255u) << 23));
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          const v8b wa =
              fp8_widen(fa[i][2 * k], fa[i][2 * k + 1], __uint_as_float((sa[i] & 255u) << 23));
#pragma unroll
          for (int j = 0; j < TN; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb[j], wa, acc[i][j], 0, 0, 0);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const v8i fa = frag(sA[buf], ra + i * 16);
#pragma unroll
        for (int j = 0; j < TN; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
              fb[j], fa, acc[i][j], 0, 0, 0, (int)sb[j], 0, (int)sa[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) sa[i] >>= 8;
#pragma unroll
    for (int j = 0; j < TN; ++j) sb[j] >>= 8;
  }

  // lane: m = l15 of the fragment, n = 4 kg .. + 3
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const long m = m0 + ra + i * 16;
    if (m >= g.M) continue;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const long n = n0 + wn * TN * 16 + j * 16 + kg * 4;
      const int left = (int)max(0L, min(4L, g.N - n));
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = acc[i][j][e];
      if (SPLIT) {
        fp8_store4(g.slab + ((long)blockIdx.z * g.M + m) * g.N + n, v, left, g.vec);
      } else {
        if (g.bias)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (e < left) v[e] += g.bias[n + e];
        fp8_store4((T*)g.c + m * g.N + n, v, left, g.vec);
      }
    }
  }
}

// C = sum of the slabs in order (+ bias)
template <typename T>
__global__ void __launch_bounds__(256)
fp8_join_kernel(const float* __restrict__ slab, int splits, const float* __restrict__ bias,
                T* __restrict__ c, long n, long N) {
  const long e = blockIdx.x * 256L + threadIdx.x;
  if (e >= n) return;
  float v[1] = {0.f};
  ordered_strided_sum<4>(v, 0, splits, 1, [&](int k, float (&o)[1]) { o[0] = slab[k * n + e]; });
  if (bias) v[0] += bias[e % N];
  st1(c + e, v[0]);
}

// Splits of the contraction: where the output has fewer than 256 tiles (one a CU), enough
// for two a CU, each of four k-tiles (one dword of scales) at least.
static int fp8_splits(long M, long N, long K) {
  const long tiles = ((M + 127) / 128) * ((N + 127) / 128);
  const long quads = (fp8_pad(K) / 128 + 3) / 4;
  if (tiles >= 256 || quads < 2) return 1;
  long s = min((512 + tiles - 1) / tiles, quads);
  const long per = (quads + s - 1) / s;
  return (int)((quads + per - 1) / per);
}

size_t fp8_gemm_elems(long M, long N, long K) {
  const int s = fp8_splits(M, N, K);
  return s > 1 ? (size_t)s * M * N : 0;
}

void fp8_gemm(const unsigned char* a, const unsigned char* sa, const unsigned char* b,
              const unsigned char* sb, const float* bias, void* c, int cdt, float* ws, long M,
              long N, long K, hipStream_t st) {
  // 256 x 256 tiles where they alone give every CU one, 128 x 128 else
  const bool big = ((M + 255) / 256) * ((N + 255) / 256) >= 256;
  const int bt = big ? 256 : 128;
  const long tm = (M + bt - 1) / bt, tn = (N + bt - 1) / bt;
  Fp8GemmArgs g;
  g.a = a; g.sa = sa; g.b = b; g.sb = sb;
  g.c = c; g.bias = bias; g.slab = ws;
  g.M = M; g.N = N; g.KP = (int)fp8_pad(K); g.SP = (int)fp8_scale_pitch(K);
  g.tiles_m = (int)tm; g.tiles_n = (int)tn;
  const int splits = fp8_splits(M, N, K);
  const int quads = (g.KP / 128 + 3) / 4;
  g.kt_per = (quads + splits - 1) / splits * 4;
  with_dt(cdt, [&](auto tag) {
    using T = decltype(tag);
    constexpr bool WIDE = sizeof(T) == 4;
    const dim3 grid((unsigned)((tm * tn + 7) / 8 * 8), 1, splits);
    if (splits > 1) {
      g.vec = N % 4 == 0 && ((uintptr_t)ws & 15) == 0;
      hipLaunchKernelGGL((fp8_gemm_kernel<T, true, WIDE, 2, 2, 4, 4>), grid, dim3(256), 0, st, g);
      hipLaunchKernelGGL(fp8_join_kernel<T>, dim3((unsigned)((M * N + 255) / 256)), dim3(256), 0,
                         st, ws, splits, bias, (T*)c, M * N, N);
      return;
    }
    g.vec = N % 4 == 0 && ((uintptr_t)c & (4 * sizeof(T) - 1)) == 0;
    if (big)
      hipLaunchKernelGGL((fp8_gemm_kernel<T, false, WIDE, 2, 4, 8, 4>), grid, dim3(512), 0, st, g);
    else
      hipLaunchKernelGGL((fp8_gemm_kernel<T, false, WIDE, 2, 2, 4, 4>), grid, dim3(256), 0, st, g);
  });
}
