// The norms around a residual block (blocknorm_fwd.hip, blocknorm_bwd.hip).
//
//   u = norm(f) * w1 + b1          the norm after the block
//   r = x + s * g * u              residual scale s [C], gate g (none, per sample, per element)
//   h = norm(r) * w2 + b2          the norm before the next block
//
// norm(v) = (v - mean(v)) / sqrt(var(v) + eps) ("layer") or v / sqrt(mean(v^2) + eps)
// ("rms"), over the C channels of a row. Rows are tokens [P][C]; sample b owns rows
// [b*L, (b+1)*L). Without f only h = norm(x) * w2 + b2 is computed.
//
// Layout shared by both directions: a row lives in the registers of 64*WPR threads, 8
// elements a thread (ITER groups of 16 bytes, group i at column (i*64*WPR + t)*VEC), so
// every tensor is read once and every statistic is a two-pass sum over registers. WPR = 1
// runs four rows in a 256-thread block (C <= 512, no barrier), longer rows take one block of
// 64*WPR threads. The next row's 16-byte groups are loaded, in their raw form, before this
// row's sums. Rows that are not whole, aligned groups are loaded 16 bytes at a time all
// the same, which the card takes at any address, and end in a partial group that is read
// and written element by element.
#pragma once
#include <type_traits>

#include "common.h"

#define BN_MAX_C 8192
#define BN_GATE_NONE 0
#define BN_GATE_SAMPLE 1
#define BN_GATE_ELEMENT 2

struct BlockNormArgs {
  const void *x, *f, *g, *dr, *dh;
  const float *w1, *b1, *s, *w2, *b2;
  void *r, *h, *dx, *df, *dg;
  float* stats;  // [P][4]: mean1, rstd1, mean2, rstd2
  float* part;   // backward: [blocks][4][C] partial sums
  float* gpart;  // backward, gate per sample split over blocks: [B*S][C]
  long P, L;     // rows, rows per sample
  int C, gmode, layer;
  float eps;
  FastDiv fL;    // forward: by L
  int G, S;      // backward: samples per block (S == 1) / blocks per sample (G == 1)
};

typedef unsigned bn_u4 __attribute__((ext_vector_type(4), aligned(2)));

// 16 bytes of a row as loaded
template <typename T>
struct BnGroup {
  static constexpr int N = 16 / sizeof(T);
  bn_u4 w;
  // element u as fp32
  ACC_DEV float get(int u) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[u]);
    else return u & 1 ? bfhi(w[u >> 1]) : bflo(w[u >> 1]);
  }
};
// How rows lie: at any address, ending in a partial group; in whole, aligned groups; the
// same with outputs stored past the caches (too large for the next kernel to find there).
enum { BN_ANY = 0, BN_FULL = 1, BN_STREAM = 2 };
// n elements at p (the rest zero); but for BN_ANY n is 0 or the whole, aligned group
template <typename T, int FORM>
ACC_DEV BnGroup<T> bn_load(const T* p, int n) {
  constexpr int N = BnGroup<T>::N;
  BnGroup<T> g;
  g.w = (bn_u4){0u, 0u, 0u, 0u};
  if (FORM != BN_ANY) {
    if (n > 0) {
      const uint4 q = *reinterpret_cast<const uint4*>(p);
      g.w = (bn_u4){q.x, q.y, q.z, q.w};
    }
  } else if (n >= N) {
    g.w = *reinterpret_cast<const bn_u4*>(p);
  } else {
#pragma unroll
    for (int u = 0; u < N; ++u)
      if (u < n) {
        if constexpr (sizeof(T) == 4) g.w[u] = __float_as_uint(p[u]);
        else g.w[u >> 1] |= (unsigned)p[u] << (16 * (u & 1));
      }
  }
  return g;
}
template <typename T, int FORM>
ACC_DEV void bn_store(T* p, int n, const float* v) {
  constexpr int N = BnGroup<T>::N;
  bn_u4 w;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (sizeof(T) == 4) w[k] = __float_as_uint(v[k]);
    else w[k] = pack_bf2(v[2 * k], v[2 * k + 1]);
  }
  if (FORM != BN_ANY) {
    const acc_u32x4 q = {w[0], w[1], w[2], w[3]};
    if (n > 0) {
      if (FORM == BN_STREAM) __builtin_nontemporal_store(q, reinterpret_cast<acc_u32x4*>(p));
      else *reinterpret_cast<acc_u32x4*>(p) = q;
    }
  } else if (n >= N) {
    *reinterpret_cast<bn_u4*>(p) = w;
  } else {
#pragma unroll
    for (int u = 0; u < N; ++u)
      if (u < n) st1(p + u, v[u]);
  }
}

// NV fp32 values at p (a parameter's, or a row of sums) where n of them are in the row, else
// and for a null p the fill
template <int NV>
ACC_DEV void bn_params(const float* p, int n, float fill, float* v) {
#pragma unroll
  for (int u = 0; u < NV; ++u) v[u] = fill;
  if (!p) return;
  if (n >= NV) {
#pragma unroll
    for (int q = 0; q < NV; q += 4) {
      const bn_u4 w = *reinterpret_cast<const bn_u4*>(p + q);
#pragma unroll
      for (int u = 0; u < 4; ++u) v[q + u] = __uint_as_float(w[u]);
    }
  } else {
#pragma unroll
    for (int u = 0; u < NV; ++u)
      if (u < n) v[u] = p[u];
  }
}
template <int NV>
ACC_DEV void bn_put(float* p, int n, const float* v) {
#pragma unroll
  for (int q = 0; q < NV; q += 4) bn_store<float, BN_ANY>(p + q, n - q, v + q);
}

// Sum over the wave in one fixed order, the same value in every lane: neighbours, pairs,
// half rows and rows of 16 by DPP moves inside the ALU, then across the rows.
template <int CTRL, int ROWS>
ACC_DEV float bn_dpp(float v) {
  return __int_as_float(
      __builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, ROWS, 15, ROWS == 15 ? false : true));
}
ACC_DEV float bn_wave_sum(float v) {
  v += bn_dpp<0xB1, 15>(v);   // lanes 1 0 3 2
  v += bn_dpp<0x4E, 15>(v);   // lanes 2 3 0 1
  v += bn_dpp<0x141, 15>(v);  // mirrored halves of a row
  v += bn_dpp<0x140, 15>(v);  // mirrored rows: each lane has its row's sum
  v += bn_dpp<0x142, 10>(v);  // rows 1, 3 take rows 0, 2
  v += bn_dpp<0x143, 12>(v);  // row 3 takes rows 0 + 1
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// Sums over the 64*WPR threads of a row, in one fixed order. Consecutive calls use the two
// halves of `red` in turn: a wave that writes a half has passed the barrier of the call
// before, which every wave reaches only after it has read that half.
template <int WPR, int NV>
ACC_DEV void bn_row_sum(float (&v)[NV], float (*red)[2][16], int& turn) {
#pragma unroll
  for (int k = 0; k < NV; ++k) v[k] = bn_wave_sum(v[k]);
  if constexpr (WPR > 1) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int h = turn & 1;
    ++turn;
    if (lane == 0)
#pragma unroll
      for (int k = 0; k < NV; ++k) red[h][k][wave] = v[k];
    // the raw barrier: global loads in flight (the next row's) stay in flight
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < WPR; ++w) t += red[h][k][w];
      v[k] = t;
    }
  }
}

// Run f(BnShape) for a row of C elements of T.
template <int I, int W, int F>
struct BnShape {
  static constexpr int ITER = I, WPR = W, FORM = F;
};
template <typename T, typename F>
static inline void bn_with_shape(long P, int C, bool aligned, F f) {
  constexpr int I = sizeof(T) == 4 ? 2 : 1;
  auto go = [&](auto ftag) {
    constexpr int FORM = decltype(ftag)::value;
    if (I > 1 && C <= 256) f(BnShape<1, 1, FORM>{});
    else if (C <= 512) f(BnShape<I, 1, FORM>{});
    else if (C <= 1024) f(BnShape<I, 2, FORM>{});
    else if (C <= 2048) f(BnShape<I, 4, FORM>{});
    else if (C <= 4096) f(BnShape<I, 8, FORM>{});
    else f(BnShape<I, 16, FORM>{});
  };
  // outputs of 64 MB and more are streamed (the last-level cache holds 256 MB)
  if (!aligned || C % (16 / (int)sizeof(T))) go(std::integral_constant<int, BN_ANY>{});
  else if (P * C * (long)sizeof(T) < (64L << 20)) go(std::integral_constant<int, BN_FULL>{});
  else go(std::integral_constant<int, BN_STREAM>{});
}

static inline bool bn_aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }
// checks shared by both directions; 0 or a status
static inline int bn_check(const void* x, const void* f, const void* g, int gmode, long P, long L,
                           int C, int dt) {
  if (P <= 0 || P > 0x7fffffffL || L <= 0 || C <= 0 || C > BN_MAX_C || P % L) return ACC_EBADSHAPE;
  if (!x || gmode < BN_GATE_NONE || gmode > BN_GATE_ELEMENT) return ACC_EBADARG;
  if ((gmode != BN_GATE_NONE) != (g != nullptr) || (g && !f)) return ACC_EBADARG;
  if (dt != ACC_F32 && dt != ACC_BF16) return ACC_EBADARG;
  return ACC_OK;
}
