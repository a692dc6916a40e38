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
// elements a thread at most (ITER groups of VEC neighbours, group i at column
// (i*64*WPR + t)*VEC), so every tensor is read once and every statistic is a two-pass sum
// over registers. WPR = 1 runs four rows in a 256-thread block (C <= 512, no barrier),
// larger rows take one block of 64*WPR threads. VEC is 16 bytes (4 fp32, 8 bf16) where C
// and every pointer allow it, else 1.
#pragma once
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
  int G, S;      // backward: samples per block (S == 1) / blocks per sample (G == 1)
};

template <int VEC>
ACC_DEV void bn_load(const float* p, float (&v)[VEC]) {
  if constexpr (VEC == 4) {
    const float4 q = ld4(p);
    v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
  } else {
    v[0] = *p;
  }
}
template <int VEC>
ACC_DEV void bn_load(const bf16_t* p, float (&v)[VEC]) {
  if constexpr (VEC == 8) {
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    v[0] = bflo(q.x); v[1] = bfhi(q.x); v[2] = bflo(q.y); v[3] = bfhi(q.y);
    v[4] = bflo(q.z); v[5] = bfhi(q.z); v[6] = bflo(q.w); v[7] = bfhi(q.w);
  } else {
    v[0] = bf2f(*p);
  }
}
template <int VEC>
ACC_DEV void bn_store(float* p, const float (&v)[VEC]) {
  if constexpr (VEC == 4) st4(p, make_float4(v[0], v[1], v[2], v[3]));
  else *p = v[0];
}
template <int VEC>
ACC_DEV void bn_store(bf16_t* p, const float (&v)[VEC]) {
  if constexpr (VEC == 8)
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]),
                                              pack_bf2(v[4], v[5]), pack_bf2(v[6], v[7]));
  else *p = f2bf(v[0]);
}
// parameters are fp32 whatever the activations' type
template <int VEC>
ACC_DEV void bn_param(const float* p, long c, float fill, float (&v)[VEC]) {
#pragma unroll
  for (int j = 0; j < VEC; ++j) v[j] = p ? p[c + j] : fill;
}

ACC_DEV float bn_wave_sum(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
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
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < WPR; ++w) t += red[h][k][w];
      v[k] = t;
    }
  }
}

// Run f(VEC, ITER, WPR as constants) for a row of C elements of T; false past BN_MAX_C.
template <int V, int I, int W>
struct BnShape {
  static constexpr int VEC = V, ITER = I, WPR = W;
};
template <typename T, typename F>
static inline bool bn_with_shape(int C, bool vec, F f) {
  constexpr int FV = sizeof(T) == 4 ? 4 : 8;
  if (C > BN_MAX_C) return false;
  if (vec && C % FV == 0) {
    constexpr int FI = 8 / FV;
    if (FI > 1 && C <= 256) f(BnShape<FV, 1, 1>{});
    else if (C <= 512) f(BnShape<FV, FI, 1>{});
    else if (C <= 1024) f(BnShape<FV, FI, 2>{});
    else if (C <= 2048) f(BnShape<FV, FI, 4>{});
    else if (C <= 4096) f(BnShape<FV, FI, 8>{});
    else f(BnShape<FV, FI, 16>{});
  } else {
    if (C <= 512) f(BnShape<1, 8, 1>{});
    else if (C <= 1024) f(BnShape<1, 8, 2>{});
    else if (C <= 2048) f(BnShape<1, 8, 4>{});
    else if (C <= 4096) f(BnShape<1, 8, 8>{});
    else f(BnShape<1, 8, 16>{});
  }
  return true;
}

static inline bool bn_aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }
// checks shared by both directions; 0 or a status
static inline int bn_check(const void* x, const void* f, const void* g, int gmode, long P, long L,
                           int C, int dt) {
  if (P <= 0 || L <= 0 || C <= 0 || C > BN_MAX_C || P % L) return ACC_EBADSHAPE;
  if (!x || gmode < BN_GATE_NONE || gmode > BN_GATE_ELEMENT) return ACC_EBADARG;
  if ((gmode != BN_GATE_NONE) != (g != nullptr) || (g && !f)) return ACC_EBADARG;
  if (dt != ACC_F32 && dt != ACC_BF16) return ACC_EBADARG;
  return ACC_OK;
}
