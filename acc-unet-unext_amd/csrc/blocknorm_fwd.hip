// Forward of the norms around a residual block; mathematics and layout in blocknorm.h.
// Bound by memory: x and f (and an element gate) are read once, r and h written once.
#include "blocknorm.h"

template <typename T, int VEC, int ITER, int WPR, bool POST>
__global__ void __launch_bounds__(WPR == 1 ? 256 : 64 * WPR)
blocknorm_fwd_kernel(const BlockNormArgs a) {
  constexpr int RT = 64 * WPR;               // threads of a row
  constexpr int RPB = WPR == 1 ? 4 : 1;      // rows of a block
  __shared__ float red[2][2][16];
  int turn = 0;
  const int t = WPR == 1 ? (threadIdx.x & 63) : threadIdx.x;
  const int sub = WPR == 1 ? (threadIdx.x >> 6) : 0;
  const int C = a.C;
  const float n = (float)C;  // divided by, not multiplied by 1/n: a constant row has mean v
  float w1[ITER][VEC], b1[ITER][VEC], s[ITER][VEC], w2[ITER][VEC], b2[ITER][VEC];
  int col[ITER];
  bool on[ITER];
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    col[i] = (i * RT + t) * VEC;
    on[i] = col[i] < C;
    if (!on[i]) col[i] = 0;
    if (POST) {
      bn_param<VEC>(a.w1, col[i], 1.f, w1[i]);
      bn_param<VEC>(a.b1, col[i], 0.f, b1[i]);
      bn_param<VEC>(a.s, col[i], 1.f, s[i]);
    }
    bn_param<VEC>(a.w2, col[i], 1.f, w2[i]);
    bn_param<VEC>(a.b2, col[i], 0.f, b2[i]);
  }
  // mean and 1/sqrt(var + eps) of v (zero off the row), v replaced by v - mean
  auto norm = [&](float (&v)[ITER][VEC], float& mean, float& rstd) {
    float q[1] = {0.f};
    mean = 0.f;
    if (a.layer) {
#pragma unroll
      for (int i = 0; i < ITER; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) q[0] += v[i][j];
      bn_row_sum<WPR, 1>(q, red, turn);
      mean = q[0] / n;
      q[0] = 0.f;
#pragma unroll
      for (int i = 0; i < ITER; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] = on[i] ? v[i][j] - mean : 0.f;
    }
#pragma unroll
    for (int i = 0; i < ITER; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) q[0] += v[i][j] * v[i][j];
    bn_row_sum<WPR, 1>(q, red, turn);
    rstd = 1.f / sqrtf(q[0] / n + a.eps);
  };
  const T* X = (const T*)a.x;
  const T* F = (const T*)a.f;
  const T* Gt = (const T*)a.g;
  for (long p0 = (long)blockIdx.x * RPB; p0 < a.P; p0 += (long)gridDim.x * RPB) {
    const long p = p0 + sub;
    if (RPB > 1 && p >= a.P) break;
    float x[ITER][VEC], f[ITER][VEC];
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) x[i][j] = f[i][j] = 0.f;
      if (on[i]) {
        if (POST) bn_load<VEC>(F + p * C + col[i], f[i]);
        bn_load<VEC>(X + p * C + col[i], x[i]);
      }
    }
    float m1 = 0.f, rs1 = 0.f, m2 = 0.f, rs2 = 0.f;
    if (POST) {
      float g[ITER][VEC];
      const long grow = a.gmode == BN_GATE_SAMPLE ? p / a.L : p;
#pragma unroll
      for (int i = 0; i < ITER; ++i) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) g[i][j] = 1.f;
        if (a.gmode != BN_GATE_NONE && on[i]) bn_load<VEC>(Gt + grow * C + col[i], g[i]);
      }
      norm(f, m1, rs1);
#pragma unroll
      for (int i = 0; i < ITER; ++i) {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          x[i][j] += s[i][j] * g[i][j] * (f[i][j] * rs1 * w1[i][j] + b1[i][j]);
        if (!on[i])
#pragma unroll
          for (int j = 0; j < VEC; ++j) x[i][j] = 0.f;
        // h is taken of the unrounded r below: its rounding to bf16 stays out of the norm
        if (on[i]) bn_store<VEC>((T*)a.r + p * C + col[i], x[i]);
      }
    }
    if (a.h) {
      norm(x, m2, rs2);
#pragma unroll
      for (int i = 0; i < ITER; ++i) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[i][j] = x[i][j] * rs2 * w2[i][j] + b2[i][j];
        if (on[i]) bn_store<VEC>((T*)a.h + p * C + col[i], x[i]);
      }
    }
    if (a.stats && t == 0) st4(a.stats + 4 * p, make_float4(m1, rs1, m2, rs2));
  }
}

extern "C" int accunet_blocknorm_fwd(const void* x, const void* f, const float* w1,
                                     const float* b1, const float* s, const void* g, int gmode,
                                     const float* w2, const float* b2, int layer, float eps,
                                     void* r, void* h, float* stats, long P, long L, int C, int dt,
                                     void* stream) {
  const int rc = bn_check(x, f, g, gmode, P, L, C, dt);
  if (rc != ACC_OK) return rc;
  if ((f != nullptr) != (r != nullptr) || (!f && !h)) return ACC_EBADARG;
  BlockNormArgs a = {};
  a.x = x; a.f = f; a.g = g;
  a.w1 = w1; a.b1 = b1; a.s = s; a.w2 = w2; a.b2 = b2;
  a.r = r; a.h = h; a.stats = stats;
  a.P = P; a.L = L; a.C = C; a.gmode = gmode; a.layer = layer != 0; a.eps = eps;
  const bool vec = bn_aligned(x) && bn_aligned(f) && bn_aligned(g) && bn_aligned(r) && bn_aligned(h);
  with_dt(dt, [&](auto tag) {
    using T = decltype(tag);
    bn_with_shape<T>(C, vec, [&](auto sh) {
      using S = decltype(sh);
      const int rpb = S::WPR == 1 ? 4 : 1;
      const int nth = S::WPR == 1 ? 256 : 64 * S::WPR;
      const long cap = 2048L * 4 / (nth / 64);  // 32 waves a CU
      const dim3 grid((unsigned)min((P + rpb - 1) / rpb, cap));
      if (f)
        hipLaunchKernelGGL((blocknorm_fwd_kernel<T, S::VEC, S::ITER, S::WPR, true>), grid,
                           dim3(nth), 0, (hipStream_t)stream, a);
      else
        hipLaunchKernelGGL((blocknorm_fwd_kernel<T, S::VEC, S::ITER, S::WPR, false>), grid,
                           dim3(nth), 0, (hipStream_t)stream, a);
    });
  });
  return hipGetLastError() == hipSuccess ? ACC_OK : ACC_ELAUNCH;
}
