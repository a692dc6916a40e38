// Forward of the norms around a residual block; mathematics and layout in blocknorm.h.
// Bound by memory: x and f (and an element gate) are read once, r and h written once.
// Kernel traces: 16384 x 4096 bf16 100-126 us, 4.3-5.4 TB/s (streaming stores are a tenth of
// it); 16384 x 2048 fp32 105 us, 5.1 TB/s; 25088 x 160 fp32 17-18 us.
#include "blocknorm.h"

template <typename T, int ITER, int WPR, int FORM, bool POST>
__global__ void __launch_bounds__(WPR == 1 ? 256 : 64 * WPR)
blocknorm_fwd_kernel(const BlockNormArgs a) {
  constexpr int N = BnGroup<T>::N, NE = ITER * N;
  constexpr int RT = 64 * WPR;               // threads of a row
  constexpr int RPB = WPR == 1 ? 4 : 1;      // rows of a block
  __shared__ float red[2][2][16];
  int turn = 0;
  const int t = WPR == 1 ? (threadIdx.x & 63) : threadIdx.x;
  const int sub = WPR == 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  const int C = a.C;
  const float len = (float)C;  // divided by, not multiplied by 1/C: a constant row has mean v
  float p1[NE], p0[NE], w2[NE], b2[NE];  // s * w1, s * b1 (the gate multiplies both)
  int col[ITER], n[ITER];
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    const int c = (i * RT + t) * N;
    n[i] = max(0, min(N, C - c));
    col[i] = n[i] > 0 ? c : 0;
    auto par = [&](const float* p, float fill, float* v) {
      bn_params<N>(p ? p + col[i] : nullptr, n[i], fill, v + i * N);
    };
    if (POST) {
      float s[NE];
      par(a.s, 1.f, s);
      par(a.w1, 1.f, p1);
      par(a.b1, 0.f, p0);
#pragma unroll
      for (int k = i * N; k < i * N + N; ++k) {
        p1[k] *= s[k];
        p0[k] *= s[k];
      }
    }
    par(a.w2, 1.f, w2);
    par(a.b2, 0.f, b2);
  }
  // mean and 1/sqrt(var + eps) of v (zero off the row), v replaced by v - mean
  auto norm = [&](float (&v)[NE], float& mean, float& rstd) {
    float q[1] = {0.f};
    mean = 0.f;
    if (a.layer) {
#pragma unroll
      for (int k = 0; k < NE; ++k) q[0] += v[k];
      bn_row_sum<WPR, 1>(q, red, turn);
      mean = q[0] / len;
      q[0] = 0.f;
#pragma unroll
      for (int k = 0; k < NE; ++k) v[k] = k % N < n[k / N] ? v[k] - mean : 0.f;
    }
#pragma unroll
    for (int k = 0; k < NE; ++k) q[0] += v[k] * v[k];
    bn_row_sum<WPR, 1>(q, red, turn);
    rstd = 1.f / sqrtf(q[0] / len + a.eps);
  };
  const bool gate = a.gmode != BN_GATE_NONE;
  auto load = [&](const void* base, long row, BnGroup<T> (&g)[ITER]) {
    const T* p = (const T*)base + row * C;
#pragma unroll
    for (int i = 0; i < ITER; ++i) g[i] = bn_load<T, FORM>(p + col[i], n[i]);
  };
  BnGroup<T> nx[ITER], nf[ITER], ng[ITER];
  auto fetch = [&](long p) {
    load(a.x, p, nx);
    if (POST) {
      load(a.f, p, nf);
      if (gate) load(a.g, a.gmode == BN_GATE_SAMPLE ? (long)fdiv((unsigned)p, a.fL) : p, ng);
    }
  };
  // a run of neighbouring rows a block
  const long run = (a.P + gridDim.x - 1) / gridDim.x;
  long p = blockIdx.x * run + sub;
  const long end = min(a.P, (blockIdx.x + 1) * run);
  const long step = RPB;
  if (p < end) fetch(p);
  for (; p < end; p += step) {
    float x[NE], f[NE], g[NE];
#pragma unroll
    for (int k = 0; k < NE; ++k) {
      x[k] = nx[k / N].get(k % N);
      if (POST) {
        f[k] = nf[k / N].get(k % N);
        g[k] = gate ? ng[k / N].get(k % N) : 1.f;
      }
    }
    if (p + step < end) fetch(p + step);
    float m1 = 0.f, rs1 = 0.f, m2 = 0.f, rs2 = 0.f;
    if (POST) {
      norm(f, m1, rs1);
#pragma unroll
      for (int k = 0; k < NE; ++k)
        x[k] = k % N < n[k / N] ? x[k] + g[k] * (f[k] * rs1 * p1[k] + p0[k]) : 0.f;
      // h is taken of the unrounded r below: its rounding to bf16 stays out of the norm
#pragma unroll
      for (int i = 0; i < ITER; ++i)
        bn_store<T, FORM>((T*)a.r + p * C + col[i], n[i], x + i * N);
    }
    if (a.h) {
      norm(x, m2, rs2);
#pragma unroll
      for (int k = 0; k < NE; ++k) x[k] = x[k] * rs2 * w2[k] + b2[k];
#pragma unroll
      for (int i = 0; i < ITER; ++i)
        bn_store<T, FORM>((T*)a.h + p * C + col[i], n[i], x + i * N);
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
  a.fL = make_fastdiv((uint32_t)L);
 
  const bool aligned =
      bn_aligned(x) && bn_aligned(f) && bn_aligned(g) && bn_aligned(r) && bn_aligned(h);
  with_dt(dt, [&](auto tag) {
    using T = decltype(tag);
    bn_with_shape<T>(P, C, aligned, [&](auto sh) {
      using S = decltype(sh);
      const int rpb = S::WPR == 1 ? 4 : 1;
      const int nth = S::WPR == 1 ? 256 : 64 * S::WPR;
      const long cap = 1024L * 4 / (nth / 64);  // 16 waves a CU
      const dim3 grid((unsigned)min((P + rpb - 1) / rpb, cap));
      if (f)
        hipLaunchKernelGGL((blocknorm_fwd_kernel<T, S::ITER, S::WPR, S::FORM, true>), grid,
                           dim3(nth), 0, (hipStream_t)stream, a);
      else
        hipLaunchKernelGGL((blocknorm_fwd_kernel<T, S::ITER, S::WPR, S::FORM, false>), grid,
                           dim3(nth), 0, (hipStream_t)stream, a);
    });
  });
  return hipGetLastError() == hipSuccess ? ACC_OK : ACC_ELAUNCH;
}
