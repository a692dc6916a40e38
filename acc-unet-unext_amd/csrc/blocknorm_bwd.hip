// Backward of the norms around a residual block; mathematics and layout in blocknorm.h.
//
//   gr = dr + norm'(dh * w2; r)      dx = gr       du = gr * s * g
//   df = norm'(du * w1; f)           dg = gr * s * u, summed over a sample's rows if shared
//   dw1 = sum du * fhat   db1 = sum du   ds = sum gr * g * u   dw2 = sum dh * rhat   db2 = sum dh
//   norm'(d; v) = rstd * (d - mean(d) [layer] - vhat * mean(d * vhat))
//
// r is not read: it is recomputed from x and f, which costs a few multiplies and keeps the
// unrounded value that the forward normalised. With A = sum gr*fhat and B = sum gr over the
// rows that share a gate, u = fhat*w1 + b1 gives dw1 = s*sum g*A, db1 = s*sum g*B,
// ds = w1*sum g*A + b1*sum g*B and dg = s*(w1*A + b1*B): four running sums a column (two for
// dw2, db2) hold every parameter gradient. Each block writes its sums once; finish kernels
// add the blocks' rows in a fixed order (no atomics).
// Bound by memory: x, f, dr, dh read once, dx, df written once (an element gate adds one
// read and one write).
#include "blocknorm.h"

template <typename T, int VEC, int ITER, int WPR, bool POST>
__global__ void __launch_bounds__(WPR == 1 ? 256 : 64 * WPR)
blocknorm_bwd_kernel(const BlockNormArgs a) {
  constexpr int RT = 64 * WPR;
  constexpr int RPB = WPR == 1 ? 4 : 1;
  constexpr int NE = ITER * VEC;
  __shared__ float red[2][2][16];
  __shared__ float fold[WPR == 1 ? 4 : 1][2][WPR == 1 ? NE * 64 : 1];
  int turn = 0;
  const int t = WPR == 1 ? (threadIdx.x & 63) : threadIdx.x;
  const int sub = WPR == 1 ? (threadIdx.x >> 6) : 0;
  const int C = a.C;
  const float inv = 1.f / (float)C;
  const float layer = a.layer ? 1.f : 0.f;
  const bool gs = a.gmode == BN_GATE_SAMPLE, ge = a.gmode == BN_GATE_ELEMENT;
  float w1[NE], b1[NE], s[NE], w2[NE], g[NE];
  float A[NE], B[NE], gA[NE], gB[NE], D[NE], E[NE];
  int col[ITER];
  bool on[ITER];
  auto each = [&](auto fn) {
#pragma unroll
    for (int i = 0; i < ITER; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) fn(i, i * VEC + j, j);
  };
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    col[i] = (i * RT + t) * VEC;
    on[i] = col[i] < C;
    if (!on[i]) col[i] = 0;
  }
  each([&](int i, int k, int j) {
    if (POST) {
      w1[k] = a.w1 ? a.w1[col[i] + j] : 1.f;
      b1[k] = a.b1 ? a.b1[col[i] + j] : 0.f;
      s[k] = a.s ? a.s[col[i] + j] : 1.f;
      gA[k] = gB[k] = 0.f;
    }
    w2[k] = a.w2 ? a.w2[col[i] + j] : 1.f;
    D[k] = E[k] = 0.f;
    g[k] = 1.f;
  });
  const T* X = (const T*)a.x;
  const T* F = (const T*)a.f;
  const T* Gt = (const T*)a.g;
  const T* DR = (const T*)a.dr;
  const T* DH = (const T*)a.dh;
  auto load = [&](const T* base, long p, float* v) {
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      float q[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) q[j] = 0.f;
      if (on[i]) bn_load<VEC>(base + p * C + col[i], q);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i * VEC + j] = q[j];
    }
  };
  auto store = [&](T* base, long p, const float* v) {
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      float q[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) q[j] = v[i * VEC + j];
      if (on[i]) bn_store<VEC>(base + p * C + col[i], q);
    }
  };
  // u, v: the sums of this block over its waves, left in wave 0 (WPR == 1)
  auto fold_waves = [&](float* u, float* v) {
    if constexpr (WPR == 1) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < NE; ++k) {
        fold[sub][0][k * 64 + t] = u[k];
        fold[sub][1][k * 64 + t] = v[k];
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < NE; ++k) {
        float p = fold[0][0][k * 64 + t], q = fold[0][1][k * 64 + t];
#pragma unroll
        for (int w = 1; w < 4; ++w) {
          p += fold[w][0][k * 64 + t];
          q += fold[w][1][k * 64 + t];
        }
        u[k] = p;
        v[k] = q;
      }
    }
  };
  const long nb = a.P / a.L;  // samples
  const long s0 = a.S > 1 ? blockIdx.x / a.S : (long)blockIdx.x * a.G;
  const long s1 = min(nb, s0 + (a.S > 1 ? 1 : a.G));
  const int part = a.S > 1 ? blockIdx.x % a.S : 0;
  const long chunk = (a.L + a.S - 1) / a.S;
  for (long smp = s0; smp < s1; ++smp) {
    if (POST) {
      if (gs) load(Gt, smp, g);
#pragma unroll
      for (int k = 0; k < NE; ++k) A[k] = B[k] = 0.f;
    }
    const long r0 = smp * a.L + part * chunk, r1 = min((smp + 1) * a.L, r0 + chunk);
    for (long p = r0 + sub; p < r1; p += RPB) {
      const float4 st = ld4(a.stats + 4 * p);
      float x[NE], f[NE], d[NE], h[NE];
      load(X, p, x);
      if (POST) load(F, p, f);
      if (a.dh) load(DH, p, h);
      if (a.dr) load(DR, p, d);
      if (POST) {
        if (ge) load(Gt, p, g);
        each([&](int i, int k, int) {
          f[k] = on[i] ? (f[k] - st.x) * st.y : 0.f;
          x[k] += s[k] * g[k] * (f[k] * w1[k] + b1[k]);
        });
      }
      if (!a.dr) each([&](int, int k, int) { d[k] = 0.f; });
      if (a.dh) {
        float q[2] = {0.f, 0.f};
        each([&](int i, int k, int) {
          x[k] = on[i] ? (x[k] - st.z) * st.w : 0.f;  // rhat
          D[k] += h[k] * x[k];
          E[k] += h[k];
          h[k] *= w2[k];
          q[0] += h[k];
          q[1] += h[k] * x[k];
        });
        bn_row_sum<WPR, 2>(q, red, turn);
        const float m0 = layer * q[0] * inv, m1 = q[1] * inv;
        each([&](int, int k, int) { d[k] += st.w * (h[k] - m0 - x[k] * m1); });
      }
      store((T*)a.dx, p, d);
      if (POST) {
        float q[2] = {0.f, 0.f};
        each([&](int i, int k, int) {
          if (!on[i]) d[k] = 0.f;
          const float dg = ge ? d[k] * g[k] : d[k];
          A[k] += dg * f[k];
          B[k] += dg;
          h[k] = d[k] * s[k] * g[k] * w1[k];
          q[0] += h[k];
          q[1] += h[k] * f[k];
          if (ge) d[k] *= s[k] * (f[k] * w1[k] + b1[k]);
        });
        if (ge && a.dg) store((T*)a.dg, p, d);
        bn_row_sum<WPR, 2>(q, red, turn);
        const float m0 = layer * q[0] * inv, m1 = q[1] * inv;
        each([&](int, int k, int) { h[k] = st.y * (h[k] - m0 - f[k] * m1); });
        store((T*)a.df, p, h);
      }
    }
    if (POST) {
      fold_waves(A, B);
      each([&](int, int k, int) {
        gA[k] += gs ? g[k] * A[k] : A[k];
        gB[k] += gs ? g[k] * B[k] : B[k];
        A[k] = s[k] * (w1[k] * A[k] + b1[k] * B[k]);
      });
      if (gs && sub == 0) {
        if (a.S == 1) {
          store((T*)a.dg, smp, A);
        } else {
#pragma unroll
          for (int i = 0; i < ITER; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j)
              if (on[i]) a.gpart[(long)blockIdx.x * C + col[i] + j] = A[i * VEC + j];
        }
      }
    }
  }
  fold_waves(D, E);
  if (sub == 0) {
    float* o = a.part + (long)blockIdx.x * 4 * C;
    each([&](int i, int k, int j) {
      if (!on[i]) return;
      const int c = col[i] + j;
      if (POST) {
        o[c] = gA[k];
        o[C + c] = gB[k];
      }
      o[2 * C + c] = D[k];
      o[3 * C + c] = E[k];
    });
  }
}

// dpar [5][C] = dw1, db1, ds, dw2, db2 from the blocks' rows part [R][4][C]: 64 columns a
// block, 16 groups of rows added in a fixed order in fp64. blockIdx.y picks the pair.
__global__ void __launch_bounds__(1024)
blocknorm_finish_kernel(const float* __restrict__ part, int R, int C, const float* __restrict__ w1,
                        const float* __restrict__ b1, const float* __restrict__ s,
                        float* __restrict__ dpar, int post) {
  __shared__ double red[2][16][64];
  const int cl = threadIdx.x & 63, gq = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + cl;
  const int pair = post ? (int)blockIdx.y : 1;
  const float* src = part + (long)pair * 2 * C;
  double v[2] = {0.0, 0.0};
  if (c < C)
    ordered_strided_sum<4>(v, gq, R, 16, [&](int r, double (&o)[2]) {
      o[0] = src[(long)r * 4 * C + c];
      o[1] = src[(long)r * 4 * C + C + c];
    });
  red[0][gq][cl] = v[0];
  red[1][gq][cl] = v[1];
  __syncthreads();
  if (gq == 0 && c < C) {
    double p = 0.0, q = 0.0;
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      p += red[0][k][cl];
      q += red[1][k][cl];
    }
    if (pair == 0) {
      const float sc = s ? s[c] : 1.f;
      dpar[c] = (float)(sc * p);
      dpar[C + c] = (float)(sc * q);
      dpar[2 * C + c] = (float)((w1 ? w1[c] : 1.f) * p + (b1 ? b1[c] : 0.f) * q);
    } else {
      dpar[3 * C + c] = (float)p;
      dpar[4 * C + c] = (float)q;
    }
  }
}

// dg[b][c] = sum over the S blocks of sample b, in order
template <typename T>
__global__ void __launch_bounds__(256)
blocknorm_gate_kernel(const float* __restrict__ gpart, T* __restrict__ dg, long n, int C, int S) {
  const long e = blockIdx.x * 256L + threadIdx.x;
  if (e >= n) return;
  const long b = e / C;
  const float* src = gpart + b * S * C + (e - b * C);
  float v[1] = {0.f};
  ordered_strided_sum<4>(v, 0, S, 1, [&](int k, float (&o)[1]) { o[0] = src[(long)k * C]; });
  st1(dg + e, v[0]);
}

// How the rows are cut over blocks: S blocks a sample, or G samples a block. Gates that are
// not shared count as one sample of P rows.
struct BnPlan {
  long L;
  int gmode, G, S, blocks;
};
static BnPlan bn_plan(long P, long L, int C, int gmode) {
  BnPlan q;
  q.gmode = gmode == BN_GATE_SAMPLE && L == 1 ? BN_GATE_ELEMENT : gmode;
  q.L = q.gmode == BN_GATE_SAMPLE ? L : P;
  const int rpb = C <= 512 ? 4 : 1;
  const long want = C <= 1024 ? 1024 : C <= 2048 ? 768 : C <= 4096 ? 512 : 256;
  const long n = P / q.L;
  q.G = n >= want ? (int)((n + want - 1) / want) : 1;
  q.S = n >= want ? 1 : (int)min((want + n - 1) / n, (q.L + rpb - 1) / rpb);
  q.blocks = q.S > 1 ? (int)(n * q.S) : (int)((n + q.G - 1) / q.G);
  return q;
}

extern "C" size_t accunet_blocknorm_ws_elems(long P, long L, int C, int gmode) {
  if (P <= 0 || L <= 0 || C <= 0 || C > BN_MAX_C || P % L) return 0;
  const BnPlan q = bn_plan(P, L, C, gmode);
  size_t n = (size_t)q.blocks * 4 * C;
  if (q.gmode == BN_GATE_SAMPLE && q.S > 1) n += (size_t)q.blocks * C;
  return n;
}

extern "C" int accunet_blocknorm_bwd(const void* x, const void* f, const float* w1,
                                     const float* b1, const float* s, const void* g, int gmode,
                                     const float* w2, int layer, const float* stats,
                                     const void* dr, const void* dh, void* dx, void* df, void* dg,
                                     float* dpar, float* ws, size_t ws_elems, long P, long L, int C,
                                     int dt, void* stream) {
  const int rc = bn_check(x, f, g, gmode, P, L, C, dt);
  if (rc != ACC_OK) return rc;
  if (!stats || !dx || !dpar || !ws || (!dr && !dh) || (f != nullptr) != (df != nullptr) ||
      (g != nullptr) != (dg != nullptr))
    return ACC_EBADARG;
  if (ws_elems < accunet_blocknorm_ws_elems(P, L, C, gmode)) return ACC_EBADARG;
  const BnPlan q = bn_plan(P, L, C, gmode);
  BlockNormArgs a = {};
  a.x = x; a.f = f; a.g = g; a.dr = dr; a.dh = dh;
  a.w1 = w1; a.b1 = b1; a.s = s; a.w2 = w2;
  a.dx = dx; a.df = df; a.dg = dg;
  a.stats = const_cast<float*>(stats);
  a.part = ws;
  a.gpart = ws + (size_t)q.blocks * 4 * C;
  a.P = P; a.L = q.L; a.C = C; a.gmode = q.gmode; a.layer = layer != 0;
  a.G = q.G; a.S = q.S;
  const bool vec = bn_aligned(x) && bn_aligned(f) && bn_aligned(g) && bn_aligned(dr) &&
                   bn_aligned(dh) && bn_aligned(dx) && bn_aligned(df) && bn_aligned(dg);
  hipStream_t st = (hipStream_t)stream;
  with_dt(dt, [&](auto tag) {
    using T = decltype(tag);
    bn_with_shape<T>(C, vec, [&](auto sh) {
      using Sh = decltype(sh);
      const int nth = Sh::WPR == 1 ? 256 : 64 * Sh::WPR;
      if (f)
        hipLaunchKernelGGL((blocknorm_bwd_kernel<T, Sh::VEC, Sh::ITER, Sh::WPR, true>),
                           dim3(q.blocks), dim3(nth), 0, st, a);
      else
        hipLaunchKernelGGL((blocknorm_bwd_kernel<T, Sh::VEC, Sh::ITER, Sh::WPR, false>),
                           dim3(q.blocks), dim3(nth), 0, st, a);
    });
    if (q.gmode == BN_GATE_SAMPLE && q.S > 1) {
      const long n = P / L * C;
      hipLaunchKernelGGL(blocknorm_gate_kernel<T>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0,
                         st, a.gpart, (T*)dg, n, C, q.S);
    }
  });
  hipLaunchKernelGGL(blocknorm_finish_kernel, dim3(ceil_div(C, 64), f ? 2 : 1), dim3(1024), 0, st,
                     ws, q.blocks, C, w1, b1, s, dpar, f ? 1 : 0);
  return hipGetLastError() == hipSuccess ? ACC_OK : ACC_ELAUNCH;
}
