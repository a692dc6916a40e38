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
// read and one write). Per-channel sums and parameters take 56 registers a thread, so a
// row's threads are few enough for 2-3 waves a SIMD and the next row's loads are issued a
// row ahead (327 -> 245 us at 16384 x 4096 bf16; parameters read 16 bytes at a time 194 us;
// one block a CU and streaming stores 171 us; 153-163 us, 4.9-5.3 TB/s, in later traces).
#include "blocknorm.h"

// ge: the gate has a row of its own for every token
template <typename T, int ITER, int WPR, int FORM, bool POST, bool ge>
__global__ void __launch_bounds__(WPR == 1 ? 256 : 64 * WPR)
blocknorm_bwd_kernel(const BlockNormArgs a) {
  constexpr int N = BnGroup<T>::N, NE = ITER * N;
  constexpr int RT = 64 * WPR;
  constexpr int RPB = WPR == 1 ? 4 : 1;
  constexpr bool AHEAD = WPR < 16;  // 16 waves leave too few registers for the next row
  __shared__ float red[2][2][16];
  __shared__ float fold[WPR == 1 ? 4 : 1][2][WPR == 1 ? NE * 64 : 1];
  // sum g*A, sum g*B over the samples of the block; each thread owns its columns
  __shared__ float tot[2][POST ? NE * RT : 1];
  int turn = 0;
  const int t = WPR == 1 ? (threadIdx.x & 63) : threadIdx.x;
  const int sub = WPR == 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  const int C = a.C;
  const float inv = 1.f / (float)C;
  const float layer = a.layer ? inv : 0.f;
  const bool gs = a.gmode == BN_GATE_SAMPLE;
  // s*w1 and s*b1, times the gate of a sample (an element gate multiplies later), and w2
  float p1[NE], p0[NE], w2[NE];
  float A[NE], B[NE], D[NE], E[NE];
  int col[ITER], n[ITER];
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    const int c = (i * RT + t) * N;
    n[i] = max(0, min(N, C - c));
    col[i] = n[i] > 0 ? c : 0;
  }
  auto each = [&](auto fn) {
#pragma unroll
    for (int k = 0; k < NE; ++k) fn(k, k % N < n[k / N], k % N < n[k / N] ? col[k / N] + k % N : 0);
  };
  auto par = [&](const float* p, float fill, float* v) {
#pragma unroll
    for (int i = 0; i < ITER; ++i)
      bn_params<N>(p ? p + col[i] : nullptr, n[i], fill, v + i * N);
  };
  par(a.w2, 1.f, w2);
  // p1, p0 = m * w1, m * b1
  auto products = [&](const float* m) {
    par(a.w1, 1.f, p1);
    par(a.b1, 0.f, p0);
    each([&](int k, bool, int) {
      p1[k] *= m[k];
      p0[k] *= m[k];
    });
  };
  each([&](int k, bool, int) { D[k] = E[k] = 0.f; });
  if (POST) {
    float m[NE];
    par(a.s, 1.f, m);
    products(m);
    if (sub == 0) each([&](int k, bool, int) { tot[0][k * RT + t] = tot[1][k * RT + t] = 0.f; });
  }
  auto load = [&](const void* base, long row, BnGroup<T> (&g)[ITER]) {
    const T* p = (const T*)base + row * C;
#pragma unroll
    for (int i = 0; i < ITER; ++i) g[i] = bn_load<T, FORM>(p + col[i], n[i]);
  };
  auto store = [&](void* base, long row, const float* v) {
    T* p = (T*)base + row * C;
#pragma unroll
    for (int i = 0; i < ITER; ++i) bn_store<T, FORM>(p + col[i], n[i], v + i * N);
  };
  // u, v: the sums of this block over its waves, in every wave (WPR == 1)
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
  BnGroup<T> nx[ITER], nf[ITER], nd[ITER], nh[ITER], ng[ITER];
  float4 nst;
  auto fetch = [&](long p) {
    nst = ld4(a.stats + 4 * p);
    load(a.x, p, nx);
    if (POST) load(a.f, p, nf);
    if (a.dh) load(a.dh, p, nh);
    if (a.dr) load(a.dr, p, nd);
    if (POST && ge) load(a.g, p, ng);
  };
  for (long smp = s0; smp < s1; ++smp) {
    if (POST) {
      if (gs) {
        float m[NE];
        par(a.s, 1.f, m);
        load(a.g, smp, ng);
        each([&](int k, bool, int) { m[k] *= ng[k / N].get(k % N); });
        products(m);
      }
#pragma unroll
      for (int k = 0; k < NE; ++k) A[k] = B[k] = 0.f;
    }
    const long r0 = smp * a.L + part * chunk, r1 = min((smp + 1) * a.L, r0 + chunk);
    if (AHEAD && r0 + sub < r1) fetch(r0 + sub);
    for (long p = r0 + sub; p < r1; p += RPB) {
      if (!AHEAD) fetch(p);
      const float4 st = nst;
      float x[NE], f[NE], d[NE], h[NE], g[NE];
#pragma unroll
      for (int k = 0; k < NE; ++k) {
        x[k] = nx[k / N].get(k % N);
        if (POST) f[k] = nf[k / N].get(k % N);
        h[k] = a.dh ? nh[k / N].get(k % N) : 0.f;
        d[k] = a.dr ? nd[k / N].get(k % N) : 0.f;
        g[k] = POST && ge ? ng[k / N].get(k % N) : 1.f;
      }
      if (AHEAD && p + RPB < r1) fetch(p + RPB);
      if (POST)
        each([&](int k, bool on, int) {
          f[k] = on ? (f[k] - st.x) * st.y : 0.f;
          x[k] += g[k] * (f[k] * p1[k] + p0[k]);
        });
      if (a.dh) {
        float q[2] = {0.f, 0.f};
        each([&](int k, bool on, int) {
          x[k] = on ? (x[k] - st.z) * st.w : 0.f;  // rhat
          D[k] += h[k] * x[k];
          E[k] += h[k];
          h[k] *= w2[k];
          q[0] += h[k];
          q[1] += h[k] * x[k];
        });
        bn_row_sum<WPR, 2>(q, red, turn);
        const float m0 = layer * q[0], m1 = q[1] * inv;
        each([&](int k, bool on, int) {
          d[k] = on ? d[k] + st.w * (h[k] - m0 - x[k] * m1) : 0.f;
        });
      }
      store(a.dx, p, d);
      if (POST) {
        float q[2] = {0.f, 0.f};
        each([&](int k, bool, int) {
          const float dg = d[k] * g[k];
          A[k] += dg * f[k];
          B[k] += dg;
          h[k] = dg * p1[k];
          q[0] += h[k];
          q[1] += h[k] * f[k];
          if (ge) d[k] *= f[k] * p1[k] + p0[k];  // the gate's gradient
        });
        if (ge) store(a.dg, p, d);
        bn_row_sum<WPR, 2>(q, red, turn);
        const float m0 = layer * q[0], m1 = q[1] * inv;
        each([&](int k, bool, int) { h[k] = st.y * (h[k] - m0 - f[k] * m1); });
        store(a.df, p, h);
      }
    }
    if (POST) {
      fold_waves(A, B);
      if (gs) load(a.g, smp, ng);
      if (sub == 0) {
        each([&](int k, bool, int) {
          const float gk = gs ? ng[k / N].get(k % N) : 1.f;
          tot[0][k * RT + t] += gk * A[k];
          tot[1][k * RT + t] += gk * B[k];
        });
        if (gs) {  // dg = s * (w1 * A + b1 * B)
          float m[NE];
          par(a.s, 1.f, m);
          products(m);
          each([&](int k, bool, int) { A[k] = p1[k] * A[k] + p0[k] * B[k]; });
          if (a.S == 1) {
            store(a.dg, smp, A);
          } else {
#pragma unroll
            for (int i = 0; i < ITER; ++i)
              bn_put<N>(a.gpart + (long)blockIdx.x * C + col[i], n[i], A + i * N);
          }
        }
      }
    }
  }
  fold_waves(D, E);
  if (sub == 0) {
    float* o = a.part + (long)blockIdx.x * 4 * C;
    if (POST) each([&](int k, bool, int) {
        A[k] = tot[0][k * RT + t];
        B[k] = tot[1][k * RT + t];
      });
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      if (POST) {
        bn_put<N>(o + col[i], n[i], A + i * N);
        bn_put<N>(o + C + col[i], n[i], B + i * N);
      }
      bn_put<N>(o + 2 * C + col[i], n[i], D + i * N);
      bn_put<N>(o + 3 * C + col[i], n[i], E + i * N);
    }
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
  // blocks that fill the card once: one a CU from 513 threads on, more of the smaller ones;
  // every block writes a row of partial sums, so more of them cost traffic (C = 4096: 512
  // blocks 194 us for 16384 bf16 rows, 256 blocks 174 us)
  const long want = C <= 1024 ? 1024 : C <= 2048 ? 768 : 256;
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
  const bool aligned = bn_aligned(x) && bn_aligned(f) && bn_aligned(g) && bn_aligned(dr) &&
                    bn_aligned(dh) && bn_aligned(dx) && bn_aligned(df) && bn_aligned(dg);
  hipStream_t st = (hipStream_t)stream;
  with_dt(dt, [&](auto tag) {
    using T = decltype(tag);
    bn_with_shape<T>(P, C, aligned, [&](auto sh) {
      using Sh = decltype(sh);
      const int nth = Sh::WPR == 1 ? 256 : 64 * Sh::WPR;
      auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(q.blocks), dim3(nth), 0, st, a);
      };
      if (!f) go(blocknorm_bwd_kernel<T, Sh::ITER, Sh::WPR, Sh::FORM, false, false>);
      else if (q.gmode == BN_GATE_ELEMENT)
        go(blocknorm_bwd_kernel<T, Sh::ITER, Sh::WPR, Sh::FORM, true, true>);
      else go(blocknorm_bwd_kernel<T, Sh::ITER, Sh::WPR, Sh::FORM, true, false>);
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
