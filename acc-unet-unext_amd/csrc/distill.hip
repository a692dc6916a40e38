// Distillation from a teacher's top logits; mathematics in distill.h. This file: the
// teacher's pass, the loss over the rows, and the layout with the classes on the channel
// axis of an image (z [B][V][S]). Rows with the classes last: distill_rows.hip.
#include "distill.h"

// ------------------------------------------------------------------ the teacher's entries
// p and the entries that count, each class once: id = the class at its first entry (p the
// sum over its entries), -1 elsewhere. tea[row] = (sum p log2 p + rest log2 rest, 1 or 0).
// Also counts the rows that have an entry (integers: the order of the adds is immaterial).
//
// One wave a row, entries k = lane + 64 i. Bound by latency: K^2 / 64 comparisons a lane.
template <typename IT, typename TT>
__global__ void __launch_bounds__(256)
distill_teacher_rows_kernel(const IT* __restrict__ idx, const TT* __restrict__ top,
                            const float* __restrict__ rest, int* __restrict__ id,
                            float* __restrict__ p, float2* __restrict__ tea, int* count, long R,
                            int V, int K, float c) {
  __shared__ int sid[4][DT_MAX_K];
  __shared__ float sp[4][DT_MAX_K];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long row = blockIdx.x * 4L + wave;
  if (row >= R) return;
  const int NI = (K + 63) / 64;
  int my[DT_MAX_K / 64];
  float a[DT_MAX_K / 64];
  float mx = -INFINITY;
  bool any = false;
#pragma unroll
  for (int i = 0; i < DT_MAX_K / 64; ++i) {
    const int k = i * 64 + lane;
    my[i] = -1;
    a[i] = -INFINITY;
    if (i < NI && k < K) {
      const long long j = (long long)idx[row * K + k];
      if (j >= 0 && j < V) {
        my[i] = (int)j;
        a[i] = ld1(top + row * K + k);
        mx = fmaxf(mx, a[i]);
        any |= !(a[i] == -INFINITY);
      }
    }
  }
  mx = dt_wave_max(mx);
  const bool live = __any(any);
  const float ref = dt_ref(mx, c);
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < DT_MAX_K / 64; ++i)
    if (my[i] >= 0) sum += dt_exp2(__builtin_fmaf(a[i], c, -ref));
  sum = dt_wave_sum(sum);
  const float r = live && rest ? rest[row] : 0.f;
  const float keep = 1.f - r, lg = log2f(sum) - log2f(keep);
  float h = 0.f;
#pragma unroll
  for (int i = 0; i < DT_MAX_K / 64; ++i) {
    const int k = i * 64 + lane;
    if (i >= NI || k >= K) continue;
    const float e = __builtin_fmaf(a[i], c, -ref);
    const float v = my[i] >= 0 && live ? keep * (dt_exp2(e) / sum) : 0.f;
    if (!(v == 0.f)) h += v * (e - lg);
    a[i] = v;
    sid[wave][k] = my[i];
    sp[wave][k] = v;
  }
  h = dt_wave_sum(h);
  if (r != 0.f) h += r * log2f(r);
  dt_wave_lds();
#pragma unroll
  for (int i = 0; i < DT_MAX_K / 64; ++i) {
    const int k = i * 64 + lane;
    if (i >= NI || k >= K) continue;
    bool first = my[i] >= 0 && live;
    float v = 0.f;
    for (int q = 0; q < K; ++q)
      if (sid[wave][q] == my[i]) {
        if (q < k) first = false;
        v += sp[wave][q];
      }
    id[row * K + k] = first ? my[i] : -1;
    p[row * K + k] = v;
  }
  if (lane == 0) {
    tea[row] = make_float2(h, live ? 1.f : 0.f);
    if (live) atomicAdd(count, 1);
  }
}

// Classes on the channel axis: idx, top [B][K][S], one thread a pixel; the entries of a
// pixel are re-read from the cache for each of the passes.
template <typename IT, typename TT>
__global__ void __launch_bounds__(256)
distill_teacher_planes_kernel(const IT* __restrict__ idx, const TT* __restrict__ top,
                              const float* __restrict__ rest, int* __restrict__ id,
                              float* __restrict__ p, float2* __restrict__ tea, int* count, long N,
                              long S, int V, int K, float c) {
  const long row = blockIdx.x * 256L + threadIdx.x;
  bool live = false;
  if (row < N) {
    const long b = row / S, base = b * K * S + (row - b * S);
    float mx = -INFINITY;
    for (int k = 0; k < K; ++k) {
      const long long j = (long long)idx[base + k * S];
      if (j >= 0 && j < V) {
        const float a = ld1(top + base + k * S);
        mx = fmaxf(mx, a);
        live |= !(a == -INFINITY);
      }
    }
    const float ref = dt_ref(mx, c);
    float sum = 0.f;
    for (int k = 0; k < K; ++k) {
      const long long j = (long long)idx[base + k * S];
      if (j >= 0 && j < V) sum += dt_exp2(__builtin_fmaf(ld1(top + base + k * S), c, -ref));
    }
    const float r = live && rest ? rest[row] : 0.f;
    const float keep = 1.f - r, lg = log2f(sum) - log2f(keep);
    float h = r != 0.f ? r * log2f(r) : 0.f;
    for (int k = 0; k < K; ++k) {
      const long long j = (long long)idx[base + k * S];
      int mine = -1;
      float v = 0.f;
      if (live && j >= 0 && j < V) {
        mine = (int)j;
        const float e = __builtin_fmaf(ld1(top + base + k * S), c, -ref);
        v = keep * (dt_exp2(e) / sum);
        if (!(v == 0.f)) h += v * (e - lg);
        for (int q = 0; q < k; ++q)  // listed before: its mass joins the first entry
          if (mine >= 0 && id[base + q * S] == mine) {
            p[base + q * S] += v;
            mine = -1;
          }
      }
      id[base + k * S] = mine;
      p[base + k * S] = mine >= 0 ? v : 0.f;
    }
    tea[row] = make_float2(h, live ? 1.f : 0.f);
  }
  const unsigned long long m = __ballot(live);
  if ((threadIdx.x & 63) == 0 && m) atomicAdd(count, __popcll(m));
}

extern "C" int accunet_distill_teacher(const void* idx, int idx64, const void* top, int top_dt,
                                       const float* rest, int* id, float* p, float* tea, int* count,
                                       long B, long S, int V, int K, float T, void* stream) {
  if (B <= 0 || S <= 0 || V <= 0 || V > DT_MAX_V || K <= 0 || K > DT_MAX_K) return ACC_EBADSHAPE;
  if (!idx || !top || !id || !p || !tea || !count || !(T > 0.f)) return ACC_EBADARG;
  const float c = (float)(DT_LOG2E / T);
  hipStream_t st = (hipStream_t)stream;
  auto go = [&](auto itag) {
    using IT = decltype(itag);
    return with_dt(top_dt, [&](auto tag) {
      using TT = decltype(tag);
      if (S == 1)
        hipLaunchKernelGGL((distill_teacher_rows_kernel<IT, TT>), dim3((unsigned)((B + 3) / 4)),
                           dim3(256), 0, st, (const IT*)idx, (const TT*)top, rest, id, p,
                           (float2*)tea, count, B, V, K, c);
      else
        hipLaunchKernelGGL((distill_teacher_planes_kernel<IT, TT>),
                           dim3((unsigned)((B * S + 255) / 256)), dim3(256), 0, st, (const IT*)idx,
                           (const TT*)top, rest, id, p, (float2*)tea, count, B * S, S, V, K, c);
    });
  };
  const int rc = idx64 ? go((long long)0) : go((int)0);
  if (rc != ACC_OK) return rc;
  return hipGetLastError() == hipSuccess ? ACC_OK : ACC_ELAUNCH;
}

// ------------------------------------------------------- classes on the channel axis
// One thread a pixel, the classes four at a time (loads of one class are contiguous over
// the pixels). Listed classes are marked in a bitmap of the thread's own in LDS.
#define DTP_MAX_V 1024
template <typename T, bool REST>
__global__ void __launch_bounds__(256)
distill_planes_fwd_kernel(const T* __restrict__ z, const float* __restrict__ rest,
                          const int* __restrict__ id, const float* __restrict__ p,
                          const float2* __restrict__ tea, float4* __restrict__ state,
                          float* __restrict__ rowloss, double* __restrict__ part, long N, long S,
                          int V, int K, float c, float scale) {
  extern __shared__ unsigned mask[];  // [words][256], REST only
  __shared__ double red[4];
  const int t = threadIdx.x;
  const long row = blockIdx.x * 256L + t;
  float loss = 0.f;
  if (row < N) {
    const long b = row / S, s0 = row - b * S;
    const float2 te = tea[row];
    if (te.y == 0.f) {
      state[row] = make_float4(0.f, 0.f, 0.f, DT_EMPTY);
    } else {
      const T* zr = z + b * V * S + s0;
      const long kb = b * K * S + s0;
      if (REST) {
        const int words = (V + 31) / 32;
        for (int w = 0; w < words; ++w) mask[w * 256 + t] = 0u;
        for (int k = 0; k < K; ++k) {
          const int j = id[kb + k * S];
          if (j >= 0) mask[(j >> 5) * 256 + t] |= 1u << (j & 31);
        }
      }
      float m = -INFINITY, s = 0.f;
      for (int j0 = 0; j0 < V; j0 += 4) {
        float v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = j0 + u < V ? ld1(zr + (long)(j0 + u) * S) : -INFINITY;
        if (REST) {
          const unsigned bits = mask[(j0 >> 5) * 256 + t] >> (j0 & 31);
#pragma unroll
          for (int u = 0; u < 4; ++u) v[u] = (bits >> u) & 1u ? -INFINITY : v[u];
        }
        const float mv = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
        if (mv > m) {
          s *= dt_rescale(m, mv, c);
          m = mv;
        }
        const float ref = dt_ref(m, c);
#pragma unroll
        for (int u = 0; u < 4; ++u) s += dt_exp2(__builtin_fmaf(v[u], c, -ref));
      }
      const float mr = m, sr = s;
      if (REST)
        for (int k = 0; k < K; ++k) {
          const int j = id[kb + k * S];
          if (j >= 0) dt_join(m, s, ld1(zr + (long)j * S), 1.f, c);
        }
      const float r = REST ? rest[row] : 0.f;
      const DtRow o = dt_row_state(m, s, mr, sr, r, REST, c);
      float dot = 0.f;
      for (int k = 0; k < K; ++k) {
        const int j = id[kb + k * S];
        const float pk = p[kb + k * S];
        if (j >= 0 && !(pk == 0.f))
          dot += pk * (__builtin_fmaf(ld1(zr + (long)j * S), c, -o.M) - o.log2S);
      }
      if (REST && !(r == 0.f)) dot += r * ((dt_ref(mr, c) - o.M) + log2f(sr) - o.log2S);
      state[row] = o.state;
      loss = scale * (te.x - dot);
    }
    if (rowloss) rowloss[row] = loss;
  }
  double d = (double)loss;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) d += __shfl_xor(d, o);
  if ((t & 63) == 0) red[t >> 6] = d;
  __syncthreads();
  if (t == 0) part[blockIdx.x] = ((red[0] + red[1]) + red[2]) + red[3];
}

template <typename T>
__global__ void __launch_bounds__(256)
distill_planes_bwd_kernel(const T* __restrict__ z, const int* __restrict__ id,
                          const float* __restrict__ p, const float4* __restrict__ state,
                          T* __restrict__ dz, long N, long S, int V, int K, float c, DtScale g) {
  const long row = blockIdx.x * 256L + threadIdx.x;
  if (row >= N) return;
  const long b = row / S, s0 = row - b * S;
  const T* zr = z + b * V * S + s0;
  T* dr = dz + b * V * S + s0;
  const float4 st = state[row];
  if (st.w == DT_EMPTY) {
    for (int j = 0; j < V; ++j) st1(dr + (long)j * S, 0.f);
    return;
  }
  const float gs = dt_scale(g, row), cu = st.y * gs;
  for (int j0 = 0; j0 < V; j0 += 4) {
    float v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = j0 + u < V ? ld1(zr + (long)(j0 + u) * S) : 0.f;
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (j0 + u < V) st1(dr + (long)(j0 + u) * S, dt_exp2(__builtin_fmaf(v[u], c, -st.x)) * cu);
  }
  const long kb = b * K * S + s0;
  for (int k = 0; k < K; ++k) {
    const int j = id[kb + k * S];
    if (j >= 0)
      st1(dr + (long)j * S, gs * (dt_exp2(__builtin_fmaf(ld1(zr + (long)j * S), c, -st.z)) * st.w -
                                  p[kb + k * S]));
  }
}

// ----------------------------------------------------------------- the loss of all rows
// out = scale * sum(part) / rows counted (mean); one block, fp64, a fixed order
__global__ void __launch_bounds__(1024)
distill_loss_kernel(const double* __restrict__ part, long n, const int* count, float* out) {
  __shared__ double red[16];
  double a[4] = {0.0, 0.0, 0.0, 0.0};
  long i = threadIdx.x;
  for (; i + 3L * 1024 < n; i += 4L * 1024)
#pragma unroll
    for (int u = 0; u < 4; ++u) a[u] += part[i + 1024L * u];
  for (; i < n; i += 1024) a[0] += part[i];
  double v = (a[0] + a[1]) + (a[2] + a[3]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
#pragma unroll
    for (int w = 0; w < 16; ++w) t += red[w];
    if (count) t /= (double)max(*count, 1);
    out[0] = (float)t;
  }
}

extern "C" int accunet_distill_loss(const double* part, long n, const int* count, float* out,
                                    void* stream) {
  if (n <= 0) return ACC_EBADSHAPE;
  if (!part || !out) return ACC_EBADARG;
  hipLaunchKernelGGL(distill_loss_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, part, n,
                     count, out);
  return hipGetLastError() == hipSuccess ? ACC_OK : ACC_ELAUNCH;
}

extern "C" int accunet_distill_planes_fwd(const void* z, const float* rest, const int* id,
                                          const float* p, const float* tea, float* state,
                                          float* rowloss, double* part, long B, long S, int V,
                                          int K, float T, float weight, int dt, void* stream) {
  if (B <= 0 || S <= 0 || V <= 0 || V > DTP_MAX_V || K <= 0 || K > DT_MAX_K) return ACC_EBADSHAPE;
  if (!z || !id || !p || !tea || !state || !part || !(T > 0.f)) return ACC_EBADARG;
  const float c = (float)(DT_LOG2E / T);
  const float scale = weight * T * T * DT_LN2;
  const dim3 grid((unsigned)((B * S + 255) / 256));
  const int rc = with_dt(dt, [&](auto tag) {
    using Z = decltype(tag);
    if (rest)
      hipLaunchKernelGGL((distill_planes_fwd_kernel<Z, true>), grid, dim3(256),
                         (V + 31) / 32 * 1024, (hipStream_t)stream, (const Z*)z, rest, id, p,
                         (const float2*)tea, (float4*)state, rowloss, part, B * S, S, V, K, c, scale);
    else
      hipLaunchKernelGGL((distill_planes_fwd_kernel<Z, false>), grid, dim3(256), 0,
                         (hipStream_t)stream, (const Z*)z, rest, id, p, (const float2*)tea,
                         (float4*)state, rowloss, part, B * S, S, V, K, c, scale);
  });
  if (rc != ACC_OK) return rc;
  return hipGetLastError() == hipSuccess ? ACC_OK : ACC_ELAUNCH;
}

extern "C" int accunet_distill_planes_bwd(const void* z, const int* id, const float* p,
                                          const float* state, const float* up, int up_rows,
                                          const int* count, void* dz, long B, long S, int V, int K,
                                          float T, float weight, int dt, void* stream) {
  if (B <= 0 || S <= 0 || V <= 0 || V > DTP_MAX_V || K <= 0 || K > DT_MAX_K) return ACC_EBADSHAPE;
  if (!z || !id || !p || !state || !dz || !(T > 0.f)) return ACC_EBADARG;
  const DtScale g = {up, up_rows, count, weight * T};
  const int rc = with_dt(dt, [&](auto tag) {
    using Z = decltype(tag);
    hipLaunchKernelGGL(distill_planes_bwd_kernel<Z>, dim3((unsigned)((B * S + 255) / 256)),
                       dim3(256), 0, (hipStream_t)stream, (const Z*)z, id, p, (const float4*)state,
                       (Z*)dz, B * S, S, V, K, (float)(DT_LOG2E / T), g);
  });
  if (rc != ACC_OK) return rc;
  return hipGetLastError() == hipSuccess ? ACC_OK : ACC_ELAUNCH;
}
