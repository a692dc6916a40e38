// Distillation from a teacher's top logits; mathematics in distill.h. This file: the
// teacher's pass, the loss over the rows, and the layout with the classes on the channel
// axis of an image (z [B][V][S]). Rows with the classes last: distill_rows.hip.
#include <type_traits>

#include "distill.h"

// ------------------------------------------------------------------ the teacher's entries
// p and the entries that count, each class once: id = the class at its first entry (p the
// sum over its entries), -1 elsewhere. tea[row] = (sum p log2 p + rest log2 rest, 1 or 0).
// cnt[block]: the rows of the block that have an entry.
//
// One wave a row, entries k = lane + 64 i. Bound by latency: K^2 / 64 comparisons a lane.
template <typename IT, typename TT>
__global__ void __launch_bounds__(256)
distill_teacher_rows_kernel(const IT* __restrict__ idx, const TT* __restrict__ top,
                            const float* __restrict__ rest, int* __restrict__ id,
                            float* __restrict__ p, float2* __restrict__ tea, int* __restrict__ cnt,
                            long R, int V, int K, float c) {
  __shared__ int alive[4];
  __shared__ int sid[4][DT_MAX_K];
  __shared__ float sp[4][DT_MAX_K];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long row = blockIdx.x * 4L + wave;
  const bool in = row < R;
  const int NI = in ? (K + 63) / 64 : 0;
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
  const float ref = dt_ref(mx);
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < DT_MAX_K / 64; ++i)
    if (my[i] >= 0) sum += dt_term(a[i], ref, c);
  sum = dt_wave_sum(sum);
  const float r = in && live && rest ? rest[row] : 0.f;
  const float keep = 1.f - r;
#pragma unroll
  for (int i = 0; i < DT_MAX_K / 64; ++i) {
    const int k = i * 64 + lane;
    if (i >= NI || k >= K) continue;
    sid[wave][k] = my[i];
    sp[wave][k] = my[i] >= 0 && live ? keep * (dt_term(a[i], ref, c) / sum) : 0.f;
  }
  float h = 0.f;  // of the classes' masses, not of their entries'
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
    if (first) h += dt_plogp(v);
  }
  h = dt_wave_sum(h) + dt_plogp(r);
  if (lane == 0) {
    if (in) tea[row] = make_float2(h, live ? 1.f : 0.f);
    alive[wave] = in && live ? 1 : 0;
  }
  __syncthreads();
  if (threadIdx.x == 0) cnt[blockIdx.x] = alive[0] + alive[1] + alive[2] + alive[3];
}

// Classes on the channel axis: idx, top [B][K][S], one thread a pixel; the entries of a
// pixel are re-read from the cache for each of the passes.
template <typename IT, typename TT>
__global__ void __launch_bounds__(256)
distill_teacher_planes_kernel(const IT* __restrict__ idx, const TT* __restrict__ top,
                              const float* __restrict__ rest, int* __restrict__ id,
                              float* __restrict__ p, float2* __restrict__ tea, int* __restrict__ cnt, long N,
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
    const float ref = dt_ref(mx);
    float sum = 0.f;
    for (int k = 0; k < K; ++k) {
      const long long j = (long long)idx[base + k * S];
      if (j >= 0 && j < V) sum += dt_term(ld1(top + base + k * S), ref, c);
    }
    const float r = live && rest ? rest[row] : 0.f;
    const float keep = 1.f - r;
    float h = dt_plogp(r);
    for (int k = 0; k < K; ++k) {
      const long long j = (long long)idx[base + k * S];
      int mine = -1;
      float v = 0.f;
      if (live && j >= 0 && j < V) {
        mine = (int)j;
        v = keep * (dt_term(ld1(top + base + k * S), ref, c) / sum);
        for (int q = 0; q < k; ++q)  // listed before: its mass joins the first entry
          if (mine >= 0 && id[base + q * S] == mine) {
            const float was = p[base + q * S];
            p[base + q * S] = was + v;
            h += dt_plogp(was + v) - dt_plogp(was);
            mine = -1;
          }
        if (mine >= 0) h += dt_plogp(v);
      }
      id[base + k * S] = mine;
      p[base + k * S] = mine >= 0 ? v : 0.f;
    }
    tea[row] = make_float2(h, live ? 1.f : 0.f);
  }
  const int m = __syncthreads_count(live);
  if (threadIdx.x == 0) cnt[blockIdx.x] = m;
}

// count = sum of the n values of cnt
__global__ void __launch_bounds__(1024)
distill_count_kernel(const int* __restrict__ cnt, int n, int* __restrict__ count) {
  __shared__ int red[16];
  int v = 0;
  for (int i = threadIdx.x; i < n; i += 1024) v += cnt[i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    int t = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) t += red[w];
    *count = t;
  }
}

// ------------------------------------------------------- classes on the channel axis
// One thread a pixel, the classes four at a time (loads of one class are contiguous over
// the pixels). Up to DTP_TAB_V classes a thread keeps a table of its own in LDS, p of a
// listed class and -1 elsewhere, and writes the gradient class by class in one coalesced
// pass; scattered over the listed classes afterwards (many classes, marked in a bitmap) the
// kernel took 62 us instead of 39 (16 x 12 x 224^2 fp32, 4 entries).
#define DTP_TAB_V 32
#define DTP_MAX_V 1024
ACC_DEV void dtp_table(float* tab, long S, int V, int K, const int* id, const float* p) {
  for (int j = 0; j < V; ++j) tab[j * 256] = -1.f;
  for (int k = 0; k < K; ++k) {
    const int j = id[k * S];
    if (j >= 0) tab[j * 256] = p[k * S];
  }
}
// The gradient of a pixel; tab: the thread's table (TAB), else every class as not listed and
// the listed ones over it.
template <typename T, bool TAB>
ACC_DEV void dtp_gradient(const T* zr, T* dr, long S, int V, int K, const int* id, const float* p,
                          const float* tab, const float4& st, float c, float gs) {
  const float cu = st.y * gs;
  for (int j0 = 0; j0 < V; j0 += 4) {
    float v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = j0 + u < V ? ld1(zr + (long)(j0 + u) * S) : 0.f;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (j0 + u >= V) continue;
      const float pj = TAB ? tab[(j0 + u) * 256] : -1.f;
      const bool free = pj == -1.f;
      const float e = dt_term(v[u], free ? st.x : st.z, c);
      st1(dr + (long)(j0 + u) * S, free ? e * cu : gs * (e * st.w - pj));
    }
  }
  if (TAB) return;
  for (int k = 0; k < K; ++k) {
    const int j = id[k * S];
    if (j >= 0)
      st1(dr + (long)j * S, gs * (dt_term(ld1(zr + (long)j * S), st.z, c) * st.w - p[k * S]));
  }
}
template <typename T>
ACC_DEV void dtp_zero(T* dr, long S, int V) {
  for (int j = 0; j < V; ++j) st1(dr + (long)j * S, 0.f);
}

// dz (or null): the gradient for an upstream of 1 too, from the logits still in the cache
template <typename T, bool REST, bool TAB>
__global__ void __launch_bounds__(256)
distill_planes_fwd_kernel(const DtArgs a, const DtScale g) {
  extern __shared__ unsigned mask[];  // [words][256] of bits (REST), or the tables [V][256]
  __shared__ double red[4];
  const int t = threadIdx.x;
  const long row = blockIdx.x * 256L + t, S = a.S;
  const int V = a.V, K = a.K;
  const float c = a.c;
  float loss = 0.f;
  if (row < a.rows) {
    const long b = row / S, s0 = row - b * S;
    const T* zr = (const T*)a.z + b * V * S + s0;
    T* dr = a.dz ? (T*)a.dz + b * V * S + s0 : nullptr;
    const long kb = b * K * S + s0;
    const float2 te = a.tea[row];
    if (te.y == 0.f) {
      a.state[row] = make_float4(0.f, 0.f, 0.f, DT_EMPTY);
      if (dr) dtp_zero(dr, S, V);
    } else {
      float* tab = reinterpret_cast<float*>(mask) + t;
      if (TAB) {
        dtp_table(tab, S, V, K, a.id + kb, a.p + kb);
      } else if (REST) {
        const int words = (V + 31) / 32;
        for (int w = 0; w < words; ++w) mask[w * 256 + t] = 0u;
        for (int k = 0; k < K; ++k) {
          const int j = a.id[kb + k * S];
          if (j >= 0) mask[(j >> 5) * 256 + t] |= 1u << (j & 31);
        }
      }
      float m = -INFINITY, s = 0.f;
      for (int j0 = 0; j0 < V; j0 += 4) {
        float v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = j0 + u < V ? ld1(zr + (long)(j0 + u) * S) : -INFINITY;
        if (REST && TAB) {
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (j0 + u < V && !(tab[(j0 + u) * 256] == -1.f)) v[u] = -INFINITY;
        } else if (REST) {
          const unsigned bits = mask[(j0 >> 5) * 256 + t] >> (j0 & 31);
#pragma unroll
          for (int u = 0; u < 4; ++u) v[u] = (bits >> u) & 1u ? -INFINITY : v[u];
        }
        const float mv = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
        if (mv > m) {
          s *= dt_rescale(m, mv, c);
          m = mv;
        }
        const float ref = dt_ref(m);
#pragma unroll
        for (int u = 0; u < 4; ++u) s += dt_term(v[u], ref, c);
      }
      const float mr = m, sr = s;
      if (REST)
        for (int k = 0; k < K; ++k) {
          const int j = a.id[kb + k * S];
          if (j >= 0) dt_join(m, s, ld1(zr + (long)j * S), 1.f, c);
        }
      const float r = REST ? a.rest[row] : 0.f;
      const DtRow o = dt_row_state(m, s, mr, sr, r, REST, c);
      float dot = 0.f;
      for (int k = 0; k < K; ++k) {
        const int j = a.id[kb + k * S];
        const float pk = a.p[kb + k * S];
        if (j >= 0 && !(pk == 0.f))
          dot += pk * dt_log2q(ld1(zr + (long)j * S), o, c);
      }
      if (REST && !(r == 0.f)) dot += r * dt_log2q_rest(mr, sr, o, c);
      a.state[row] = o.state;
      loss = a.scale * (te.x - dot);
      if (dr)
        dtp_gradient<T, TAB>(zr, dr, S, V, K, a.id + kb, a.p + kb, tab, o.state, c,
                             dt_scale(g, row));
    }
    if (a.none) a.loss[row] = loss;
  }
  if (t == 0 && a.applied) a.applied[blockIdx.x] = 1.f;
  double d = (double)loss;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) d += __shfl_xor(d, o);
  if ((t & 63) == 0) red[t >> 6] = d;
  __syncthreads();
  if (t == 0) a.part[blockIdx.x] = ((red[0] + red[1]) + red[2]) + red[3];
}

template <typename T, bool TAB>
__global__ void __launch_bounds__(256)
distill_planes_bwd_kernel(const DtArgs a, const DtScale g) {
  extern __shared__ unsigned mask[];  // the tables [V][256]
  const long row = blockIdx.x * 256L + threadIdx.x, S = a.S;
  if (a.applied) {  // dz holds the gradient for this upstream already?
    const float up = *g.up;
    const bool done = a.applied[blockIdx.x] == up;
    __syncthreads();
    if (done) return;
    if (threadIdx.x == 0) a.applied[blockIdx.x] = up;
  }
  if (row >= a.rows) return;
  const long b = row / S, s0 = row - b * S;
  const T* zr = (const T*)a.z + b * a.V * S + s0;
  T* dr = (T*)a.dz + b * a.V * S + s0;
  const long kb = b * a.K * S + s0;
  const float4 st = a.state[row];
  if (st.w == DT_EMPTY) {
    dtp_zero(dr, S, a.V);
    return;
  }
  float* tab = reinterpret_cast<float*>(mask) + threadIdx.x;
  if (TAB) dtp_table(tab, S, a.V, a.K, a.id + kb, a.p + kb);
  dtp_gradient<T, TAB>(zr, dr, S, a.V, a.K, a.id + kb, a.p + kb, tab, st, a.c, dt_scale(g, row));
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

// ------------------------------------------------------------------------------- calls
static long dt_up16(long n) { return (n + 15) / 16 * 16; }
static bool dt_planes(long S) { return S > 1; }
// kept for the backward: state, applied, count, id, p
static long dt_carve_save(DtArgs& a, char* base) {
  long o = 0;
  auto take = [&](auto*& ptr, long bytes) {
    ptr = reinterpret_cast<std::remove_reference_t<decltype(ptr)>>(base + o);
    o = dt_up16(o + bytes);
  };
  take(a.state, a.rows * 16);
  take(a.applied, a.rows * 4);
  take(a.count, 16);
  take(a.id, a.rows * a.K * 4);
  take(a.p, a.rows * a.K * 4);
  return o;
}
static long dt_carve_ws(DtArgs& a, char* base, int dt) {
  long o = 0;
  auto take = [&](auto*& ptr, long bytes) {
    ptr = reinterpret_cast<std::remove_reference_t<decltype(ptr)>>(base + o);
    o = dt_up16(o + bytes);
  };
  take(a.tea, a.rows * 8);
  take(a.part, a.rows * 8);
  take(a.cnt, a.rows * 4);
  take(a.ms, dt_planes(a.S) ? 0 : a.rows * dt_rows_runs(a.rows, a.V, dt) * 8);
  return o;
}
static int dt_check(long B, long S, int V, int K, float T) {
  if (B <= 0 || S <= 0 || B * S > 0x7fffffffL || V <= 0 || V > DT_MAX_V || K <= 0 || K > DT_MAX_K)
    return ACC_EBADSHAPE;
  if (dt_planes(S) && V > DTP_MAX_V) return ACC_EBADSHAPE;
  if (!dt_planes(S) && B > (V <= DTR_WAVE_V ? DTR_WAVE_ROWS : DTR_LONG_ROWS)) return ACC_EBADSHAPE;
  return T >= DT_MIN_T && T <= DT_MAX_T ? ACC_OK : ACC_EBADARG;
}
static DtArgs dt_args(long B, long S, int V, int K, float T, float weight) {
  DtArgs a = {};
  a.rows = B * S; a.S = S; a.V = V; a.K = K;
  a.T = T; a.c = (float)(DT_LOG2E / T); a.weight = weight;
  a.scale = weight * T * T * DT_LN2;
  return a;
}

extern "C" size_t accunet_distill_save_bytes(long B, long S, int V, int K) {
  if (dt_check(B, S, V, K, 1.f) != ACC_OK) return 0;
  DtArgs a = dt_args(B, S, V, K, 1.f, 1.f);
  return (size_t)dt_carve_save(a, nullptr);
}
extern "C" size_t accunet_distill_ws_bytes(long B, long S, int V, int K, int dt) {
  if (dt_check(B, S, V, K, 1.f) != ACC_OK) return 0;
  DtArgs a = dt_args(B, S, V, K, 1.f, 1.f);
  return (size_t)dt_carve_ws(a, nullptr, dt);
}
// the capture that `stream` is part of, 0 outside one (the null stream is never captured)
extern "C" long long accunet_stream_capture_id(void* stream) {
  if (!stream) return 0;
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (hipStreamGetCaptureInfo((hipStream_t)stream, &status, &id) != hipSuccess) {
    (void)hipGetLastError();
    return -1;
  }
  return status == hipStreamCaptureStatusActive ? (long long)id : 0;
}
// one block a row (or pixel), so the gradient can follow the sum in the same kernel
extern "C" int accunet_distill_fused(long B, long S, int V, int dt) {
  return dt_planes(S) || dt_rows_runs(B, V, dt) == 1;
}

extern "C" int accunet_distill_fwd(const void* z, const void* idx, int idx64, const void* top,
                                   int top_dt, const float* rest, float* loss, int reduction,
                                   void* dz, void* save, size_t save_bytes, void* ws,
                                   size_t ws_bytes, long B, long S, int V, int K, float T,
                                   float weight, int dt, void* stream) {
  const int rc = dt_check(B, S, V, K, T);
  if (rc != ACC_OK) return rc;
  if (!z || !idx || !top || !loss || !save || !ws || reduction < 0 || reduction > 2 ||
      (dt != ACC_F32 && dt != ACC_BF16) || (top_dt != ACC_F32 && top_dt != ACC_BF16))
    return ACC_EBADARG;
  if (((uintptr_t)save | (uintptr_t)ws | (uintptr_t)z) & 15) return ACC_EBADARG;
  if (dz && (reduction == 0 || !accunet_distill_fused(B, S, V, dt) ||
             (((uintptr_t)z ^ (uintptr_t)dz) & 15)))
    return ACC_EBADARG;
  DtArgs a = dt_args(B, S, V, K, T, weight);
  if ((size_t)dt_carve_save(a, (char*)save) > save_bytes) return ACC_EBADARG;
  if ((size_t)dt_carve_ws(a, (char*)ws, dt) > ws_bytes) return ACC_EBADARG;
  a.z = z; a.rest = rest; a.loss = loss; a.dz = dz;
  a.none = reduction == 0;
  a.mean = reduction == 2;
  if (!dz) a.applied = nullptr;
  hipStream_t st = (hipStream_t)stream;
  const bool planes = dt_planes(S);
  const unsigned pix = (unsigned)((a.rows + 255) / 256), quad = (unsigned)((a.rows + 3) / 4);
  const int nb = (int)(planes ? pix : quad);
  // one block counts straight into its place
  int* cnt = nb == 1 ? a.count : a.cnt;
  auto teacher = [&](auto itag) {
    using IT = decltype(itag);
    with_dt(top_dt, [&](auto tag) {
      using TT = decltype(tag);
      if (planes)
        hipLaunchKernelGGL((distill_teacher_planes_kernel<IT, TT>), dim3(pix), dim3(256), 0, st,
                           (const IT*)idx, (const TT*)top, rest, a.id, a.p, a.tea, cnt, a.rows, S,
                           V, K, a.c);
      else
        hipLaunchKernelGGL((distill_teacher_rows_kernel<IT, TT>), dim3(quad), dim3(256), 0, st,
                           (const IT*)idx, (const TT*)top, rest, a.id, a.p, a.tea, cnt, a.rows, V,
                           K, a.c);
    });
  };
  if (idx64) teacher((long long)0);
  else teacher((int)0);
  if (nb > 1 && a.mean)
    hipLaunchKernelGGL(distill_count_kernel, dim3(1), dim3(1024), 0, st, a.cnt, nb, a.count);
  if (planes) {
    const DtScale g = {nullptr, 0, a.mean ? a.count : nullptr, weight * T};
    with_dt(dt, [&](auto tag) {
      using Z = decltype(tag);
      auto go = [&](auto kernel, int lds) {
        hipLaunchKernelGGL(kernel, dim3(pix), dim3(256), lds, st, a, g);
      };
      const int words = (V + 31) / 32 * 1024;
      if (V <= DTP_TAB_V) {
        if (rest) go(distill_planes_fwd_kernel<Z, true, true>, V * 1024);
        else go(distill_planes_fwd_kernel<Z, false, true>, V * 1024);
      } else {
        if (rest) go(distill_planes_fwd_kernel<Z, true, false>, words);
        else go(distill_planes_fwd_kernel<Z, false, false>, 0);
      }
    });
  } else {
    dt_rows_forward(a, dt, st);
  }
  // four rows at most in one block write the loss themselves
  const bool inside =
      !planes && nb == 1 && (V <= DTR_WAVE_V || dt_rows_runs(a.rows, V, dt) > 1);
  if (!a.none && !inside)
    hipLaunchKernelGGL(distill_loss_kernel, dim3(1), dim3(1024), 0, st, a.part,
                       planes ? (long)pix : a.rows, a.mean ? a.count : nullptr, loss);
  return hipGetLastError() == hipSuccess ? ACC_OK : ACC_ELAUNCH;
}

extern "C" int accunet_distill_bwd(const void* z, void* save, size_t save_bytes, const float* up,
                                   int reduction, int held, void* dz, long B, long S, int V, int K,
                                   float T, float weight, int dt, void* stream) {
  const int rc = dt_check(B, S, V, K, T);
  if (rc != ACC_OK) return rc;
  if (!z || !save || !up || !dz || reduction < 0 || reduction > 2 || (held && reduction == 0) ||
      (dt != ACC_F32 && dt != ACC_BF16))
    return ACC_EBADARG;
  if ((uintptr_t)save & 15 || (((uintptr_t)z ^ (uintptr_t)dz) & 15)) return ACC_EBADARG;
  DtArgs a = dt_args(B, S, V, K, T, weight);
  if ((size_t)dt_carve_save(a, (char*)save) > save_bytes) return ACC_EBADARG;
  a.z = z; a.dz = dz;
  if (!held) a.applied = nullptr;
  const DtScale g = {up, reduction == 0, reduction == 2 ? a.count : nullptr, weight * T};
  hipStream_t st = (hipStream_t)stream;
  if (dt_planes(S))
    with_dt(dt, [&](auto tag) {
      using Z = decltype(tag);
      const dim3 grid((unsigned)((a.rows + 255) / 256));
      if (V <= DTP_TAB_V)
        hipLaunchKernelGGL((distill_planes_bwd_kernel<Z, true>), grid, dim3(256), V * 1024, st, a, g);
      else
        hipLaunchKernelGGL((distill_planes_bwd_kernel<Z, false>), grid, dim3(256), 0, st, a, g);
    });
  else
    dt_rows_backward(a, g, dt, st);
  return hipGetLastError() == hipSuccess ? ACC_OK : ACC_ELAUNCH;
}
