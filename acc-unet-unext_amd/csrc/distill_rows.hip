// Distillation with the classes last (z [R][V]); mathematics and row state in distill.h.
//
// A row is a run of 16-byte vectors from the aligned address at or below its first class;
// its first and last vector may be partial (an odd V puts rows at any address) and are then
// read and written class by class. Rows up to DTR_WAVE_V classes take one wave each, longer
// ones blocks of 256 threads, several blocks a row where the rows alone do not fill the
// card. With a remaining mass the listed classes are kept out of the sum by a byte of marks
// per vector in LDS (one read per vector, nearly always zero).
#include <type_traits>

#include "distill.h"

#define DTR_WAVE_V 2048
#define DTR_CHUNK 16384  // vectors whose marks are held at once

template <typename T>
struct DtVec;
template <>
struct DtVec<float> {
  static constexpr int N = 4;
  static ACC_DEV void ld(const float* p, float (&v)[4]) {
    const float4 q = ld4(p);
    v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
  }
  static ACC_DEV void st(float* p, const float (&v)[4]) { st4(p, make_float4(v[0], v[1], v[2], v[3])); }
};
template <>
struct DtVec<bf16_t> {
  static constexpr int N = 8;
  static ACC_DEV void ld(const bf16_t* p, float (&v)[8]) {
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    v[0] = bflo(q.x); v[1] = bfhi(q.x); v[2] = bflo(q.y); v[3] = bfhi(q.y);
    v[4] = bflo(q.z); v[5] = bfhi(q.z); v[6] = bflo(q.w); v[7] = bfhi(q.w);
  }
  static ACC_DEV void st(bf16_t* p, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]),
                                              pack_bf2(v[4], v[5]), pack_bf2(v[6], v[7]));
  }
};

// vector q of the row at z (V classes, `off` elements past the aligned address): classes
// outside the row read as -inf
template <typename T>
ACC_DEV void dt_load(const T* z, int off, int V, int q, float (&v)[DtVec<T>::N]) {
  constexpr int N = DtVec<T>::N;
  const int j = q * N - off;
  if (j >= 0 && j + N <= V) {
    DtVec<T>::ld(z + j, v);
  } else {
#pragma unroll
    for (int u = 0; u < N; ++u) v[u] = j + u >= 0 && j + u < V ? ld1(z + j + u) : -INFINITY;
  }
}
template <typename T>
ACC_DEV int dt_offset(const T* p) { return (int)(((uintptr_t)p & 15) / sizeof(T)); }

// (m, s) over vectors [q0, q1) of a row, by threads t of NT; `mark`: DTR_CHUNK bytes
template <typename T, bool REST, int NT>
ACC_DEV void dt_stream(const T* z, int off, int V, int q0, int q1, const int* id, int K, int t,
                       unsigned* mark, float c, float& m, float& s) {
  constexpr int N = DtVec<T>::N;
  constexpr int U = 4;
  auto sync = [&]() {
    if constexpr (NT > 64) __syncthreads();
    else dt_wave_lds();
  };
  for (int qc = q0; qc < q1; qc += DTR_CHUNK) {
    const int qe = min(q1, qc + DTR_CHUNK);
    if (REST) {
      sync();
      for (int w = t; w < (qe - qc + 3) / 4; w += NT) mark[w] = 0u;
      sync();
      for (int k = t; k < K; k += NT) {
        const int j = id[k];
        const int q = (j + off) / N - qc;
        if (j >= 0 && q >= 0 && q < qe - qc)
          atomicOr(&mark[q >> 2], 1u << ((q & 3) * 8 + (j + off) % N));
      }
      sync();
    }
    for (int q = qc + t; q < qe; q += NT * U) {
      float v[U][N];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (q + u * NT < qe) dt_load(z, off, V, q + u * NT, v[u]);
        else
#pragma unroll
          for (int e = 0; e < N; ++e) v[u][e] = -INFINITY;
      if (REST) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (q + u * NT >= qe) continue;
          const unsigned bits = reinterpret_cast<const unsigned char*>(mark)[q + u * NT - qc];
          if (bits)
#pragma unroll
            for (int e = 0; e < N; ++e) v[u][e] = (bits >> e) & 1u ? -INFINITY : v[u][e];
        }
      }
      float mv = v[0][0];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < N; ++e) mv = fmaxf(mv, v[u][e]);
      if (mv > m) {
        s *= dt_rescale(m, mv, c);
        m = mv;
      }
      const float ref = dt_ref(m, c);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < N; ++e) s += dt_exp2(__builtin_fmaf(v[u][e], c, -ref));
    }
  }
}

// One wave: the row's state and loss from (m, s) over the streamed classes.
template <typename T>
ACC_DEV void dt_finish_row(const T* z, const int* id, const float* p, int K, float m, float s,
                           float rest, bool has_rest, float h, float c, float scale, int lane,
                           float4* state, float* rowloss, double* part) {
  const float mr = m, sr = s;
  if (has_rest) {
    float lm = -INFINITY, ls = 0.f;
    for (int k = lane; k < K; k += 64)
      if (id[k] >= 0) dt_join(lm, ls, ld1(z + id[k]), 1.f, c);
    dt_wave_join(lm, ls, c);
    dt_join(m, s, lm, ls, c);
  }
  const DtRow o = dt_row_state(m, s, mr, sr, rest, has_rest, c);
  float dot = 0.f;
  for (int k = lane; k < K; k += 64) {
    const float pk = p[k];
    if (id[k] >= 0 && !(pk == 0.f))
      dot += pk * (__builtin_fmaf(ld1(z + id[k]), c, -o.M) - o.log2S);
  }
  dot = dt_wave_sum(dot);
  if (has_rest && !(rest == 0.f)) dot += rest * ((dt_ref(mr, c) - o.M) + log2f(sr) - o.log2S);
  if (lane == 0) {
    const float loss = scale * (h - dot);
    *state = o.state;
    if (rowloss) *rowloss = loss;
    *part = (double)loss;
  }
}

ACC_DEV void dt_empty_row(int lane, float4* state, float* rowloss, double* part) {
  if (lane == 0) {
    *state = make_float4(0.f, 0.f, 0.f, DT_EMPTY);
    if (rowloss) *rowloss = 0.f;
    *part = 0.0;
  }
}

// short rows: one wave a row, everything in one pass
template <typename T, bool REST>
__global__ void __launch_bounds__(256)
distill_rows_wave_kernel(const T* __restrict__ z, const float* __restrict__ rest,
                         const int* __restrict__ id, const float* __restrict__ p,
                         const float2* __restrict__ tea, float4* __restrict__ state,
                         float* __restrict__ rowloss, double* __restrict__ part, long R, int V,
                         int K, float c, float scale) {
  __shared__ unsigned mark[4][(DTR_WAVE_V / 4 + 2 + 3) / 4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long row = blockIdx.x * 4L + wave;
  if (row >= R) return;
  float* rl = rowloss ? rowloss + row : nullptr;
  const float2 te = tea[row];
  if (te.y == 0.f) {
    dt_empty_row(lane, state + row, rl, part + row);
    return;
  }
  const T* zr = z + row * V;
  const int off = dt_offset(zr);
  float m = -INFINITY, s = 0.f;
  dt_stream<T, REST, 64>(zr, off, V, 0, (off + V + DtVec<T>::N - 1) / DtVec<T>::N, id + row * K, K,
                         lane, mark[wave], c, m, s);
  dt_wave_join(m, s, c);
  dt_finish_row(zr, id + row * K, p + row * K, K, m, s, REST ? rest[row] : 0.f, REST, te.x, c,
                scale, lane, state + row, rl, part + row);
}

// long rows: block (x, row) streams the x-th run of vectors into ms[row][x]
template <typename T, bool REST>
__global__ void __launch_bounds__(256)
distill_rows_sum_kernel(const T* __restrict__ z, const int* __restrict__ id,
                        const float2* __restrict__ tea, float2* __restrict__ ms, int V, int K,
                        int run, float c) {
  __shared__ unsigned mark[REST ? DTR_CHUNK / 4 : 1];
  __shared__ float2 red[4];
  const long r = blockIdx.x;
  if (tea[r].y == 0.f) return;
  const T* zr = z + r * V;
  const int off = dt_offset(zr);
  const int nq = (off + V + DtVec<T>::N - 1) / DtVec<T>::N;
  const int q0 = min(nq, (int)blockIdx.y * run), q1 = min(nq, q0 + run);
  float m = -INFINITY, s = 0.f;
  dt_stream<T, REST, 256>(zr, off, V, q0, q1, id + r * K, K, threadIdx.x, mark, c, m, s);
  dt_wave_join(m, s, c);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = make_float2(m, s);
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 4; ++w) dt_join(m, s, red[w].x, red[w].y, c);
    ms[r * gridDim.y + blockIdx.y] = make_float2(m, s);
  }
}

template <typename T, bool REST>
__global__ void __launch_bounds__(256)
distill_rows_finish_kernel(const T* __restrict__ z, const float* __restrict__ rest,
                           const int* __restrict__ id, const float* __restrict__ p,
                           const float2* __restrict__ tea, const float2* __restrict__ ms, int runs,
                           float4* __restrict__ state, float* __restrict__ rowloss,
                           double* __restrict__ part, long R, int V, int K, float c, float scale) {
  const int lane = threadIdx.x & 63;
  const long row = blockIdx.x * 4L + (threadIdx.x >> 6);
  if (row >= R) return;
  float* rl = rowloss ? rowloss + row : nullptr;
  const float2 te = tea[row];
  if (te.y == 0.f) {
    dt_empty_row(lane, state + row, rl, part + row);
    return;
  }
  float m = -INFINITY, s = 0.f;
  for (int i = lane; i < runs; i += 64) {
    const float2 v = ms[row * runs + i];
    dt_join(m, s, v.x, v.y, c);
  }
  dt_wave_join(m, s, c);
  dt_finish_row(z + row * V, id + row * K, p + row * K, K, m, s, REST ? rest[row] : 0.f, REST,
                te.x, c, scale, lane, state + row, rl, part + row);
}

// Gradient: every class as not listed, then, behind a barrier (the block's own stores),
// the listed classes of this run over it. NT threads a row, run vectors each.
template <typename T, int NT>
__global__ void __launch_bounds__(256)
distill_rows_bwd_kernel(const T* __restrict__ z, const int* __restrict__ id,
                        const float* __restrict__ p, const float4* __restrict__ state,
                        T* __restrict__ dz, long R, int V, int K, int run, float c, DtScale g) {
  constexpr int N = DtVec<T>::N;
  const int t = NT == 64 ? (threadIdx.x & 63) : threadIdx.x;
  const long row = NT == 64 ? blockIdx.x * 4L + (threadIdx.x >> 6) : (long)blockIdx.x;
  if (NT == 64 && row >= R) return;
  const T* zr = z + row * V;
  T* dr = dz + row * V;
  const int off = dt_offset(zr);  // dz has z's alignment (checked by the host)
  const int nq = (off + V + N - 1) / N;
  const int q0 = min(nq, (int)blockIdx.y * run), q1 = min(nq, q0 + run);
  const float4 st = state[row];
  const bool live = !(st.w == DT_EMPTY);
  const float gs = live ? dt_scale(g, row) : 0.f, cu = live ? st.y * gs : 0.f;
  for (int q = q0 + t; q < q1; q += NT) {
    float v[N];
    if (live) {
      dt_load(zr, off, V, q, v);
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] = dt_exp2(__builtin_fmaf(v[e], c, -st.x)) * cu;
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] = 0.f;
    }
    const int j = q * N - off;
    if (j >= 0 && j + N <= V) {
      DtVec<T>::st(dr + j, v);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (j + e >= 0 && j + e < V) st1(dr + j + e, v[e]);
    }
  }
  if (!live) return;
  __threadfence_block();
  if (NT > 64) __syncthreads();
  else __builtin_amdgcn_s_waitcnt(0);  // one wave: its stores are done before the next ones
  for (int k = t; k < K; k += NT) {
    const int j = id[row * K + k];
    const int q = (j + off) / N;
    if (j >= 0 && q >= q0 && q < q1)
      st1(dr + j, gs * (dt_exp2(__builtin_fmaf(ld1(zr + j), c, -st.z)) * st.w - p[row * K + k]));
  }
}

// runs of vectors a long row is cut into: enough blocks for the card, 1024 vectors at least
static int dt_runs(long R, int V, int dt) {
  const int n = dt == ACC_F32 ? 4 : 8;
  const long nq = ((long)V + n - 1) / n + 1;
  const long want = (2048 + R - 1) / R, most = (nq + 1023) / 1024;
  return (int)max(1L, min(want, most));
}
static int dt_run_len(int runs, int V, int dt) {
  const int n = dt == ACC_F32 ? 4 : 8;
  return ceil_div(((long)V + n - 1) / n + 1, runs);
}

extern "C" size_t accunet_distill_rows_ws_elems(long R, int V, int dt) {
  if (R <= 0 || V <= 0 || V <= DTR_WAVE_V) return 0;
  return (size_t)R * dt_runs(R, V, dt) * 2;
}

extern "C" int accunet_distill_rows_fwd(const void* z, const float* rest, const int* id,
                                        const float* p, const float* tea, float* state,
                                        float* rowloss, double* part, float* ws, size_t ws_elems,
                                        long R, int V, int K, float T, float weight, int dt,
                                        void* stream) {
  if (R <= 0 || R > 0x7fffffffL || V <= 0 || V > DT_MAX_V || K <= 0 || K > DT_MAX_K) return ACC_EBADSHAPE;
  if (!z || !id || !p || !tea || !state || !part || !(T > 0.f)) return ACC_EBADARG;
  if (ws_elems < accunet_distill_rows_ws_elems(R, V, dt)) return ACC_EBADARG;
  const float c = (float)(DT_LOG2E / T);
  const float scale = weight * T * T * DT_LN2;
  hipStream_t st = (hipStream_t)stream;
  const int rc = with_dt(dt, [&](auto tag) {
    using Z = decltype(tag);
    auto go = [&](auto rtag) {
      constexpr bool REST = decltype(rtag)::value;
      const dim3 g4((unsigned)((R + 3) / 4));
      if (V <= DTR_WAVE_V) {
        hipLaunchKernelGGL((distill_rows_wave_kernel<Z, REST>), g4, dim3(256), 0, st, (const Z*)z,
                           rest, id, p, (const float2*)tea, (float4*)state, rowloss, part, R, V, K,
                           c, scale);
        return;
      }
      const int runs = dt_runs(R, V, dt);
      hipLaunchKernelGGL((distill_rows_sum_kernel<Z, REST>), dim3((unsigned)R, runs), dim3(256), 0,
                         st, (const Z*)z, id, (const float2*)tea, (float2*)ws, V, K,
                         dt_run_len(runs, V, dt), c);
      hipLaunchKernelGGL((distill_rows_finish_kernel<Z, REST>), g4, dim3(256), 0, st, (const Z*)z,
                         rest, id, p, (const float2*)tea, (const float2*)ws, runs, (float4*)state,
                         rowloss, part, R, V, K, c, scale);
    };
    if (rest) go(std::true_type{});
    else go(std::false_type{});
  });
  if (rc != ACC_OK) return rc;
  return hipGetLastError() == hipSuccess ? ACC_OK : ACC_ELAUNCH;
}

extern "C" int accunet_distill_rows_bwd(const void* z, const int* id, const float* p,
                                        const float* state, const float* up, int up_rows,
                                        const int* count, void* dz, long R, int V, int K, float T,
                                        float weight, int dt, void* stream) {
  if (R <= 0 || R > 0x7fffffffL || V <= 0 || V > DT_MAX_V || K <= 0 || K > DT_MAX_K) return ACC_EBADSHAPE;
  if (!z || !id || !p || !state || !dz || !(T > 0.f)) return ACC_EBADARG;
  if (((uintptr_t)z ^ (uintptr_t)dz) & 15) return ACC_EBADARG;
  const float c = (float)(DT_LOG2E / T);
  const DtScale g = {up, up_rows, count, weight * T};
  const int rc = with_dt(dt, [&](auto tag) {
    using Z = decltype(tag);
    if (V <= DTR_WAVE_V) {
      hipLaunchKernelGGL((distill_rows_bwd_kernel<Z, 64>), dim3((unsigned)((R + 3) / 4)), dim3(256),
                         0, (hipStream_t)stream, (const Z*)z, id, p, (const float4*)state, (Z*)dz,
                         R, V, K, dt_run_len(1, V, dt), c, g);
    } else {
      const int runs = dt_runs(R, V, dt);
      hipLaunchKernelGGL((distill_rows_bwd_kernel<Z, 256>), dim3((unsigned)R, runs), dim3(256), 0,
                         (hipStream_t)stream, (const Z*)z, id, p, (const float4*)state, (Z*)dz, R,
                         V, K, dt_run_len(runs, V, dt), c, g);
    }
  });
  if (rc != ACC_OK) return rc;
  return hipGetLastError() == hipSuccess ? ACC_OK : ACC_ELAUNCH;
}
