// Distillation with the classes last (z [R][V]); mathematics and row state in distill.h.
//
// A row is a run of 16-byte vectors from the aligned address at or below its first class;
// its first and last vector may be partial (an odd V puts rows at any address) and are then
// read and written class by class. Rows up to DTR_WAVE_V classes take one wave each, longer
// ones blocks of 256 threads, several blocks a row where the rows alone do not fill the
// card. Where one block has a whole row, the gradient for an upstream of 1 is written by the
// same kernel (short rows: from registers).
// With a remaining mass the listed classes are kept out of the sum by a byte of marks
// per vector in LDS (one read per vector, nearly always zero).
#include <type_traits>

#include "distill.h"

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
  template <bool STREAM>
  static ACC_DEV void st(float* p, const float (&v)[4]) {
    const float4 q = make_float4(v[0], v[1], v[2], v[3]);
    if (STREAM) st4_nt(p, q);
    else st4(p, q);
  }
};
template <>
struct DtVec<bf16_t> {
  static constexpr int N = 8;
  static ACC_DEV void ld(const bf16_t* p, float (&v)[8]) {
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    v[0] = bflo(q.x); v[1] = bfhi(q.x); v[2] = bflo(q.y); v[3] = bfhi(q.y);
    v[4] = bflo(q.z); v[5] = bfhi(q.z); v[6] = bflo(q.w); v[7] = bfhi(q.w);
  }
  template <bool STREAM>
  static ACC_DEV void st(bf16_t* p, const float (&v)[8]) {
    const acc_u32x4 q = {pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]), pack_bf2(v[4], v[5]),
                         pack_bf2(v[6], v[7])};
    if (STREAM) __builtin_nontemporal_store(q, reinterpret_cast<acc_u32x4*>(p));
    else *reinterpret_cast<acc_u32x4*>(p) = q;
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
// A row's whole vectors: [lo, hi) of its nq, and its aligned base. What a wave reads between
// them needs no look at the row's ends.
template <typename T>
struct DtRun {
  const acc_u32x4* base;
  int lo, hi;
  ACC_DEV DtRun(const T* z, int off, int V) {
    constexpr int N = DtVec<T>::N;
    base = reinterpret_cast<const acc_u32x4*>(z - off);
    lo = off ? 1 : 0;
    hi = (off + V) / N;
  }
  // vectors q, q + step, .. (n of them) of every lane of the wave, q0 the first lane's q
  ACC_DEV bool whole(int q0, int step, int n, int end) const {
    return q0 >= lo && q0 + (n - 1) * step + 64 <= min(hi, end);
  }
};
template <typename T>
ACC_DEV float dt_get(const acc_u32x4& w, int e) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(w[e]);
  else return e & 1 ? bfhi(w[e >> 1]) : bflo(w[e >> 1]);
}
template <typename T>
ACC_DEV int dt_offset(const T* p) { return (int)(((uintptr_t)p & 15) / sizeof(T)); }

// marks of the listed classes of vectors [qc, qe), one byte a vector, by threads t of NT
template <int N, int NT>
ACC_DEV void dt_marks(unsigned* mark, int qc, int qe, const int* id, int K, int off, int t) {
  auto sync = [&]() {
    if constexpr (NT > 64) __syncthreads();
    else dt_wave_lds();
  };
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
ACC_DEV unsigned dt_mark(const unsigned* mark, int q) {
  return reinterpret_cast<const unsigned char*>(mark)[q];
}

// gradient vector q of a row: whole, or class by class at the row's ends and around listed
// classes (`bits`), which others write
template <typename T, bool STREAM>
ACC_DEV void dt_put(T* dr, int off, int V, int q, unsigned bits, const float (&v)[DtVec<T>::N]) {
  constexpr int N = DtVec<T>::N;
  const int j = q * N - off;
  if (j >= 0 && j + N <= V && bits == 0u) {
    DtVec<T>::template st<STREAM>(dr + j, v);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (j + e >= 0 && j + e < V && !((bits >> e) & 1u)) st1(dr + j + e, v[e]);
  }
}

// (m, s) over vectors [q0, q1) of a row, by threads t of NT; `mark`: DTR_CHUNK bytes
template <typename T, bool REST, int NT>
ACC_DEV void dt_stream(const T* z, int off, int V, int q0, int q1, const int* id, int K, int t,
                       unsigned* mark, float c, float& m, float& s) {
  constexpr int N = DtVec<T>::N;
  constexpr int U = sizeof(T) == 4 ? 4 : 2;  // vectors in flight a thread
  const DtRun<T> run(z, off, V);
  for (int qc = q0; qc < q1; qc += DTR_CHUNK) {
    const int qe = min(q1, qc + DTR_CHUNK);
    if (REST) dt_marks<N, NT>(mark, qc, qe, id, K, off, t);
    // sums U vectors, get(u, e) a class
    auto add = [&](auto get) {
      float mv = get(0, 0);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < N; ++e) mv = fmaxf(mv, get(u, e));
      if (mv > m) {
        s *= dt_rescale(m, mv, c);
        m = mv;
      }
      const float ref = dt_ref(m);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < N; ++e) s += dt_term(get(u, e), ref, c);
    };
    for (int q = qc + t; q < qe; q += NT * U) {
      if (run.whole(__builtin_amdgcn_readfirstlane(q), NT, U, qe)) {
        acc_u32x4 w[U];
        unsigned bits[U], any = 0u;
#pragma unroll
        for (int u = 0; u < U; ++u) w[u] = run.base[q + u * NT];
        if (REST)
#pragma unroll
          for (int u = 0; u < U; ++u) any |= bits[u] = dt_mark(mark, q + u * NT - qc);
        if (!REST || !__any(any)) {
          add([&](int u, int e) { return dt_get<T>(w[u], e); });
        } else {
          add([&](int u, int e) { return (bits[u] >> e) & 1u ? -INFINITY : dt_get<T>(w[u], e); });
        }
        continue;
      }
      float v[U][N];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (q + u * NT < qe) {
          dt_load(z, off, V, q + u * NT, v[u]);
          const unsigned bits = REST ? dt_mark(mark, q + u * NT - qc) : 0u;
          if (REST && bits)
#pragma unroll
            for (int e = 0; e < N; ++e) v[u][e] = (bits >> e) & 1u ? -INFINITY : v[u][e];
        } else {
#pragma unroll
          for (int e = 0; e < N; ++e) v[u][e] = -INFINITY;
        }
      }
      add([&](int u, int e) { return v[u][e]; });
    }
  }
}

// One wave: the row's state and loss from (m, s) over the streamed classes.
// zk(k): the logit of listed entry k.
template <typename F>
ACC_DEV float4 dt_finish_row(F zk, const int* id, const float* p, int K, float m, float s,
                           float rest, bool has_rest, float h, float c, float scale, int lane,
                           float4* state, float* rowloss, double* part) {
  const float mr = m, sr = s;
  if (has_rest) {
    float lm = -INFINITY, ls = 0.f;
    for (int k = lane; k < K; k += 64)
      if (id[k] >= 0) dt_join(lm, ls, zk(k), 1.f, c);
    dt_wave_join(lm, ls, c);
    dt_join(m, s, lm, ls, c);
  }
  const DtRow o = dt_row_state(m, s, mr, sr, rest, has_rest, c);
  float dot = 0.f;
  for (int k = lane; k < K; k += 64) {
    const float pk = p[k];
    if (id[k] >= 0 && !(pk == 0.f)) dot += pk * dt_log2q(zk(k), o, c);
  }
  dot = dt_wave_sum(dot);
  if (has_rest && !(rest == 0.f)) dot += rest * dt_log2q_rest(mr, sr, o, c);
  if (lane == 0) {
    const float loss = scale * (h - dot);
    *state = o.state;
    if (rowloss) *rowloss = loss;
    *part = (double)loss;
  }
  return o.state;
}

// One wave: a row that does not count.
ACC_DEV void dt_empty_row(int lane, float4* state, float* rowloss, double* part) {
  if (lane == 0) {
    *state = make_float4(0.f, 0.f, 0.f, DT_EMPTY);
    if (rowloss) *rowloss = 0.f;
    *part = 0.0;
  }
}

template <typename T>
ACC_DEV void dt_put_listed(const T* zr, T* dr, int j, float p, const float4& st, float c,
                           float gs) {
  st1(dr + j, gs * (dt_term(ld1(zr + j), st.z, c) * st.w - p));
}

// Gradient of vectors [q0, q1) of a row by threads t of NT: every class as not listed, then,
// behind a barrier, the listed classes over it. `dr` has z's alignment (checked by the host).
// STREAM: stored past the caches.
template <typename T, int NT, bool STREAM>
ACC_DEV void dt_gradient(const T* zr, T* dr, int off, int V, int q0, int q1, const int* id,
                         const float* p, int K, int t, const float4& st, float c, float gs) {
  constexpr int N = DtVec<T>::N;
  constexpr int U = sizeof(T) == 4 ? 4 : 2;
  const bool live = !(st.w == DT_EMPTY);
  const float cu = st.y * gs;
  for (int q = q0 + t; q < q1; q += NT * U) {
    float v[U][N];
    if (live) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (q + u * NT < q1) dt_load(zr, off, V, q + u * NT, v[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (q + u * NT >= q1) continue;
#pragma unroll
      for (int e = 0; e < N; ++e)
        v[u][e] = live ? dt_term(v[u][e], st.x, c) * cu : 0.f;
      dt_put<T, STREAM>(dr, off, V, q + u * NT, 0u, v[u]);
    }
  }
  if (!live) return;  // the same for the whole row
  __threadfence_block();
  if (NT > 64) __syncthreads();
  else __builtin_amdgcn_s_waitcnt(0);  // one wave: its stores are done before the next ones
  for (int k = t; k < K; k += NT) {
    const int j = id[k];
    const int q = (j + off) / N;
    if (j >= 0 && q >= q0 && q < q1) dt_put_listed(zr, dr, j, p[k], st, c, gs);
  }
}

// four rows at most (one block): their loss without another kernel
ACC_DEV void dt_small_loss(const DtArgs& a, double* red) {
  if (gridDim.x != 1 || a.none) return;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int w = 0; w < 4; ++w) t += w < a.rows ? red[w] : 0.0;
    if (a.mean) t /= (double)max(*a.count, 1);
    a.loss[0] = (float)t;
  }
}

// short rows: one wave a row, NQ vectors a lane in registers. The exponentials are relative
// to the largest streamed class, which is the gradient's reference too (mu), so each is
// computed once: dz = e * cu. 65536 x 2000 bf16 with 8 entries: 141-144
// us of 203 for the whole pass.
template <typename T, bool REST, int NQ>
__global__ void __launch_bounds__(256)
distill_rows_wave_kernel(const DtArgs a, const DtScale g) {
  constexpr int N = DtVec<T>::N;
  __shared__ unsigned mark[4][NQ * 16];
  __shared__ double red[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long row = blockIdx.x * 4L + wave;
  const int V = a.V, K = a.K;
  if (row < a.rows) {
    float* rl = a.none ? a.loss + row : nullptr;
    const float2 te = a.tea[row];
    const T* zr = (const T*)a.z + row * V;
    T* dr = (T*)a.dz + row * V;
    const int* id = a.id + row * K;
    const float* p = a.p + row * K;
    const int off = dt_offset(zr), nq = (off + V + N - 1) / N;
    if (te.y == 0.f) {
      dt_empty_row(lane, a.state + row, rl, &red[wave]);
      if (a.dz) {
        float v[N];
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = 0.f;
        for (int q = lane; q < nq; q += 64) dt_put<T, false>(dr, off, V, q, 0u, v);
      }
    } else {
      float v[NQ][N];
#pragma unroll
      for (int u = 0; u < NQ; ++u) {
#pragma unroll
        for (int e = 0; e < N; ++e) v[u][e] = -INFINITY;
        if (u * 64 + lane < nq) dt_load(zr, off, V, u * 64 + lane, v[u]);
      }
      if (REST || a.dz) dt_marks<N, 64>(mark[wave], 0, nq, id, K, off, lane);
      unsigned bits[NQ];
#pragma unroll
      for (int u = 0; u < NQ; ++u) {
        bits[u] = (REST || a.dz) && u * 64 + lane < nq ? dt_mark(mark[wave], u * 64 + lane) : 0u;
        if (REST && bits[u])
#pragma unroll
          for (int e = 0; e < N; ++e) v[u][e] = (bits[u] >> e) & 1u ? -INFINITY : v[u][e];
      }
      float m = v[0][0];
#pragma unroll
      for (int u = 0; u < NQ; ++u)
#pragma unroll
        for (int e = 0; e < N; ++e) m = fmaxf(m, v[u][e]);
      m = dt_wave_max(m);
      const float ref = dt_ref(m);
      float s = 0.f;
#pragma unroll
      for (int u = 0; u < NQ; ++u)
#pragma unroll
        for (int e = 0; e < N; ++e) {
          v[u][e] = dt_term(v[u][e], ref, a.c);
          s += v[u][e];
        }
      s = dt_wave_sum(s);
      const float4 st = dt_finish_row([&](int k) { return ld1(zr + id[k]); }, id, p, K, m, s,
                                      REST ? a.rest[row] : 0.f, REST, te.x, a.c, a.scale, lane,
                                      a.state + row, rl, &red[wave]);
      if (a.dz) {
        const float gs = dt_scale(g, row), cu = st.y * gs;
#pragma unroll
        for (int u = 0; u < NQ; ++u) {
          if (u * 64 + lane >= nq) continue;
#pragma unroll
          for (int e = 0; e < N; ++e) v[u][e] *= cu;
          dt_put<T, false>(dr, off, V, u * 64 + lane, bits[u], v[u]);
        }
        for (int k = lane; k < K; k += 64)
          if (id[k] >= 0) dt_put_listed(zr, dr, id[k], p[k], st, a.c, gs);
      }
    }
    if (lane == 0) {
      a.part[row] = red[wave];
      if (a.applied) a.applied[row] = 1.f;
    }
  }
  dt_small_loss(a, red);
}

// long rows, one block each: the sum, the row's loss and the gradient. The listed entries
// are fetched at the start, beside the stream, and marked in LDS for the whole row where it
// has at most DTR_CHUNK vectors: the gradient then goes around them and they are written
// without waiting for it.
// The gradient's second read of the row misses the L2 but not the last-level cache (4096 x
// 128000 bf16: 1.05 GB fetched from memory, 1.06 GB written), so two reads and a write cross
// the fabric: 3.15 GB in 476-518 us, 6.1-6.6 TB/s, what a copy reaches. Loads a step ahead
// (488-571 us) or the row from its end changed nothing. Held in registers instead (64 a
// thread for the row, one block a CU) it took 592-860 us: sums, barriers and stores of one
// row then stand one behind another on each CU.
template <typename T, bool REST, int NT, bool STREAM>
__global__ void __launch_bounds__(NT)
distill_rows_fused_kernel(const DtArgs a, const DtScale g) {
  constexpr int N = DtVec<T>::N;
  __shared__ unsigned mark[DTR_CHUNK / 4];
  __shared__ float2 red[NT / 64];
  __shared__ float4 rs;
  __shared__ int lid[DT_MAX_K];
  __shared__ float lp[DT_MAX_K], lz[DT_MAX_K];
  const long row = blockIdx.x;
  const int t = threadIdx.x, V = a.V, K = a.K;
  const T* zr = (const T*)a.z + row * V;
  T* dr = (T*)a.dz + row * V;
  const int off = dt_offset(zr), nq = (off + V + N - 1) / N;
  float* rl = a.none ? a.loss + row : nullptr;
  const float2 te = a.tea[row];
  if (t == 0 && a.applied) a.applied[row] = 1.f;
  if (te.y == 0.f) {
    dt_empty_row(t, a.state + row, rl, a.part + row);
    if (a.dz) {
      float v[N];
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] = 0.f;
      for (int q = t; q < nq; q += NT) dt_put<T, STREAM>(dr, off, V, q, 0u, v);
    }
    return;
  }
  int my = -1;  // K <= DT_MAX_K <= NT: an entry a thread
  float mp = 0.f, mz = 0.f;
  if (t < K) {
    my = a.id[row * K + t];
    mp = a.p[row * K + t];
    mz = my >= 0 ? ld1(zr + my) : 0.f;
    lid[t] = my;
  }
  __syncthreads();
  const bool one = nq <= DTR_CHUNK;
  if (one && !REST && a.dz) dt_marks<N, NT>(mark, 0, nq, lid, K, off, t);
  float m = -INFINITY, s = 0.f;
  dt_stream<T, REST, NT>(zr, off, V, 0, nq, lid, K, t, mark, a.c, m, s);
  dt_wave_join(m, s, a.c);
  if ((t & 63) == 0) red[t >> 6] = make_float2(m, s);
  if (t < K) {
    lp[t] = mp;
    lz[t] = mz;
  }
  __syncthreads();
  if (t < 64) {
    m = red[0].x;
    s = red[0].y;
    for (int w = 1; w < NT / 64; ++w) dt_join(m, s, red[w].x, red[w].y, a.c);
    const float4 st = dt_finish_row([&](int k) { return lz[k]; }, lid, lp, K, m, s,
                                    REST ? a.rest[row] : 0.f, REST, te.x, a.c, a.scale, t,
                                    a.state + row, rl, a.part + row);
    if (t == 0) rs = st;
  }
  if (!a.dz) return;
  __syncthreads();
  const float4 st = rs;
  const float gs = dt_scale(g, row), cu = st.y * gs;
  if (!one) {
    dt_gradient<T, NT, STREAM>(zr, dr, off, V, 0, nq, lid, lp, K, t, st, a.c, gs);
    return;
  }
  if (my >= 0) dt_put_listed(zr, dr, my, mp, st, a.c, gs);
  constexpr int U = sizeof(T) == 4 ? 4 : 2;
  const DtRun<T> run(zr, off, V);
  for (int q = t; q < nq; q += NT * U) {
    if (run.whole(__builtin_amdgcn_readfirstlane(q), NT, U, nq)) {
      acc_u32x4 w[U];
      unsigned bits[U], any = 0u;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        w[u] = run.base[q + u * NT];
        any |= bits[u] = dt_mark(mark, q + u * NT);
      }
      const bool plain = !__any(any);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float v[N];
#pragma unroll
        for (int e = 0; e < N; ++e)
          v[e] = dt_term(dt_get<T>(w[u], e), st.x, a.c) * cu;
        if (plain) DtVec<T>::template st<STREAM>(dr + (q + u * NT) * N - off, v);
        else dt_put<T, STREAM>(dr, off, V, q + u * NT, bits[u], v);
      }
      continue;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (q + u * NT >= nq) continue;
      float v[N];
      dt_load(zr, off, V, q + u * NT, v);
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] = dt_term(v[e], st.x, a.c) * cu;
      dt_put<T, STREAM>(dr, off, V, q + u * NT, dt_mark(mark, q + u * NT), v);
    }
  }
}

// long rows, several blocks each: block (row, y) streams the y-th run into ms[row][y]
template <typename T, bool REST>
__global__ void __launch_bounds__(256)
distill_rows_sum_kernel(const DtArgs a, int run) {
  __shared__ unsigned mark[REST ? DTR_CHUNK / 4 : 1];
  __shared__ float2 red[4];
  const long r = blockIdx.x;
  const int V = a.V, K = a.K;
  if (a.tea[r].y == 0.f) return;
  const T* zr = (const T*)a.z + r * V;
  const int off = dt_offset(zr);
  const int nq = (off + V + DtVec<T>::N - 1) / DtVec<T>::N;
  const int q0 = min(nq, (int)blockIdx.y * run), q1 = min(nq, q0 + run);
  float m = -INFINITY, s = 0.f;
  dt_stream<T, REST, 256>(zr, off, V, q0, q1, a.id + r * K, K, threadIdx.x, mark, a.c, m, s);
  dt_wave_join(m, s, a.c);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = make_float2(m, s);
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 4; ++w) dt_join(m, s, red[w].x, red[w].y, a.c);
    a.ms[r * gridDim.y + blockIdx.y] = make_float2(m, s);
  }
}

template <typename T, bool REST>
__global__ void __launch_bounds__(256)
distill_rows_finish_kernel(const DtArgs a, int runs) {
  __shared__ double red[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long row = blockIdx.x * 4L + wave;
  const int V = a.V, K = a.K;
  if (row < a.rows) {
    float* rl = a.none ? a.loss + row : nullptr;
    const float2 te = a.tea[row];
    if (te.y == 0.f) {
      dt_empty_row(lane, a.state + row, rl, &red[wave]);
    } else {
      float m = -INFINITY, s = 0.f;
      for (int i = lane; i < runs; i += 64) {
        const float2 v = a.ms[row * runs + i];
        dt_join(m, s, v.x, v.y, a.c);
      }
      dt_wave_join(m, s, a.c);
      const T* zr = (const T*)a.z + row * V;
      const int* id = a.id + row * K;
      dt_finish_row([&](int k) { return ld1(zr + id[k]); }, id, a.p + row * K, K, m, s,
                    REST ? a.rest[row] : 0.f, REST, te.x, a.c, a.scale, lane, a.state + row, rl,
                    &red[wave]);
    }
    if (lane == 0) a.part[row] = red[wave];
  }
  dt_small_loss(a, red);
}

// The gradient from the kept state. NT threads a row (or a run of it).
template <typename T, int NT, bool STREAM>
__global__ void __launch_bounds__(256)
distill_rows_bwd_kernel(const DtArgs a, const DtScale g, int run) {
  const int t = NT == 64 ? (threadIdx.x & 63) : threadIdx.x;
  const long row = NT == 64 ? blockIdx.x * 4L + (threadIdx.x >> 6) : (long)blockIdx.x;
  if (NT == 64 && row >= a.rows) return;
  if (a.applied) {  // dz holds the gradient for this upstream already? (one run a row)
    const float up = *g.up;
    const bool done = a.applied[row] == up;
    if (NT > 64) __syncthreads();
    if (done) return;
    if (t == 0) a.applied[row] = up;
  }
  const int V = a.V, K = a.K;
  const T* zr = (const T*)a.z + row * V;
  const int off = dt_offset(zr);
  const int nq = (off + V + DtVec<T>::N - 1) / DtVec<T>::N;
  const int q0 = min(nq, (int)blockIdx.y * run), q1 = min(nq, q0 + run);
  const float4 st = a.state[row];
  dt_gradient<T, NT, STREAM>(zr, (T*)a.dz + row * V, off, V, q0, q1, a.id + row * K, a.p + row * K,
                             K, t, st, a.c, st.w == DT_EMPTY ? 0.f : dt_scale(g, row));
}

// runs of vectors a long row is cut into: one where the rows alone give every CU a block,
// else enough for 8 blocks a CU, 1024 vectors at least
int dt_rows_runs(long R, int V, int dt) {
  if (V <= DTR_WAVE_V || R >= 256) return 1;
  const int n = dt == ACC_F32 ? 4 : 8;
  const long nq = ((long)V + n - 1) / n + 1;
  const long want = (2048 + R - 1) / R, most = (nq + 1023) / 1024;
  return (int)max(1L, min(want, most));
}
static int dt_run_len(int runs, int V, int dt) {
  const int n = dt == ACC_F32 ? 4 : 8;
  return ceil_div(((long)V + n - 1) / n + 1, runs);
}
// gradients of 64 MB and more are streamed (the last-level cache holds 256 MB)
template <typename T>
static bool dt_large(const DtArgs& a) { return a.rows * a.V * (long)sizeof(T) >= (64L << 20); }

void dt_rows_forward(const DtArgs& a, int dt, hipStream_t st) {
  const DtScale g = {nullptr, 0, a.mean ? a.count : nullptr, a.weight * a.T};
  with_dt(dt, [&](auto tag) {
    using Z = decltype(tag);
    auto go = [&](auto rtag) {
      constexpr bool REST = decltype(rtag)::value;
      const dim3 g4((unsigned)((a.rows + 3) / 4));
      if (a.V <= DTR_WAVE_V) {
        // vectors a row has at most: a row of whole vectors starts at an aligned address
        constexpr int N = 16 / sizeof(Z);
        const int nq = (a.V + (a.V % N ? 2 * N - 2 : 0)) / N;
        auto nt = [&](auto tag2) {
          constexpr int NQ = decltype(tag2)::value;
          hipLaunchKernelGGL((distill_rows_wave_kernel<Z, REST, NQ>), g4, dim3(256), 0, st, a, g);
        };
        if (nq <= 64) nt(std::integral_constant<int, 1>{});
        else if (nq <= 128) nt(std::integral_constant<int, 2>{});
        else if (nq <= 256) nt(std::integral_constant<int, 4>{});
        else nt(std::integral_constant<int, 8>{});
        return;
      }
      const int runs = dt_rows_runs(a.rows, a.V, dt);
      if (runs == 1) {
        const dim3 grid((unsigned)a.rows);
        auto run = [&](auto ntag) {
          constexpr int NT = decltype(ntag)::value;
          if (dt_large<Z>(a))
            hipLaunchKernelGGL((distill_rows_fused_kernel<Z, REST, NT, true>), grid, dim3(NT), 0,
                               st, a, g);
          else
            hipLaunchKernelGGL((distill_rows_fused_kernel<Z, REST, NT, false>), grid, dim3(NT), 0,
                               st, a, g);
        };
        // threads a row: 2048 a CU then hold 512 KB of rows at most; 4096 x 128000 bf16 took
        // 522 us with 1024 threads, 555 with 512, 650 with 256, 16384 x 32000 took 617 us
        // with 1024, 531 with 512, 553 with 256
        const long bytes = (long)a.V * sizeof(Z);
        if (bytes <= (64 << 10)) run(std::integral_constant<int, 256>{});
        else if (bytes <= (128 << 10)) run(std::integral_constant<int, 512>{});
        else run(std::integral_constant<int, 1024>{});
        return;
      }
      hipLaunchKernelGGL((distill_rows_sum_kernel<Z, REST>), dim3((unsigned)a.rows, runs),
                         dim3(256), 0, st, a, dt_run_len(runs, a.V, dt));
      hipLaunchKernelGGL((distill_rows_finish_kernel<Z, REST>), g4, dim3(256), 0, st, a, runs);
    };
    if (a.rest) go(std::true_type{});
    else go(std::false_type{});
  });
}

void dt_rows_backward(const DtArgs& a, const DtScale& g, int dt, hipStream_t st) {
  with_dt(dt, [&](auto tag) {
    using Z = decltype(tag);
    const int runs = dt_rows_runs(a.rows, a.V, dt), len = dt_run_len(runs, a.V, dt);
    if (a.V <= DTR_WAVE_V)
      hipLaunchKernelGGL((distill_rows_bwd_kernel<Z, 64, false>),
                         dim3((unsigned)((a.rows + 3) / 4)), dim3(256), 0, st, a, g, len);
    else if (dt_large<Z>(a))
      hipLaunchKernelGGL((distill_rows_bwd_kernel<Z, 256, true>), dim3((unsigned)a.rows, runs),
                         dim3(256), 0, st, a, g, len);
    else
      hipLaunchKernelGGL((distill_rows_bwd_kernel<Z, 256, false>), dim3((unsigned)a.rows, runs),
                         dim3(256), 0, st, a, g, len);
  });
}
