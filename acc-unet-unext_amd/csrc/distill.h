// Distillation from a teacher's top logits (distill.hip, distill_rows.hip).
//
// Row i: student logits z[0..V), the teacher's entries (idx_k, t_k), k < K, an optional
// mass `rest` of the teacher outside them, temperature T.
//   p_k   = (1 - rest) * softmax(t / T)_k over the entries with 0 <= idx_k < V; entries of one
//           class are one entry with their sum from here on
//   q     = softmax(z / T) over all V classes, q_rest = sum of q over classes not listed
//   loss  = T^2 * [ sum_k p_k (log p_k - log q_idx_k) + rest (log rest - log q_rest) ]
//   dloss/dz_j = T * (q_j - p_j)                  listed
//              = T * (q_j - rest * q_j / q_rest)  not listed
// A row without a valid entry (or whose valid t are all -inf) has loss 0 and gradient 0
// and is not counted by the mean.
//
// Arithmetic is in base 2: with c = log2(e) / T a softmax term is 2^((z - m)*c), a difference,
// a product and one v_exp_f32. Of the difference, not z*c - m*c: each thread and block sums
// relative to its own m, and what rounding m*c loses grows with the logits' offset from zero
// and differs from one to the next; and the lowest value of a type times c may pass fp32's.
// q_rest is summed over the classes not listed, never as 1 - sum of the others, and a row's
// state keeps it relative to the largest such class, so it may be far below fp32's range:
//   not listed: dz = 2^((z - mu)*c) * cu,  cu = 2^((mu - m)*c) / S - rest / S_rest
//   listed:     dz = 2^((z - m)*c) / S - p
#pragma once
#include "common.h"

#define DT_MAX_K 256
#define DT_MAX_V (1 << 30)
// T^2 and log2(e) / T are normal fp32 numbers
#define DT_MIN_T 0x1p-60f
#define DT_MAX_T 0x1p60f
#define DT_LN2 0.69314718055994531f
#define DT_LOG2E 1.4426950408889634

// one row's state between the passes
//   x: mu, y: cu, z: m (logits), w: 1/S, or DT_EMPTY for a row that does not count
#define DT_EMPTY (-1.f)

ACC_DEV float dt_exp2(float v) { return __builtin_amdgcn_exp2f(v); }
// 2^((m - M) * c), 1 where both are the same infinity
ACC_DEV float dt_rescale(float m, float M, float c) { return m == M ? 1.f : dt_exp2((m - M) * c); }
// m as the reference of terms; 0 where no class is left (every term is 2^-inf then)
ACC_DEV float dt_ref(float m) { return m == -INFINITY ? 0.f : m; }
// 2^((z - ref) * c)
ACC_DEV float dt_term(float z, float ref, float c) { return dt_exp2((z - ref) * c); }
// p log2 p
ACC_DEV float dt_plogp(float p) { return p == 0.f ? 0.f : p * log2f(p); }
// (m, s) joined with (m2, s2)
ACC_DEV void dt_join(float& m, float& s, float m2, float s2, float c) {
  const float M = fmaxf(m, m2);
  s = s * dt_rescale(m, M, c) + s2 * dt_rescale(m2, M, c);
  m = M;
}
// LDS written by one lane of a wave and read by another of the same wave
ACC_DEV void dt_wave_lds() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
ACC_DEV float dt_wave_sum(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
ACC_DEV float dt_wave_max(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}
ACC_DEV void dt_wave_join(float& m, float& s, float c) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float m2 = __shfl_xor(m, o), s2 = __shfl_xor(s, o);
    dt_join(m, s, m2, s2, c);
  }
  // partners round their joint sum differently: every lane takes the first lane's
  m = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(m)));
  s = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(s)));
}

// The row's state and loss (base 2, before T^2 ln 2) once (m, s) over the streamed classes,
// and over the listed ones if they were left out (REST), are known. `dot` is the caller's
// sum over listed entries of p * log2 q.
struct DtRow {
  float4 state;
  float M, log2S;
};
ACC_DEV DtRow dt_row_state(float m, float s, float mr, float sr, float rest, bool has_rest, float c) {
  DtRow o;
  const float ref = dt_ref(m);
  o.M = ref;
  o.log2S = log2f(s);
  o.state.z = ref;
  o.state.w = 1.f / s;
  o.state.x = ref;
  o.state.y = o.state.w;
  if (has_rest) {
    o.state.x = dt_ref(mr);
    o.state.y = sr > 0.f ? dt_rescale(mr, m, c) / s - rest / sr : (sr == 0.f ? 0.f : sr);
  }
  return o;
}
// log2 of q of a class with logit z, and of all classes not listed
ACC_DEV float dt_log2q(float z, const DtRow& o, float c) {
  return __builtin_fmaf(z - o.M, c, -o.log2S);
}
ACC_DEV float dt_log2q_rest(float mr, float sr, const DtRow& o, float c) {
  return sr == 0.f ? -INFINITY : __builtin_fmaf(dt_ref(mr) - o.M, c, log2f(sr) - o.log2S);
}

// the step from a row's sums to its gradient: weight * T * upstream / rows counted
struct DtScale {
  const float* up;      // upstream gradient: one value, or one per row (up_rows); null: 1
  int up_rows;
  const int* count;     // rows counted (mean), or null
  float k;              // weight * T
};
ACC_DEV float dt_scale(const DtScale& g, long row) {
  float v = g.k;
  if (g.up) v *= g.up[g.up_rows ? row : 0];
  if (g.count) v /= (float)max(*g.count, 1);
  return v;
}

// One call's arguments. `rows` = B * S; S = 1 with the classes last.
struct DtArgs {
  const void* z;
  const float* rest;
  // kept for the backward
  float4* state;      // [rows]
  float* applied;     // upstream gradient that dz holds: [rows], or one a block of 256 pixels
  int* count;         // rows counted
  int* id;            // [rows][K]
  float* p;           // [rows][K]
  // scratch of the forward
  float2* tea;        // [rows]
  double* part;       // partial losses
  int* cnt;           // rows counted by each block of the teacher's pass
  float2* ms;         // [rows][runs]
  float* loss;        // the loss, or one a row (none)
  void* dz;
  long rows, S;
  int V, K;
  float T, c, scale, weight;
  int none, mean;
};

// rows with the classes last (distill_rows.hip); up to DTR_WAVE_V classes a wave has a row
// in registers (512 vectors of 4 fp32 at most, partial ones at both ends included)
#define DTR_WAVE_V 2032
// a launch holds fewer than 2^32 threads: 64 a row, 256 a long one (the 512 and 1024 of rows
// above 64 KB and 128 KB end at 550 GB of logits)
#define DTR_WAVE_ROWS ((1L << 26) - 4)
#define DTR_LONG_ROWS ((1L << 24) - 1)
int dt_rows_runs(long R, int V, int dt);
void dt_rows_forward(const DtArgs& a, int dt, hipStream_t st);
void dt_rows_backward(const DtArgs& a, const DtScale& g, int dt, hipStream_t st);
