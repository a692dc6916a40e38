// The 8-bit linear layer's forward and backward as one call each (formats in fp8.h): the
// quantisers and products behind one another on the stream, scratch in one block.
#include "fp8.h"

namespace {
struct Carve {
  char* base;
  size_t used = 0;
  template <typename T>
  T* take(size_t bytes) {
    T* p = reinterpret_cast<T*>(base + used);
    used += (bytes + 255) / 256 * 256;
    return p;
  }
};
struct Blocks {
  unsigned char *q = nullptr, *s = nullptr;
};
Blocks blocks(Carve& c, long R, long C) {
  Blocks b;
  b.q = c.take<unsigned char>((size_t)R * fp8_pad(C));
  b.s = c.take<unsigned char>((size_t)R * fp8_scale_pitch(C));
  return b;
}

// kept for the backward: the transposed x (the weight's gradient) and weight (x's)
struct Save {
  Blocks xt, wt;
  size_t bytes;
};
Save save_of(char* base, long M, long N, long K, bool need_w, bool need_wt) {
  Carve c{base};
  Save s;
  if (need_w) s.xt = blocks(c, K, M);
  if (need_wt) s.wt = blocks(c, K, N);
  s.bytes = c.used;
  return s;
}
struct Forward {
  Blocks xq, wq;
  float* slab;
  size_t bytes;
};
Forward forward_of(char* base, long M, long N, long K, bool own_w) {
  Carve c{base};
  Forward f;
  f.xq = blocks(c, M, K);
  if (own_w) f.wq = blocks(c, N, K);
  f.slab = c.take<float>(fp8_gemm_elems(M, N, K) * 4);
  f.bytes = c.used;
  return f;
}
struct Backward {
  Blocks rows, cols;
  float *sum, *slab;
  size_t bytes;
};
Backward backward_of(char* base, long M, long N, long K, bool dx, bool dw, bool db) {
  Carve c{base};
  Backward b;
  // the bias alone needs no quantised matrix, but shares the pass that makes one
  if (dx || !dw) b.rows = blocks(c, M, N);
  if (dw) b.cols = blocks(c, N, M);
  b.sum = db ? c.take<float>(fp8_sum_elems(M, (int)N) * 4) : nullptr;
  const size_t nx = dx ? fp8_gemm_elems(M, K, N) : 0, nw = dw ? fp8_gemm_elems(N, K, M) : 0;
  b.slab = c.take<float>((nx > nw ? nx : nw) * 4);  // one product after the other
  b.bytes = c.used;
  return b;
}
bool aligned(const void* p, unsigned to) { return ((uintptr_t)p & (to - 1)) == 0; }
}  // namespace

extern "C" size_t accunet_fp8_linear_save_bytes(long M, long N, long K, int need_w, int need_wt) {
  if (fp8_check(M, K, N, ACC_F32) != ACC_OK) return 0;
  return save_of(nullptr, M, N, K, need_w != 0, need_wt != 0).bytes;
}
extern "C" size_t accunet_fp8_linear_ws_bytes(long M, long N, long K, int own_w) {
  if (fp8_check(M, K, N, ACC_F32) != ACC_OK) return 0;
  return forward_of(nullptr, M, N, K, own_w != 0).bytes;
}
extern "C" size_t accunet_fp8_linear_bwd_ws_bytes(long M, long N, long K, int dx, int dw, int db) {
  if (fp8_check(M, K, N, ACC_F32) != ACC_OK) return 0;
  return backward_of(nullptr, M, N, K, dx != 0, dw != 0, db != 0).bytes;
}

extern "C" int accunet_fp8_linear_fwd(const void* x, const float* w, const void* wq,
                                      const void* wqs, const float* bias, void* y, int need_w,
                                      int need_wt, void* save, size_t save_bytes, void* ws,
                                      size_t ws_bytes, long M, long N, long K, int dt,
                                      void* stream) {
  const int rc = fp8_check(M, K, N, dt);
  if (rc != ACC_OK) return rc;
  if (!x || !y || !ws || (w != nullptr) == (wq != nullptr) || (wq != nullptr) != (wqs != nullptr) ||
      (need_wt && !w))
    return ACC_EBADARG;
  if (!aligned(wq, 16) || !aligned(wqs, 4) || !aligned(ws, 256)) return ACC_EBADARG;
  if ((need_w || need_wt) && (!save || !aligned(save, 256))) return ACC_EBADARG;
  const Save keep = save_of((char*)save, M, N, K, need_w != 0, need_wt != 0);
  const Forward f = forward_of((char*)ws, M, N, K, w != nullptr);
  if (keep.bytes > save_bytes || f.bytes > ws_bytes) return ACC_EBADARG;
  hipStream_t st = (hipStream_t)stream;
  const unsigned char *b = (const unsigned char*)wq, *sb = (const unsigned char*)wqs;
  if (w) {
    fp8_quantize(w, ACC_F32, true, f.wq.q, f.wq.s, keep.wt.q, keep.wt.s, nullptr, nullptr, N,
                 (int)K, st);
    b = f.wq.q;
    sb = f.wq.s;
  }
  if (M <= FP8_TOKENS && !need_w) {
    fp8_token(x, b, sb, bias, y, dt, (int)M, (int)N, (int)K, st);
  } else {
    fp8_quantize(x, dt, false, f.xq.q, f.xq.s, keep.xt.q, keep.xt.s, nullptr, nullptr, M, (int)K, st);
    fp8_gemm(f.xq.q, f.xq.s, b, sb, bias, y, dt, f.slab, M, N, K, st);
  }
  return hipGetLastError() == hipSuccess ? ACC_OK : ACC_ELAUNCH;
}

extern "C" int accunet_fp8_linear_bwd(const void* dy, const void* save, int need_w, int need_wt,
                                      const void* wt, const void* wts, void* dx, float* dw,
                                      float* db, void* ws, size_t ws_bytes, long M, long N, long K,
                                      int dt, void* stream) {
  const int rc = fp8_check(M, K, N, dt);
  if (rc != ACC_OK) return rc;
  if (!dy || !ws || (!dx && !dw && !db) || (dw && !need_w) || ((dw || need_wt) && !save))
    return ACC_EBADARG;
  if (dx && !need_wt && (!wt || !wts)) return ACC_EBADARG;
  if (!aligned(save, 256) || !aligned(ws, 256) || !aligned(wt, 16) || !aligned(wts, 4))
    return ACC_EBADARG;
  const Save keep = save_of((char*)const_cast<void*>(save), M, N, K, need_w != 0, need_wt != 0);
  const Backward g = backward_of((char*)ws, M, N, K, dx, dw, db);
  if (g.bytes > ws_bytes) return ACC_EBADARG;
  hipStream_t st = (hipStream_t)stream;
  fp8_quantize(dy, dt, false, g.rows.q, g.rows.s, g.cols.q, g.cols.s, db, g.sum, M, (int)N, st);
  if (dx)
    fp8_gemm(g.rows.q, g.rows.s, need_wt ? keep.wt.q : (const unsigned char*)wt,
             need_wt ? keep.wt.s : (const unsigned char*)wts, nullptr, dx, dt, g.slab, M, K, N, st);
  if (dw)
    fp8_gemm(g.cols.q, g.cols.s, keep.xt.q, keep.xt.s, nullptr, dw, ACC_F32, g.slab, N, K, M, st);
  return hipGetLastError() == hipSuccess ? ACC_OK : ACC_ELAUNCH;
}
