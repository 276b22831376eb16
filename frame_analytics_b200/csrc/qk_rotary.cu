// Norm of query and key heads with the position rotation in the same pass.
//
// A head vector x of D components at position p becomes
//   r = 1 / sqrt(mean(x^2) + eps)
//   y = R_p (w o x r)
// where w is a learned weight (one of D components shared by the heads, one
// for each head, or none) and R_p turns the pairs of the first `rotary`
// components by the angles of row p of the cos / sin tables: pair i is
// (i, i + rotary/2), or (2i, 2i + 1) when `interleaved`.
//
// Backward, with g = R_p^T dy:
//   dx = r (w o g - x r mean(w o g o x r)),   dw = sum over rows of g o x r.
//
// r and the sums are float32 (float32 holds the mean of up to thousands of
// squares to a few 1e-7 relative; the outputs are rounded once).  The weight
// gradient is summed in two fixed-order passes without atomics, so it is the
// same bits on every run.
#include "common.cuh"

#include <algorithm>

#include "train.cuh"

namespace fab {

constexpr int kMaxDim = 512;

// One of the two operands (queries or keys).
struct QkSide {
  const void* x;   // [B, L, heads, D]
  const void* g;   // upstream gradient (backward)
  void* out;       // y, or dx
  const void* w;   // weight or null
  int heads;
  long long xb, xl, xh, gb, gl, gh, ob, ol, oh;
};

struct QkArgs {
  QkSide s[2];
  int B, L, D, half;          // half = rotary / 2
  int interleaved, per_head, w32;
  const float* cos_;
  const float* sin_;
  int table;
  const void* pos;
  int pos64;
  long long pos_b, pos_l;
  float eps, inv_d;
  double eps64;
  float* rstd;                // backward: 1 / rms of every row, for the weight pass
};

// Position of token (b, l); -1 when it is outside the tables.
__device__ __forceinline__ int qk_position(const QkArgs& a, int b, int l) {
  long long p = l;
  if (a.pos) {
    const long long o = b * a.pos_b + l * a.pos_l;
    p = a.pos64 ? __ldg(reinterpret_cast<const long long*>(a.pos) + o)
                : (long long)__ldg(reinterpret_cast<const int*>(a.pos) + o);
  }
  return p >= 0 && p < a.table ? (int)p : -1;
}

template <typename T>
__device__ __forceinline__ float qk_weight(const QkArgs& a, const QkSide& s, int head, int d) {
  if (!s.w) return 1.f;
  const long long o = (a.per_head ? (long long)head * a.D : 0) + d;
  return a.w32 ? __ldg(reinterpret_cast<const float*>(s.w) + o)
               : Ld<T>::f(ldro(reinterpret_cast<const T*>(s.w) + o));
}

// Row index -> side, token, head.  Rows are ordered token-major, queries
// before keys within a token.
struct QkRow { int side, b, l, head; };
__device__ __forceinline__ QkRow qk_row(const QkArgs& a, long long row) {
  const int per = a.s[0].heads + a.s[1].heads;
  const long long t = row / per;
  int h = (int)(row - t * per);
  QkRow r;
  r.b = (int)(t / a.L);
  r.l = (int)(t - (long long)r.b * a.L);
  r.side = h >= a.s[0].heads;
  r.head = r.side ? h - a.s[0].heads : h;
  return r;
}

// Any head size, alignment and stride: one warp for each head vector, one
// component at a time.  Component d < 2 half belongs to pair i with partner e.
__device__ __forceinline__ void qk_pair(const QkArgs& a, int d, int* pair, int* partner,
                                        bool* second) {
  if (a.interleaved) {
    *pair = d >> 1;
    *second = d & 1;
    *partner = d ^ 1;
  } else {
    *second = d >= a.half;
    *pair = *second ? d - a.half : d;
    *partner = *second ? d - a.half : d + a.half;
  }
}

template <typename T>
__global__ void __launch_bounds__(256) qk_fwd_any_kernel(const __grid_constant__ QkArgs a,
                                                         long long rows) {
  const int lane = threadIdx.x & 31;
  for (long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); row < rows;
       row += (long long)gridDim.x * 8) {
    const QkRow q = qk_row(a, row);
    const QkSide& s = a.s[q.side];
    const T* x = reinterpret_cast<const T*>(s.x) + q.b * s.xb + q.l * s.xl + q.head * s.xh;
    T* y = reinterpret_cast<T*>(s.out) + q.b * s.ob + q.l * s.ol + q.head * s.oh;
    float ss = 0.f;
    for (int d = lane; d < a.D; d += 32) {
      const float v = Ld<T>::f(x[d]);
      ss = fmaf(v, v, ss);
    }
    const float r = rsqrtf(fmaf(warp_sum(ss), a.inv_d, a.eps));
    const int p = qk_position(a, q.b, q.l);
    // a row may be normalised in place: every component is read before any is written
    float v[kMaxDim / 32];
#pragma unroll
    for (int k = 0; k < kMaxDim / 32; ++k) {
      const int d = k * 32 + lane;
      if (d < a.D) {
        v[k] = Ld<T>::f(x[d]) * r * qk_weight<T>(a, s, q.head, d);
        if (d < 2 * a.half) {
          int pair, e;
          bool second;
          qk_pair(a, d, &pair, &e, &second);
          const float u = Ld<T>::f(x[e]) * r * qk_weight<T>(a, s, q.head, e);
          const long long o = (long long)max(p, 0) * a.half + pair;
          const float c = __ldg(a.cos_ + o), sn = __ldg(a.sin_ + o);
          v[k] = second ? fmaf(v[k], c, u * sn) : fmaf(v[k], c, -u * sn);
        }
        if (p < 0) v[k] = __int_as_float(0x7fffffff);
      }
    }
    __syncwarp();
#pragma unroll
    for (int k = 0; k < kMaxDim / 32; ++k) {
      const int d = k * 32 + lane;
      if (d < a.D) y[d] = St<T>::v(v[k]);
    }
  }
}

// Double sums: in a short head the two terms of dx nearly cancel (with D = 1
// they differ by eps alone), and this kernel serves the odd sizes.
template <typename T>
__device__ __forceinline__ double qk_unrotated(const QkArgs& a, const T* g, int p, int d) {
  double v = Ld<T>::d(g[d]);
  if (d < 2 * a.half) {
    int pair, e;
    bool second;
    qk_pair(a, d, &pair, &e, &second);
    const double u = Ld<T>::d(g[e]);
    const long long o = (long long)max(p, 0) * a.half + pair;
    const double c = __ldg(a.cos_ + o), sn = __ldg(a.sin_ + o);
    v = second ? fma(v, c, -u * sn) : fma(v, c, u * sn);
  }
  return p < 0 ? (double)__int_as_float(0x7fffffff) : v;
}

template <typename T>
__global__ void __launch_bounds__(256) qk_bwd_any_kernel(const __grid_constant__ QkArgs a,
                                                         long long rows) {
  const int lane = threadIdx.x & 31;
  for (long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); row < rows;
       row += (long long)gridDim.x * 8) {
    const QkRow q = qk_row(a, row);
    const QkSide& s = a.s[q.side];
    const T* x = reinterpret_cast<const T*>(s.x) + q.b * s.xb + q.l * s.xl + q.head * s.xh;
    const T* g = reinterpret_cast<const T*>(s.g) + q.b * s.gb + q.l * s.gl + q.head * s.gh;
    T* dx = reinterpret_cast<T*>(s.out) + q.b * s.ob + q.l * s.ol + q.head * s.oh;
    const int p = qk_position(a, q.b, q.l);
    double ss = 0, dot = 0;
    for (int d = lane; d < a.D; d += 32) {
      const double v = Ld<T>::d(x[d]);
      ss = fma(v, v, ss);
      dot = fma(v * qk_weight<T>(a, s, q.head, d), qk_unrotated(a, g, p, d), dot);
    }
    const double r = 1.0 / sqrt(warp_sum(ss) / a.D + a.eps64);
    const double m = warp_sum(dot) * r / a.D;
    if (a.rstd && lane == 0) a.rstd[row] = (float)r;
    for (int d = lane; d < a.D; d += 32) {
      const double u = qk_weight<T>(a, s, q.head, d) * qk_unrotated(a, g, p, d);
      dx[d] = St<T>::v((float)(r * fma(-Ld<T>::d(x[d]) * r, m, u)));
    }
  }
}

// Weight gradient, first pass: block (chunk, head) sums g o x r over the
// chunk's tokens; part[side][chunk][head][D].
template <typename T>
__global__ void __launch_bounds__(256) qk_dw_any_kernel(const __grid_constant__ QkArgs a,
                                                        float* part, int chunks) {
  const int per = a.s[0].heads + a.s[1].heads;
  const int hh = blockIdx.y;
  const int side = hh >= a.s[0].heads;
  const int head = side ? hh - a.s[0].heads : hh;
  const QkSide& s = a.s[side];
  if (!s.w || !s.g) return;
  const long long tokens = (long long)a.B * a.L;
  const long long per_chunk = (tokens + chunks - 1) / chunks;
  const long long t0 = blockIdx.x * per_chunk, t1 = min(tokens, t0 + per_chunk);
  for (int d = threadIdx.x; d < a.D; d += blockDim.x) {
    float sum = 0.f;
    for (long long t = t0; t < t1; ++t) {
      const int b = (int)(t / a.L), l = (int)(t - (long long)b * a.L);
      const T* x = reinterpret_cast<const T*>(s.x) + b * s.xb + l * s.xl + head * s.xh;
      const T* g = reinterpret_cast<const T*>(s.g) + b * s.gb + l * s.gl + head * s.gh;
      sum = fmaf((float)qk_unrotated(a, g, qk_position(a, b, l), d) * Ld<T>::f(x[d]),
                 a.rstd[t * per + hh], sum);
    }
    part[((long long)blockIdx.x * per + hh) * a.D + d] = sum;
  }
}

// Second pass: sums the partials of one weight component in a fixed order.
template <typename T>
__global__ void __launch_bounds__(128) qk_dw_sum_kernel(const float* part, int chunks, int hq,
                                                        int hk, int D, int per_head, int w32,
                                                        void* dqw, void* dkw) {
  const int per = hq + hk;
  const int side = blockIdx.y;
  const int heads = side ? hk : hq, first = side ? hq : 0;
  void* out = side ? dkw : dqw;
  if (!out) return;
  const int n = per_head ? heads * D : D;
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int d = per_head ? i % D : i;
  const int h0 = per_head ? i / D : 0, h1 = per_head ? h0 + 1 : heads;
  float sum = 0.f;
  for (int c = 0; c < chunks; ++c) {
    float part_sum = 0.f;
    for (int h = h0; h < h1; ++h) part_sum += part[((long long)c * per + first + h) * D + d];
    sum += part_sum;
  }
  if (w32) reinterpret_cast<float*>(out)[i] = sum;
  else reinterpret_cast<T*>(out)[i] = St<T>::v(sum);
}

static int qk_dw_chunks(long long tokens) {
  return (int)std::max<long long>(1, std::min<long long>(tokens / 16, 256));
}

size_t qk_backward_ws_bytes(int batch, int length, int q_heads, int k_heads, int dim) {
  const long long tokens = (long long)batch * length;
  const long long per = q_heads + k_heads;
  return (size_t)(4 * (tokens * per + (long long)qk_dw_chunks(tokens) * per * dim));
}

template <typename T>
static int qk_run(const QkArgs& a, bool backward, void* ws, void* dqw, void* dkw, int device,
                  cudaStream_t st) {
  const long long tokens = (long long)a.B * a.L;
  const int per = a.s[0].heads + a.s[1].heads;
  const long long rows = tokens * per;
  const long long want = (rows + 7) / 8;
  const unsigned grid = (unsigned)std::min<long long>(want, (long long)sm_count(device) * 8);
  if (!backward) {
    qk_fwd_any_kernel<T><<<grid, 256, 0, st>>>(a, rows);
    FAB_LAUNCH_CHECK();
    return FA_OK;
  }
  QkArgs b = a;
  b.rstd = reinterpret_cast<float*>(ws);
  qk_bwd_any_kernel<T><<<grid, 256, 0, st>>>(b, rows);
  FAB_LAUNCH_CHECK();
  if (dqw || dkw) {
    const int chunks = qk_dw_chunks(tokens);
    float* part = b.rstd + rows;
    qk_dw_any_kernel<T><<<dim3((unsigned)chunks, (unsigned)per), 256, 0, st>>>(b, part, chunks);
    FAB_LAUNCH_CHECK();
    const int n = a.per_head ? std::max(a.s[0].heads, a.s[1].heads) * a.D : a.D;
    qk_dw_sum_kernel<T><<<dim3((unsigned)((n + 127) / 128), 2), 128, 0, st>>>(
        part, chunks, a.s[0].heads, a.s[1].heads, a.D, a.per_head, a.w32, dqw, dkw);
    FAB_LAUNCH_CHECK();
  }
  return FA_OK;
}

static void qk_fill(QkSide* s, const fa_heads* x, const fa_heads* g, const fa_heads* out,
                    const void* w) {
  s->x = x->data;
  s->heads = x->heads;
  s->xb = x->stride_b; s->xl = x->stride_l; s->xh = x->stride_h;
  if (g) {
    s->g = g->data;
    s->gb = g->stride_b; s->gl = g->stride_l; s->gh = g->stride_h;
  }
  s->out = out->data;
  s->ob = out->stride_b; s->ol = out->stride_l; s->oh = out->stride_h;
  s->w = w;
}

static bool qk_heads_ok(const fa_heads* h, int heads) {
  return h && h->data && h->heads > 0 && h->heads == heads;
}

int qk_impl(const fa_heads* q, const fa_heads* k, const fa_heads* gq, const fa_heads* gk,
            const fa_heads* oq, const fa_heads* ok, bool backward, const fa_qk_params* pr,
            void* ws, size_t ws_bytes, void* dqw, void* dkw, int device, cudaStream_t st) {
  if (!pr || !q || !k) return FA_E_ARG;
  if (!qk_heads_ok(q, q->heads) || !qk_heads_ok(k, k->heads) || !qk_heads_ok(oq, q->heads) ||
      !qk_heads_ok(ok, k->heads))
    return FA_E_ARG;
  if (backward && (!qk_heads_ok(gq, q->heads) || !qk_heads_ok(gk, k->heads))) return FA_E_ARG;
  if (pr->dtype != FA_F16 && pr->dtype != FA_BF16 && pr->dtype != FA_F32) return FA_E_DTYPE;
  if (pr->weight_dtype != pr->dtype && pr->weight_dtype != FA_F32) return FA_E_DTYPE;
  if (pr->batch <= 0 || pr->length <= 0 || pr->dim <= 0 || pr->rotary < 0 || pr->rotary % 2 ||
      pr->rotary > pr->dim || pr->dim > kMaxDim || pr->table < 0)
    return FA_E_SHAPE;
  if (pr->rotary && (!pr->cos_table || !pr->sin_table || pr->table == 0)) return FA_E_ARG;
  if ((dqw && !pr->q_weight) || (dkw && !pr->k_weight)) return FA_E_ARG;
  if ((long long)pr->batch * pr->length > 0x7fffffffLL || q->heads + (long long)k->heads > 65535)
    return FA_E_SHAPE;
  if (backward && (!ws || ws_bytes < qk_backward_ws_bytes(pr->batch, pr->length, q->heads,
                                                          k->heads, pr->dim)))
    return FA_E_ARG;
  QkArgs a{};
  qk_fill(&a.s[0], q, gq, oq, pr->q_weight);
  qk_fill(&a.s[1], k, gk, ok, pr->k_weight);
  a.B = pr->batch; a.L = pr->length; a.D = pr->dim; a.half = pr->rotary / 2;
  a.interleaved = pr->interleaved != 0;
  a.per_head = pr->weight_per_head != 0;
  a.w32 = pr->weight_dtype == FA_F32;
  a.cos_ = pr->cos_table; a.sin_ = pr->sin_table;
  // without a rotation no position is looked up, so none is out of range
  a.table = pr->rotary ? pr->table : 0x7fffffff;
  a.pos = pr->rotary ? pr->positions : nullptr;
  a.pos64 = pr->positions_64 != 0;
  a.pos_b = pr->pos_stride_b; a.pos_l = pr->pos_stride_l;
  a.eps = (float)pr->eps;
  a.eps64 = pr->eps;
  a.inv_d = 1.0f / (float)pr->dim;
  switch (pr->dtype) {
    case FA_F16: return qk_run<f16_t>(a, backward, ws, dqw, dkw, device, st);
    case FA_BF16: return qk_run<bf16_t>(a, backward, ws, dqw, dkw, device, st);
    default: return qk_run<float>(a, backward, ws, dqw, dkw, device, st);
  }
}

}  // namespace fab
