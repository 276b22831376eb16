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

// ---------------------------------------------------------------------------
// Vector kernels: head sizes and alignments that whole vectors cover.
//
// A head vector is held by a group of G lanes (a power of two); a lane owns two
// chunks of V components, A and B.  Adjacent halves rotate (A with B), so
// chunk A lies in the first half of the rotated part and B V-for-V in the
// second; lanes past the rotated part own two chunks of the rest.  Interleaved
// pairs lie inside a chunk, and A and B are chunks of the two halves of the
// head.  So no component changes lanes and a row costs two vector loads and
// stores a lane and log2(G) shuffles.  The angles of a token are loaded once
// and serve a lane's chunk in `hpi` heads.
//
// Both kernels are bound by HBM: the work per component is about 10 (backward:
// 25) float operations for 4 to 12 bytes.  Measured on one B200: forward, 1 x
// 32761 tokens of 32 + 8 heads of 128, float16: 132 us, 5.1 TB/s of the bytes
// it cannot do without (0.79 of the measured copy rate); backward, 2 x 8160
// tokens of 16 + 16 heads of 64, bfloat16: 62 us, 3.2 TB/s (0.50), held back by
// load latency at the 16 warps a multiprocessor that its registers leave.
// ---------------------------------------------------------------------------
// V components as they lie in memory: rows in flight wait unconverted.
template <typename T, int V> using Raw = typename RawOf<sizeof(T) * V>::type;

template <typename T, int V>
__device__ __forceinline__ Raw<T, V> qk_raw(const T* p, bool live) {
  Raw<T, V> u{};
  if (live) u = *reinterpret_cast<const Raw<T, V>*>(p);
  return u;
}
template <typename T, int V>
__device__ __forceinline__ void qk_wide(const Raw<T, V>& u, float (&v)[V]) {
  const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = Ld<T>::f(e[i]);
}
template <typename T, int V>
__device__ __forceinline__ void qk_store(T* p, const float (&v)[V]) {
  Raw<T, V> u;
  T* e = reinterpret_cast<T*>(&u);
#pragma unroll
  for (int i = 0; i < V; ++i) e[i] = St<T>::v(v[i]);
  *reinterpret_cast<Raw<T, V>*>(p) = u;
}

// What a lane owns: the offsets of its chunks and whether they turn.
struct QkLane {
  int a0, b0, t0;     // chunk offsets; first table column (of A when interleaved)
  int t1;             // interleaved: first table column of B
  bool live, turn, turn_b;
};
template <int V>
__device__ __forceinline__ QkLane qk_lane(const QkArgs& a, int j) {
  QkLane q;
  const int pairs = a.D / (2 * V);
  q.live = j < pairs;
  if (!q.live) j = 0;
  if (a.interleaved) {
    q.a0 = j * V;
    q.b0 = a.D / 2 + j * V;
    q.t0 = q.a0 / 2;
    q.t1 = q.b0 / 2;
    q.turn = q.a0 < 2 * a.half;
    q.turn_b = q.b0 < 2 * a.half;
  } else {
    const int rot = a.half / V;
    q.turn = q.turn_b = j < rot;
    q.t0 = q.t1 = j * V;
    const int rest = j - rot, r = 2 * a.half;
    q.a0 = q.turn ? j * V : r + rest * V;
    q.b0 = q.turn ? a.half + j * V : r + (a.D - r) / 2 + rest * V;
  }
  return q;
}

// cos and sin of the lane's V pairs: (A[i], B[i]), or interleaved the V/2 pairs
// of A and then those of B.
template <int V>
__device__ __forceinline__ void qk_angles(const QkArgs& a, const QkLane& q, int p, float (&c)[V],
                                          float (&s)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    c[i] = 1.f;
    s[i] = 0.f;
  }
  const long long o = (long long)max(p, 0) * a.half;
  if (a.interleaved) {
    if constexpr (V == 8) {
      if (q.turn) {
        *reinterpret_cast<float4*>(c) = __ldg(reinterpret_cast<const float4*>(a.cos_ + o + q.t0));
        *reinterpret_cast<float4*>(s) = __ldg(reinterpret_cast<const float4*>(a.sin_ + o + q.t0));
      }
      if (q.turn_b) {
        *reinterpret_cast<float4*>(c + 4) = __ldg(reinterpret_cast<const float4*>(a.cos_ + o + q.t1));
        *reinterpret_cast<float4*>(s + 4) = __ldg(reinterpret_cast<const float4*>(a.sin_ + o + q.t1));
      }
    } else {
      if (q.turn) {
        *reinterpret_cast<float2*>(c) = __ldg(reinterpret_cast<const float2*>(a.cos_ + o + q.t0));
        *reinterpret_cast<float2*>(s) = __ldg(reinterpret_cast<const float2*>(a.sin_ + o + q.t0));
      }
      if (q.turn_b) {
        *reinterpret_cast<float2*>(c + 2) = __ldg(reinterpret_cast<const float2*>(a.cos_ + o + q.t1));
        *reinterpret_cast<float2*>(s + 2) = __ldg(reinterpret_cast<const float2*>(a.sin_ + o + q.t1));
      }
    }
  } else if (q.turn) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      *reinterpret_cast<float4*>(c + i) = __ldg(reinterpret_cast<const float4*>(a.cos_ + o + q.t0 + i));
      *reinterpret_cast<float4*>(s + i) = __ldg(reinterpret_cast<const float4*>(a.sin_ + o + q.t0 + i));
    }
  }
}

// Turns the chunks that turn by the angles (sign -1: back).  The others are not
// multiplied by an identity: 0 times an infinity would be NaN.
template <int V>
__device__ __forceinline__ void qk_turn(const QkArgs& a, const QkLane& q, float (&x)[V],
                                        float (&y)[V], const float (&c)[V], const float (&s)[V],
                                        float sign) {
  if (a.interleaved) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float x0 = x[2 * i], x1 = x[2 * i + 1], y0 = y[2 * i], y1 = y[2 * i + 1];
      const float sx = sign * s[i], sy = sign * s[V / 2 + i];
      if (q.turn) {
        x[2 * i] = fmaf(x0, c[i], -x1 * sx);
        x[2 * i + 1] = fmaf(x1, c[i], x0 * sx);
      }
      if (q.turn_b) {
        y[2 * i] = fmaf(y0, c[V / 2 + i], -y1 * sy);
        y[2 * i + 1] = fmaf(y1, c[V / 2 + i], y0 * sy);
      }
    }
  } else if (q.turn) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float x0 = x[i], y0 = y[i], si = sign * s[i];
      x[i] = fmaf(x0, c[i], -y0 * si);
      y[i] = fmaf(y0, c[i], x0 * si);
    }
  }
}

template <typename T, int V>
__device__ __forceinline__ void qk_weights(const QkArgs& a, const QkSide& s, const QkLane& q,
                                           int head, float (&wa)[V], float (&wb)[V]) {
  if (!s.w) {
#pragma unroll
    for (int i = 0; i < V; ++i) wa[i] = wb[i] = 1.f;
    return;
  }
  const long long o = a.per_head ? (long long)head * a.D : 0;
  if (a.w32) {
    const float* w = reinterpret_cast<const float*>(s.w) + o;
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      *reinterpret_cast<float4*>(wa + i) = __ldg(reinterpret_cast<const float4*>(w + q.a0 + i));
      *reinterpret_cast<float4*>(wb + i) = __ldg(reinterpret_cast<const float4*>(w + q.b0 + i));
    }
  } else {
    const T* w = reinterpret_cast<const T*>(s.w) + o;
    qk_wide<T, V>(qk_raw<T, V>(w + q.a0, true), wa);
    qk_wide<T, V>(qk_raw<T, V>(w + q.b0, true), wb);
  }
}

template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Items of `hpi` heads of one side of one token, the items of a token side by
// side; U rows of a lane are in flight.
template <typename T, int V, int G, int U>
__global__ void __launch_bounds__(256, 2) qk_fwd_kernel(const __grid_constant__ QkArgs a, int hpi,
                                                     int items_q, int items, long long total) {
  const QkLane q = qk_lane<V>(a, threadIdx.x & (G - 1));
  const long long item = ((long long)blockIdx.x * 256 + threadIdx.x) / G;
  // lanes of idle groups stay: the shuffles name the whole warp
  const bool busy = item < total && q.live;
  const int t = item < total ? (int)(item / items) : 0;
  const int it = item < total ? (int)(item - (long long)t * items) : 0;
  const int b = t / a.L, l = t - b * a.L;
  const QkSide& s = a.s[it >= items_q];
  const int h0 = (it >= items_q ? it - items_q : it) * hpi, h1 = min(s.heads, h0 + hpi);
  __align__(16) float c[V], sn[V], wa[V], wb[V];
  const int p = qk_position(a, b, l);
  qk_angles<V>(a, q, p, c, sn);
  if (!a.per_head) qk_weights<T, V>(a, s, q, 0, wa, wb);
  const T* x = reinterpret_cast<const T*>(s.x) + b * s.xb + l * s.xl;
  T* y = reinterpret_cast<T*>(s.out) + b * s.ob + l * s.ol;
  for (int r = 0; r < hpi; r += U) {
    Raw<T, V> ra[U], rb[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + r + u;
      ra[u] = qk_raw<T, V>(x + h * s.xh + q.a0, busy && h < h1);
      rb[u] = qk_raw<T, V>(x + h * s.xh + q.b0, busy && h < h1);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float xa[V], xb[V], ss = 0.f;
      qk_wide<T, V>(ra[u], xa);
      qk_wide<T, V>(rb[u], xb);
#pragma unroll
      for (int i = 0; i < V; ++i) ss = fmaf(xa[i], xa[i], fmaf(xb[i], xb[i], ss));
      float rs = rsqrtf(fmaf(group_sum<G>(ss), a.inv_d, a.eps));
      if (p < 0) rs = __int_as_float(0x7fffffff);
      const int h = h0 + r + u;
      if (busy && h < h1) {
        if (a.per_head) qk_weights<T, V>(a, s, q, h, wa, wb);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          xa[i] *= rs * wa[i];
          xb[i] *= rs * wb[i];
        }
        qk_turn<V>(a, q, xa, xb, c, sn, 1.f);
        qk_store<T, V>(y + h * s.oh + q.a0, xa);
        qk_store<T, V>(y + h * s.oh + q.b0, xb);
      }
    }
  }
}

// Sums the blocks' partial weight gradients part[block][D] in a fixed order.
// Blocks whose number is `it` modulo `items` hold item `it`.
template <typename T>
__device__ __forceinline__ void qk_dw_finish(const QkArgs& a, const float* part, int rounds,
                                             int items, int first, int count, int heads, void* out,
                                             float* sm) {
  const int n = a.per_head ? heads * a.D : a.D;
  int w = 32;
  while (w < 256 && w < n) w *= 2;
  const int sub = 256 / w, o0 = threadIdx.x % w, sb = threadIdx.x / w;
  for (int base = 0; base < n; base += w) {
    const int o = base + o0;
    float sum = 0.f;
    if (o < n) {
      const int d = a.per_head ? o % a.D : o;
      const int lo = a.per_head ? first + o / a.D : first, nit = a.per_head ? 1 : count;
      const int terms = rounds * nit;
#pragma unroll 8
      for (int k = sb; k < terms; k += sub) {
        const int blk = (k / nit) * items + lo + k % nit;
        sum += __ldcg(part + (long long)blk * a.D + d);
      }
    }
    __syncthreads();
    sm[threadIdx.x] = sum;
    __syncthreads();
    if (sb == 0 && o < n) {
      for (int i = 1; i < sub; ++i) sum += sm[i * w + o0];
      if (a.w32) reinterpret_cast<float*>(out)[o] = sum;
      else reinterpret_cast<T*>(out)[o] = St<T>::v(sum);
    }
  }
}

// A block keeps one item (one side, `hpi` heads; one head when the weights are
// per head) and walks over tokens, so that each lane sums the weight gradient
// of its chunks in registers; the block's sums go to `part`, and the last block
// adds the blocks up.  One head vector of a lane in flight: a second one costs
// the registers of a load batch and measured slower (62 against 68 us on
// 2 x 8160 tokens of 16 + 16 heads of 64, bfloat16), as did three blocks a
// multiprocessor.
template <typename T, int V, int G>
__global__ void __launch_bounds__(256, 2) qk_bwd_kernel(const __grid_constant__ QkArgs a, int hpi,
                                                     int items_q, int items, unsigned* counter,
                                                     float* part, void* dqw, void* dkw) {
  __shared__ float sm[8 * kMaxDim];
  __shared__ int flag;
  const QkLane q = qk_lane<V>(a, threadIdx.x & (G - 1));
  const int it = blockIdx.x % items, round = blockIdx.x / items, rounds = gridDim.x / items;
  const QkSide& s = a.s[it >= items_q];
  const int h0 = (it >= items_q ? it - items_q : it) * hpi, h1 = min(s.heads, h0 + hpi);
  const int tokens = a.B * a.L;
  constexpr int GPB = 256 / G;
  __align__(16) float c[V], sn[V], wa[V], wb[V];
  float da[V], db[V];
  qk_weights<T, V>(a, s, q, h0, wa, wb);  // per head: hpi is 1
#pragma unroll
  for (int i = 0; i < V; ++i) da[i] = db[i] = 0.f;
  for (int t0 = round * GPB; t0 < tokens; t0 += rounds * GPB) {
    const int t = t0 + threadIdx.x / G;
    const bool busy = t < tokens && q.live;
    const int b = t < tokens ? t / a.L : 0, l = t < tokens ? t - b * a.L : 0;
    const int p = qk_position(a, b, l);
    qk_angles<V>(a, q, p, c, sn);
    const T* x = reinterpret_cast<const T*>(s.x) + b * s.xb + l * s.xl;
    const T* g = reinterpret_cast<const T*>(s.g) + b * s.gb + l * s.gl;
    T* dx = reinterpret_cast<T*>(s.out) + b * s.ob + l * s.ol;
    for (int r = 0; r < hpi; ++r) {
      const int h = h0 + r;
      const bool live = busy && h < h1;
      const Raw<T, V> ra = qk_raw<T, V>(x + h * s.xh + q.a0, live);
      const Raw<T, V> rb = qk_raw<T, V>(x + h * s.xh + q.b0, live);
      const Raw<T, V> sa = qk_raw<T, V>(g + h * s.gh + q.a0, live);
      const Raw<T, V> sb = qk_raw<T, V>(g + h * s.gh + q.b0, live);
      float xa[V], xb[V], ga[V], gb[V];
      qk_wide<T, V>(ra, xa);
      qk_wide<T, V>(rb, xb);
      qk_wide<T, V>(sa, ga);
      qk_wide<T, V>(sb, gb);
      qk_turn<V>(a, q, ga, gb, c, sn, -1.f);
      float ss = 0.f, dot = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        ss = fmaf(xa[i], xa[i], fmaf(xb[i], xb[i], ss));
        dot = fmaf(xa[i] * wa[i], ga[i], fmaf(xb[i] * wb[i], gb[i], dot));
      }
      float rs = rsqrtf(fmaf(group_sum<G>(ss), a.inv_d, a.eps));
      if (p < 0) rs = __int_as_float(0x7fffffff);
      const float m = group_sum<G>(dot) * rs * a.inv_d;
      if (live) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float ha = xa[i] * rs, hb = xb[i] * rs;
          da[i] = fmaf(ga[i], ha, da[i]);
          db[i] = fmaf(gb[i], hb, db[i]);
          xa[i] = rs * fmaf(-ha, m, wa[i] * ga[i]);
          xb[i] = rs * fmaf(-hb, m, wb[i] * gb[i]);
        }
        qk_store<T, V>(dx + h * s.oh + q.a0, xa);
        qk_store<T, V>(dx + h * s.oh + q.b0, xb);
      }
    }
  }
  if (!dqw && !dkw) return;
#pragma unroll
  for (int i = 0; i < V; ++i) {
#pragma unroll
    for (int o = G; o < 32; o <<= 1) {
      da[i] += __shfl_xor_sync(0xffffffffu, da[i], o);
      db[i] += __shfl_xor_sync(0xffffffffu, db[i], o);
    }
  }
  if (q.live && (threadIdx.x & 31) < G) {
    float* w = sm + (threadIdx.x >> 5) * a.D;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      w[q.a0 + i] = da[i];
      w[q.b0 + i] = db[i];
    }
  }
  __syncthreads();
  for (int d = threadIdx.x; d < a.D; d += 256) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += sm[i * a.D + d];
    part[(long long)blockIdx.x * a.D + d] = sum;
  }
  if (!last_block_arrived(counter, gridDim.x, &flag)) return;
  if (dqw) qk_dw_finish<T>(a, part, rounds, items, 0, items_q, a.s[0].heads, dqw, sm);
  if (dkw)
    qk_dw_finish<T>(a, part, rounds, items, items_q, items - items_q, a.s[1].heads, dkw, sm);
}

static int qk_dw_chunks(long long tokens) {
  return (int)std::max<long long>(1, std::min<long long>(tokens / 16, 256));
}

// Blocks of the vector backward: as many as run at once (two a multiprocessor
// at its registers), a whole number of rounds over the items.
static int qk_bwd_rounds(long long tokens, int items, int groups, int sms) {
  const long long need = (tokens + groups - 1) / groups;
  return (int)std::max<long long>(1, std::min<long long>(need, std::max(1, 2 * sms / items)));
}

size_t qk_backward_ws_bytes(int batch, int length, int q_heads, int k_heads, int dim) {
  const long long tokens = (long long)batch * length;
  const long long per = q_heads + k_heads;
  const size_t any = (size_t)(4 * (tokens * per + (long long)qk_dw_chunks(tokens) * per * dim));
  const size_t vec = (size_t)4 * dim * std::max<long long>(512, 2 * per);
  return FAB_COUNTER_BYTES + std::max(any, vec);
}

// Whether the vector kernels with V components a chunk serve this call.
static bool qk_vector(const QkArgs& a, int V, int item, bool backward) {
  if (a.D < 16 || a.D % (2 * V) || a.D / (2 * V) > 32 || a.half % 4) return false;
  if (a.interleaved ? (2 * a.half) % V : a.half % V || ((a.D - 2 * a.half) / 2) % V) return false;
  if ((long long)a.B * a.L > 0x7fff0000LL) return false;
  uintptr_t bits = 0;
  auto side = [&](const void* p, long long sb, long long sl, long long sh, int heads) {
    bits |= reinterpret_cast<uintptr_t>(p);
    if (a.B > 1) bits |= (uintptr_t)(sb * item);
    if (a.L > 1) bits |= (uintptr_t)(sl * item);
    if (heads > 1) bits |= (uintptr_t)(sh * item);
  };
  for (const QkSide& s : a.s) {
    side(s.x, s.xb, s.xl, s.xh, s.heads);
    side(s.out, s.ob, s.ol, s.oh, s.heads);
    if (backward) side(s.g, s.gb, s.gl, s.gh, s.heads);
    if (s.w && !a.w32) bits |= reinterpret_cast<uintptr_t>(s.w);
  }
  uintptr_t wide = 0;
  for (const QkSide& s : a.s)
    if (s.w && a.w32) wide |= reinterpret_cast<uintptr_t>(s.w);
  wide |= reinterpret_cast<uintptr_t>(a.cos_) | reinterpret_cast<uintptr_t>(a.sin_);
  return bits % (V * item) == 0 && wide % 16 == 0;
}

template <typename T, int V, int G>
static int qk_launch(const QkArgs& a, bool backward, char* ws, void* dqw, void* dkw, int device,
                     cudaStream_t st) {
  const long long tokens = (long long)a.B * a.L;
  const int hq = a.s[0].heads, hk = a.s[1].heads, sms = sm_count(device);
  // Heads an item: the angles serve more of them, but every multiprocessor gets
  // its 1024 lanes first.
  auto lanes = [&](int hpi) { return tokens * ((hq + hpi - 1) / hpi + (hk + hpi - 1) / hpi) * G; };
  const int hpi = backward && a.per_head ? 1
                  : lanes(8) >= 1024ll * sms ? 8 : lanes(4) >= 1024ll * sms ? 4 : 1;
  const int items_q = (hq + hpi - 1) / hpi, items = items_q + (hk + hpi - 1) / hpi;
  if (!backward) {
    const long long total = tokens * items;
    const long long blocks = (total * G + 255) / 256;
    if (blocks > 0x7fffffffLL) return FA_E_SHAPE;
    if (hpi == 1)
      qk_fwd_kernel<T, V, G, 1><<<(unsigned)blocks, 256, 0, st>>>(a, hpi, items_q, items, total);
    else
      qk_fwd_kernel<T, V, G, 4><<<(unsigned)blocks, 256, 0, st>>>(a, hpi, items_q, items, total);
  } else {
    const int rounds = qk_bwd_rounds(tokens, items, 256 / G, sms);
    unsigned* counter = reinterpret_cast<unsigned*>(ws);
    float* part = reinterpret_cast<float*>(ws + FAB_COUNTER_BYTES);
    const unsigned blocks = (unsigned)(rounds * items);
    qk_bwd_kernel<T, V, G><<<blocks, 256, 0, st>>>(a, hpi, items_q, items, counter, part, dqw, dkw);
  }
  FAB_LAUNCH_CHECK();
  return FA_OK;
}

template <typename T, int V>
static int qk_group(const QkArgs& a, bool backward, char* ws, void* dqw, void* dkw, int device,
                    cudaStream_t st) {
  const int pairs = a.D / (2 * V);
  if (pairs <= 4) return qk_launch<T, V, 4>(a, backward, ws, dqw, dkw, device, st);
  if (pairs <= 8) return qk_launch<T, V, 8>(a, backward, ws, dqw, dkw, device, st);
  if (pairs <= 16) return qk_launch<T, V, 16>(a, backward, ws, dqw, dkw, device, st);
  return qk_launch<T, V, 32>(a, backward, ws, dqw, dkw, device, st);
}

template <typename T>
static int qk_run(const QkArgs& a, bool backward, void* wsv, void* dqw, void* dkw, int device,
                  cudaStream_t st) {
  char* ws = static_cast<char*>(wsv);
  if constexpr (sizeof(T) == 2) {
    if (qk_vector(a, 8, 2, backward)) return qk_group<T, 8>(a, backward, ws, dqw, dkw, device, st);
    if (qk_vector(a, 4, 2, backward)) return qk_group<T, 4>(a, backward, ws, dqw, dkw, device, st);
  } else {
    if (qk_vector(a, 4, 4, backward)) return qk_group<T, 4>(a, backward, ws, dqw, dkw, device, st);
  }
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
  b.rstd = reinterpret_cast<float*>(ws + FAB_COUNTER_BYTES);
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
