// Layer norm over the last dimension, with the residual sum before it and the
// packing of its input in the same pass.
//
//   s = fl_T(x + residual),  m = mean s,  r = 1 / sqrt(mean (s - m)^2 + eps),
//   h = (s - m) r,  y = h w + b;
//   backward, with dy and the sum's own gradient ds:  g = dy w,
//   dx = r (g - mean g - h mean(g h)) + ds,   dw = sum dy h,   db = sum dy,
// where h comes from s, or from what its packed copy (keep8.cuh) stands for; m
// and r are those of s either way, kept in float32.
//
// The variance is summed about a first mean (not as a difference of squares, which a
// common offset would cancel), and the same pass sums the values' distances from it: a
// float32 sum of n values is up to n 2^-24 of their size off, which against eps is not
// little for a row of one value (0.15 instead of 0 at 4096 columns around 1000), while
// the sum of the distances carries no common part any more.  With d = s - m0:
//   m = m0 + mean d,  variance = mean d^2 - (mean d)^2.
// All sums are float32.  dw and db are summed in a fixed order without atomics, so they
// are the same bits on every run.
//
// Measured on one B200, 65280 x 4096 bfloat16: forward 211 us (0.77 of the copy rate),
// with the residual sum 313 us (1.0), with packing too 358 us (1.0); backward 377 us
// (0.65), with the sum's gradient 407 us (0.80), from packed input 412 us (0.70).  The
// forward pass is bound by bytes where there are more than a read and a write of each
// value; the backward pass by the latency of joining a row's two sums, with 16 warps a
// multiprocessor that its registers allow.
#include <algorithm>

#include "keep8.cuh"

namespace fab {

struct NormArgs {
  const void *x, *res;          // input (backward: s or null), residual or null
  long long x_row, res_row;
  const void *w, *b;            // or null
  int w32;                      // weights are float32
  int w_vec;                    // and start at whole vectors
  void *y, *sum;                // forward: outputs, sum or null; backward: y is dx
  const void *dy, *ds;          // upstream gradients, ds or null
  long long dy_row, ds_row;
  float2* stats;                // mean, 1 / deviation of every row; forward: or null
  unsigned char* codes;         // packed s, or null
  void* ranges;
  long long rows;
  int width, groups;
  float eps, inv_width;
  // weight gradients
  float* part;                  // [splits][2][width] partial sums
  void *dw, *db;                // or null
  int splits;
};

// n weights from column c; `none` where there are none.
template <typename T, bool VEC>
__device__ __forceinline__ F8 weights8(const NormArgs& a, const void* w, int c, int n, float none) {
  F8 x;
  if (!w) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x.v[i] = both(none);
  } else if (a.w32) {
    const float* p = reinterpret_cast<const float*>(w) + c;
    x = VEC && a.w_vec && n == 8 ? widen8(get8<float>(p)) : few8<float>(p, n);
  } else {
    const T* p = reinterpret_cast<const T*>(w) + c;
    x = VEC && a.w_vec && n == 8 ? widen8(get8<T>(p)) : few8<T>(p, n);
  }
  return x;
}
// (x - m) r
__device__ __forceinline__ void normalise8(F8& x, float m, float r) {
#pragma unroll
  for (int i = 0; i < 4; ++i) x.v[i] = __fmul2_rn(__fadd2_rn(x.v[i], both(-m)), both(r));
}

// s of 8 columns, from the inputs.
template <typename T, bool VEC>
__device__ __forceinline__ F8 input8(const NormArgs& a, long long row, int c, int n, Turn8<T>* t) {
  F8 x = widen8(fetch8<T, VEC>(reinterpret_cast<const T*>(a.x) + row * a.x_row + c, n, t));
  if (a.res) {
    const F8 y =
        widen8(fetch8<T, VEC>(reinterpret_cast<const T*>(a.res) + row * a.res_row + c, n, t));
#pragma unroll
    for (int i = 0; i < 4; ++i) x.v[i] = __fadd2_rn(x.v[i], y.v[i]);
    round8(x, T());
  }
  return x;
}
// s of 8 columns in the backward pass: kept, or from its codes.
template <typename T, bool VEC>
__device__ __forceinline__ F8 kept8(const NormArgs& a, long long row, int c, int n, Turn8<T>* t) {
  if (!a.codes)
    return widen8(fetch8<T, VEC>(reinterpret_cast<const T*>(a.x) + row * a.x_row + c, n, t));
  uint2 q = make_uint2(0u, 0u);
  typename RangeBits<T>::type bits = {};
  if (n) {
    q = __ldg(reinterpret_cast<const uint2*>(a.codes + row * a.groups * kGroup8 + c));
    bits = __ldg(reinterpret_cast<const typename RangeBits<T>::type*>(a.ranges) + row * a.groups +
                 c / kGroup8);
  }
  return decode8<T>(q, range_of(bits, T()));
}
template <typename T, bool VEC>
__device__ __forceinline__ F8 grad8(const void* g, long long g_row, long long row, int c, int n,
                                    Turn8<T>* t) {
  return widen8(fetch8<T, VEC>(reinterpret_cast<const T*>(g) + row * g_row + c, n, t));
}
// Codes and range of 8 columns of s.
template <typename T, bool VEC, typename X>
__device__ __forceinline__ void keep8(const NormArgs& a, long long row, int u, int n, bool in,
                                      const F8& x, const X& as_extent) {
  Range8 r;
  float lo, hi;
  extent8<VEC>(as_extent, n, &lo, &hi);
  const uint2 q = encode8<T, VEC>(x, n, lo, hi, &r);
  if (!in) return;
  reinterpret_cast<uint2*>(a.codes)[row * a.groups * 8 + u] = q;
  if ((u & 7) == 0)
    reinterpret_cast<typename RangeBits<T>::type*>(a.ranges)[row * a.groups + u / 8] =
        range_bits(r, T());
}

// 1 / sqrt(v): the fast root and a Newton step.
__device__ __forceinline__ float inv_sqrt(float v) {
  const float r = rsqrtf(v);
  // of an infinite variance (0) or a variance and eps of 0 (infinity) there is no step
  return r > 0.f && r < __uint_as_float(0x7f800000u) ? r * fmaf(-0.5f * v * r, r, 1.5f) : r;
}

// Mean and 1 / deviation from a first mean m0 and the sums of the distances from it and
// of their squares.
__device__ __forceinline__ float2 moments(float m0, float d, float d2, float inv_width, float eps) {
  const float mean = d * inv_width;
  const float v = fmaf(d2, inv_width, -mean * mean);
  // rounding may leave a row of one value less than nothing
  return make_float2(m0 + mean, inv_sqrt((v < 0.f ? 0.f : v) + eps));
}

// Two sums over the warp with the shuffles of little more than one: the halves of the
// warp take one each.  Lane 0 has the first, lane 16 the second.
__device__ __forceinline__ float warp_sum2(float a, float b) {
  const bool low = (threadIdx.x & 16) == 0;
  const float give = low ? b : a;
  float t = (low ? a : b) + __shfl_xor_sync(0xffffffffu, give, 16);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  return t;
}

// Both passes below keep a row in the registers of `wpr` warps, E units of 256 columns
// a warp, and read and write every byte once.  What a row costs apart from its values
// (addresses, the joining of sums) bounds them as much as bytes do.
//
// How rows lie: in any way; in whole aligned vectors; or so that every lane's units are
// whole and weights of the operands' type lie so too, which leaves the loops without
// conditions and with one address an operand.
enum RowKind { ODD, VECTORS, FULL };

template <typename T, RowKind KIND, int E, int NT>
__global__ void __launch_bounds__(NT, NT > 512 ? 1 : 768 / NT) norm_kernel(const NormArgs a, int wpr) {
  constexpr bool VEC = KIND != ODD;
  typedef typename RangeBits<T>::type Bits;
  __shared__ float sm[32];
  __shared__ float2 sm2[32];
  __shared__ __align__(16) Turn8<T> turns[VEC ? 1 : NT / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Turn8<T>* const turn = turns + (VEC ? 0 : warp);
  const int at = warp % wpr, first = warp - at;          // this warp in its row, the row's first
  const int c0 = (at * E * 32 + lane) * 8;
  const long long row = (long long)blockIdx.x * (blockDim.x / 32 / wpr) + warp / wpr;
  const bool in = row < a.rows;
  if (KIND == FULL && !in) return;                       // a row of one warp: no barrier waits
  int n[E];
#pragma unroll
  for (int e = 0; e < E; ++e)
    n[e] = KIND == FULL ? 8 : in ? max(0, min(8, a.width - c0 - 256 * e)) : 0;
  const T* const xp = reinterpret_cast<const T*>(a.x) + row * a.x_row + c0;
  T* const yp = reinterpret_cast<T*>(a.y) + row * a.width + c0;
  // s stays as it lies in memory and is widened for each of the three passes over it:
  // half the registers of float32 values, so twice the rows under way
  Raw8<T> s[E];
  if (a.res) {
    const T* const rp = reinterpret_cast<const T*>(a.res) + row * a.res_row + c0;
    Raw8<T> q[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      s[e] = fetch8<T, VEC>(xp + 256 * e, n[e], turn);
      q[e] = fetch8<T, VEC>(rp + 256 * e, n[e], turn);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      F8 x = widen8(s[e]);
      const F8 y = widen8(q[e]);
#pragma unroll
      for (int i = 0; i < 4; ++i) x.v[i] = __fadd2_rn(x.v[i], y.v[i]);
      s[e] = narrow8(x, T());
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) s[e] = fetch8<T, VEC>(xp + 256 * e, n[e], turn);
  }
  float2 t = both(0.f);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const F8 x = widen8(s[e]);
#pragma unroll
    for (int i = 0; i < 4; ++i) t = __fadd2_rn(t, x.v[i]);
  }
  float total = warp_sum(t.x + t.y);
  if (wpr > 1) {
    if (lane == 0) sm[warp] = total;
    __syncthreads();
    total = 0.f;
    for (int w = 0; w < wpr; ++w) total += sm[first + w];
  }
  const float m0 = total * a.inv_width;
  float2 t1 = both(0.f), t2 = both(0.f);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (KIND == VECTORS && n[e] == 0) continue;
    F8 x = widen8(s[e]);
    if (!VEC) fill_from(x, n[e], m0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 d = __fadd2_rn(x.v[i], both(-m0));
      t1 = __fadd2_rn(t1, d);
      t2 = __ffma2_rn(d, d, t2);
    }
  }
  const float both_sums = warp_sum2(t1.x + t1.y, t2.x + t2.y);
  float2 sums;
  if (wpr > 1) {
    if ((lane & 15) == 0) reinterpret_cast<float*>(sm2 + warp)[lane >> 4] = both_sums;
    __syncthreads();
    sums = both(0.f);
    for (int w = 0; w < wpr; ++w) sums = __fadd2_rn(sums, sm2[first + w]);
  } else {
    sums.x = __shfl_sync(0xffffffffu, both_sums, 0);
    sums.y = __shfl_sync(0xffffffffu, both_sums, 16);
  }
  const float2 moment = moments(m0, sums.x, sums.y, a.inv_width, a.eps);
  const float m = moment.x, r = moment.y;
  if (a.stats && in && at == 0 && lane == 0) a.stats[row] = make_float2(m, r);
  if (a.sum) {
    T* const sp = reinterpret_cast<T*>(a.sum) + row * a.width + c0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if constexpr (VEC) {
        if (n[e]) put8<T>(sp + 256 * e, s[e]);
      } else {
        scatter8<T>(sp + 256 * e, n[e], s[e], turn);
      }
    }
  }
  if (a.codes) {
    uint2* const cp = reinterpret_cast<uint2*>(a.codes) + (row * a.groups * 8 + c0 / 8);
    Bits* const bp = reinterpret_cast<Bits*>(a.ranges) + (row * a.groups + c0 / kGroup8);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      Range8 range;
      float lo, hi;
      extent8<VEC>(s[e], n[e], &lo, &hi);
      const uint2 q = encode8<T, VEC>(widen8(s[e]), n[e], lo, hi, &range);
      if (KIND == FULL || (in && c0 / 8 + 32 * e < a.groups * 8)) {
        cp[32 * e] = q;
        if ((lane & 7) == 0) bp[4 * e] = range_bits(range, T());
      }
    }
  }
  const T* const wp = reinterpret_cast<const T*>(a.w) + c0;
  const T* const bp = reinterpret_cast<const T*>(a.b) + c0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    F8 x = widen8(s[e]);
    normalise8(x, m, r);
    if constexpr (KIND == FULL) {
      if (a.w) {
        const F8 w = widen8(get8<T>(wp + 256 * e));
#pragma unroll
        for (int i = 0; i < 4; ++i) x.v[i] = __fmul2_rn(x.v[i], w.v[i]);
      }
      if (a.b) {
        const F8 b = widen8(get8<T>(bp + 256 * e));
#pragma unroll
        for (int i = 0; i < 4; ++i) x.v[i] = __fadd2_rn(x.v[i], b.v[i]);
      }
    } else if (a.w || a.b) {
      const F8 w = weights8<T, VEC>(a, a.w, c0 + 256 * e, n[e], 1.f),
               b = weights8<T, VEC>(a, a.b, c0 + 256 * e, n[e], 0.f);
#pragma unroll
      for (int i = 0; i < 4; ++i) x.v[i] = __fadd2_rn(__fmul2_rn(x.v[i], w.v[i]), b.v[i]);
    }
    store8<T, VEC>(yp + 256 * e, n[e], x, turn);
  }
}

// Backward: a lane keeps the weight gradients of its columns in registers, the block
// adds its rows' at the end and writes one part.  The next row's loads are under way
// while a row's sums run.
template <typename T, RowKind KIND, int E, bool CODES, int NT>
__global__ void __launch_bounds__(NT, 512 / NT) norm_grad_kernel(const NormArgs a, int wpr) {
  constexpr bool VEC = KIND != ODD;
  __shared__ float2 sm[2][NT / 32];
  __shared__ float join[NT / 32][32 * 9];
  __shared__ __align__(16) Turn8<T> turns[VEC ? 1 : NT / 32];
  typedef typename RangeBits<T>::type Bits;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Turn8<T>* const turn = turns + (VEC ? 0 : warp);
  const int at = warp % wpr, first = warp - at, rpb = NT / 32 / wpr;
  const int c0 = (at * E * 32 + lane) * 8;
  F8 dw[E], db[E];
  Raw8<T> w[E];                 // weights of the operands' type stay; others are read anew
  int n[E];
  const bool w_kept = VEC && a.w && (KIND == FULL || (a.w_vec && (sizeof(T) == 4 || !a.w32)));
#pragma unroll
  for (int e = 0; e < E; ++e) {
#pragma unroll
    for (int i = 0; i < 4; ++i) dw[e].v[i] = db[e].v[i] = both(0.f);
    n[e] = KIND == FULL ? 8 : max(0, min(8, a.width - c0 - 256 * e));
    w[e] = w_kept && n[e] ? get8<T>(reinterpret_cast<const T*>(a.w) + c0 + 256 * e) : zero8<T>();
  }
  const long long start = (long long)blockIdx.x * rpb + warp / wpr;
  const long long step = (long long)gridDim.x * rpb;
  const T* gp = reinterpret_cast<const T*>(a.dy) + start * a.dy_row + c0;
  const T* sp = reinterpret_cast<const T*>(a.ds) + (a.ds ? start * a.ds_row + c0 : 0);
  const T* xp = reinterpret_cast<const T*>(a.x) + (CODES ? 0 : start * a.x_row + c0);
  const uint2* cp = reinterpret_cast<const uint2*>(a.codes) + (start * a.groups * 8 + c0 / 8);
  const Bits* bp = reinterpret_cast<const Bits*>(a.ranges) + (start * a.groups + c0 / kGroup8);
  T* yp = reinterpret_cast<T*>(a.y) + start * a.width + c0;
  struct Row {                  // as it lies in memory
    Raw8<T> x[E], g[E], s[E];
    uint2 code[E];
    Bits bits[E];
    float2 st;
  };
  const auto load = [&](long long row, Row& o) {  // and on to the next
    const bool in = row < a.rows;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int k = in ? n[e] : 0;
      if constexpr (CODES) {
        if (!VEC || k) {
          o.code[e] = k ? __ldg(cp + 32 * e) : make_uint2(0u, 0u);
          o.bits[e] = k ? __ldg(bp + 4 * e) : Bits();
        }
      } else {
        o.x[e] = fetch8<T, VEC>(xp + 256 * e, k, turn);
      }
      o.g[e] = fetch8<T, VEC>(gp + 256 * e, k, turn);
      if (a.ds) o.s[e] = fetch8<T, VEC>(sp + 256 * e, k, turn);
    }
    if (in) o.st = __ldg(a.stats + row);
    if constexpr (CODES) {
      cp += step * a.groups * 8;
      bp += step * a.groups;
    } else {
      xp += step * a.x_row;
    }
    gp += step * a.dy_row;
    sp += step * a.ds_row;
  };
  int half = 0;
  Row now;
  now.st = make_float2(0.f, 0.f);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    now.code[e] = make_uint2(0u, 0u);
    now.bits[e] = Bits();
  }
  long long row = start;
  load(row, now);
  for (long long row0 = (long long)blockIdx.x * rpb; row0 < a.rows; row0 += step, half ^= 1) {
    const bool in = row < a.rows;
    const float m = now.st.x, r = now.st.y;
    F8 h[E], g[E];
    float2 c1 = both(0.f), c2 = both(0.f);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (VEC && (!in || (KIND != FULL && !n[e]))) continue;
      if constexpr (CODES) h[e] = decode8<T>(now.code[e], range_of(now.bits[e], T()));
      else h[e] = widen8(now.x[e]);
      g[e] = widen8(now.g[e]);
      normalise8(h[e], m, r);
      if (!VEC) fill_from(h[e], in ? n[e] : 0, 0.f);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        dw[e].v[i] = __ffma2_rn(g[e].v[i], h[e].v[i], dw[e].v[i]);
        db[e].v[i] = __fadd2_rn(db[e].v[i], g[e].v[i]);
      }
      if (a.w) {
        const F8 f = KIND == FULL || w_kept ? widen8(w[e])
                                            : weights8<T, VEC>(a, a.w, c0 + 256 * e, n[e], 1.f);
#pragma unroll
        for (int i = 0; i < 4; ++i) g[e].v[i] = __fmul2_rn(g[e].v[i], f.v[i]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        c1 = __fadd2_rn(c1, g[e].v[i]);
        c2 = __ffma2_rn(g[e].v[i], h[e].v[i], c2);
      }
    }
    Raw8<T> s[E];
    if (a.ds) {
#pragma unroll
      for (int e = 0; e < E; ++e) s[e] = now.s[e];
    }
    row += step;
    load(row, now);
    const float both_sums = warp_sum2(c1.x + c1.y, c2.x + c2.y);
    float s1, s2;
    if (wpr > 1) {
      if ((lane & 15) == 0) reinterpret_cast<float*>(&sm[half][warp])[lane >> 4] = both_sums;
      __syncthreads();          // one a row: the next row's sums have the other half
      s1 = s2 = 0.f;
      for (int i = 0; i < wpr; ++i) {
        s1 += sm[half][first + i].x;
        s2 += sm[half][first + i].y;
      }
    } else {
      s1 = __shfl_sync(0xffffffffu, both_sums, 0);
      s2 = __shfl_sync(0xffffffffu, both_sums, 16);
    }
    // dx = r (g - s1 / N - h s2 / N)
    s1 *= -a.inv_width * r;
    s2 *= -a.inv_width * r;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int k = in ? n[e] : 0;
      if (VEC && !k) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        g[e].v[i] = __ffma2_rn(h[e].v[i], both(s2), __ffma2_rn(g[e].v[i], both(r), both(s1)));
      if (a.ds) {
        const F8 d = widen8(s[e]);
#pragma unroll
        for (int i = 0; i < 4; ++i) g[e].v[i] = __fadd2_rn(g[e].v[i], d.v[i]);
      }
      store8<T, VEC>(yp + 256 * e, k, g[e], turn);
    }
    yp += step * a.width;
  }
  if (!a.dw && !a.db) return;
  // warps that hold the same columns, in the order of their rows
#pragma unroll
  for (int e = 0; e < E; ++e)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (!(k ? a.db : a.dw)) continue;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 8; ++i) join[warp][lane * 9 + i] = k ? db[e].at(i) : dw[e].at(i);
      __syncthreads();
      for (int j = threadIdx.x; j < wpr * 256; j += NT) {
        const int w0 = j / 256, l = j % 256, col = (w0 * E + e) * 256 + l;
        float t = 0.f;
        for (int q = 0; q < rpb; ++q) t += join[q * wpr + w0][l / 8 * 9 + l % 8];
        if (col < a.width) a.part[((long long)blockIdx.x * 2 + k) * a.width + col] = t;
      }
    }
}

// A block to a row, which it reads again for each of its sums (from the
// second-level cache): for rows that fit no block's registers.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) norm_rows_kernel(const NormArgs a) {
  __shared__ float sm[32];
  __shared__ __align__(16) Turn8<T> turns[VEC ? 1 : 8];
  Turn8<T>* const turn = turns + (VEC ? 0 : threadIdx.x / 32);
  const int units = a.groups * 8;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    float t = 0.f;
    for (int u0 = 0; u0 < units; u0 += 256) {
      const int c = (u0 + threadIdx.x) * 8, n = max(0, min(8, a.width - c));
      t += sum8(input8<T, VEC>(a, row, c, n, turn));
    }
    const float m0 = block_sum(t, sm) * a.inv_width;
    float2 t1 = both(0.f), t2 = both(0.f);
    for (int u0 = 0; u0 < units; u0 += 256) {
      const int c = (u0 + threadIdx.x) * 8, n = max(0, min(8, a.width - c));
      F8 x = input8<T, VEC>(a, row, c, n, turn);
      fill_from(x, n, m0);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 d = __fadd2_rn(x.v[i], both(-m0));
        t1 = __fadd2_rn(t1, d);
        t2 = __ffma2_rn(d, d, t2);
      }
    }
    const float s1 = block_sum(t1.x + t1.y, sm), s2 = block_sum(t2.x + t2.y, sm);
    const float2 moment = moments(m0, s1, s2, a.inv_width, a.eps);
    const float m = moment.x, r = moment.y;
    if (a.stats && threadIdx.x == 0) a.stats[row] = make_float2(m, r);
    for (int u0 = 0; u0 < units; u0 += 256) {
      const int u = u0 + threadIdx.x, c = u * 8, n = max(0, min(8, a.width - c));
      F8 x = input8<T, VEC>(a, row, c, n, turn);
      if (a.sum) store8<T, VEC>(reinterpret_cast<T*>(a.sum) + row * a.width + c, n, x, turn);
      if (a.codes) keep8<T, VEC>(a, row, u, n, u < units, x, x);
      const F8 w = weights8<T, VEC>(a, a.w, c, n, 1.f), b = weights8<T, VEC>(a, a.b, c, n, 0.f);
      normalise8(x, m, r);
#pragma unroll
      for (int i = 0; i < 4; ++i) x.v[i] = __ffma2_rn(x.v[i], w.v[i], b.v[i]);
      store8<T, VEC>(reinterpret_cast<T*>(a.y) + row * a.width + c, n, x, turn);
    }
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) norm_grad_rows_kernel(const NormArgs a) {
  __shared__ float sm[32];
  __shared__ __align__(16) Turn8<T> turns[VEC ? 1 : 8];
  Turn8<T>* const turn = turns + (VEC ? 0 : threadIdx.x / 32);
  const int units = a.groups * 8;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float2 st = a.stats[row];
    float c1 = 0.f, c2 = 0.f;
    for (int u0 = 0; u0 < units; u0 += 256) {
      const int c = (u0 + threadIdx.x) * 8, n = max(0, min(8, a.width - c));
      F8 h = kept8<T, VEC>(a, row, c, n, turn);
      F8 g = grad8<T, VEC>(a.dy, a.dy_row, row, c, n, turn);
      const F8 w = weights8<T, VEC>(a, a.w, c, n, 1.f);
      normalise8(h, st.x, st.y);
      fill_from(h, n, 0.f);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        g.v[i] = __fmul2_rn(g.v[i], w.v[i]);
        h.v[i] = __fmul2_rn(g.v[i], h.v[i]);
      }
      c1 += sum8(g);
      c2 += sum8(h);
    }
    c1 = -block_sum(c1, sm) / (float)a.width;
    c2 = -block_sum(c2, sm) / (float)a.width;
    for (int u0 = 0; u0 < units; u0 += 256) {
      const int c = (u0 + threadIdx.x) * 8, n = max(0, min(8, a.width - c));
      F8 h = kept8<T, VEC>(a, row, c, n, turn);
      F8 g = grad8<T, VEC>(a.dy, a.dy_row, row, c, n, turn);
      const F8 w = weights8<T, VEC>(a, a.w, c, n, 1.f);
      normalise8(h, st.x, st.y);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        g.v[i] = __fmul2_rn(__ffma2_rn(h.v[i], both(c2), __ffma2_rn(g.v[i], w.v[i], both(c1))),
                            both(st.y));
      if (a.ds) {
        const F8 d = grad8<T, VEC>(a.ds, a.ds_row, row, c, n, turn);
#pragma unroll
        for (int i = 0; i < 4; ++i) g.v[i] = __fadd2_rn(g.v[i], d.v[i]);
      }
      store8<T, VEC>(reinterpret_cast<T*>(a.y) + row * a.width + c, n, g, turn);
    }
  }
}

// Column sums dw, db of one part of the rows: a block has 256 columns, a warp
// every eighth row, four at a time.  Without HATS db alone.
template <typename T, bool VEC, bool HATS>
__global__ void __launch_bounds__(256) column_sums_kernel(const NormArgs a) {
  __shared__ float sm[8][32 * 9];
  __shared__ __align__(16) Turn8<T> turns[VEC ? 1 : 8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Turn8<T>* const turn = turns + (VEC ? 0 : warp);
  const int c = (blockIdx.x * 32 + lane) * 8, n = max(0, min(8, a.width - c));
  F8 dw, db;
#pragma unroll
  for (int i = 0; i < 4; ++i) dw.v[i] = db.v[i] = both(0.f);
  const long long step = (long long)gridDim.y * 8;
  for (long long row0 = blockIdx.y * 8ll + warp; row0 < a.rows; row0 += 4 * step) {
    Raw8<T> g[4];
    F8 h[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const long long row = row0 + q * step;
      const bool in = row < a.rows;
      g[q] = fetch8<T, VEC>(reinterpret_cast<const T*>(a.dy) + (in ? row : 0) * a.dy_row + c,
                            in ? n : 0, turn);
      if constexpr (HATS) {
        h[q] = kept8<T, VEC>(a, in ? row : 0, c, in ? n : 0, turn);
        const float2 st = in ? __ldg(a.stats + row) : make_float2(0.f, 0.f);
        normalise8(h[q], st.x, st.y);
        fill_from(h[q], n, 0.f);
      }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const F8 x = widen8(g[q]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (HATS) dw.v[i] = __ffma2_rn(x.v[i], h[q].v[i], dw.v[i]);
        db.v[i] = __fadd2_rn(db.v[i], x.v[i]);
      }
    }
  }
#pragma unroll
  for (int k = HATS ? 0 : 1; k < 2; ++k) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) sm[warp][lane * 9 + i] = k ? db.at(i) : dw.at(i);
    __syncthreads();
    const int col = blockIdx.x * 256 + threadIdx.x;
    if (col < a.width) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) t += sm[w][threadIdx.x / 8 * 9 + threadIdx.x % 8];
      a.part[((long long)blockIdx.y * 2 + k) * a.width + col] = t;
    }
  }
}

// The parts' sums in their order, rounded to the weights' type.
template <typename T>
__global__ void __launch_bounds__(1024) column_join_kernel(const NormArgs a) {
  __shared__ float sm[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
  void* const out = blockIdx.y ? a.db : a.dw;
  if (!out) return;
  float t = 0.f;
  if (col < a.width)
#pragma unroll 8
    for (int i = warp; i < a.splits; i += 32)
      t += a.part[((long long)i * 2 + blockIdx.y) * a.width + col];
  sm[warp][lane] = t;
  __syncthreads();
  if (warp || col >= a.width) return;
  t = 0.f;
#pragma unroll
  for (int w = 0; w < 32; ++w) t += sm[w][lane];
  if (a.w32)
    reinterpret_cast<float*>(out)[col] = t;
  else
    reinterpret_cast<T*>(out)[col] = St<T>::v(t);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

// Parts of the rows in the column sums: four blocks a multiprocessor run at once,
// at least 8 rows to a warp.
static int column_splits(long long rows, int width, int device) {
  const int strips = (width + 255) / 256;
  const long long most = std::max(1ll, (rows + 63) / 64);
  return (int)std::min(most, (long long)std::max(1, sm_count(device) * 4 / strips));
}

// Warps that share a row and units of 8 columns a lane; 0 where a row does not fit.
struct RowShape {
  int wpr, e;
};
static RowShape forward_shape(int width) {
  const long long units = groups8(width) * 8;
  if (units <= 32) return {1, 1};
  if (units <= 64) return {1, 2};
  const long long wpr = (units + 127) / 128;
  return wpr <= 32 ? RowShape{(int)wpr, 4} : RowShape{0, 0};
}
// float32 rows hold one unit a lane where that covers the row: two take more registers
// than there are.
static RowShape backward_shape(int width, int item) {
  const long long units = groups8(width) * 8;
  for (int e = 1; e <= 2; ++e)
    for (int wpr = 1; wpr <= 16; wpr *= 2)
      if (units <= 32ll * e * wpr && (e == 2 || item == 4 || wpr == 1)) return {wpr, e};
  return {0, 0};
}
// Blocks of the backward pass: 512 threads a multiprocessor, each with rows to take.
static int backward_blocks(long long rows, int rpb, int threads, int device) {
  return (int)std::min((rows + rpb - 1) / rpb, (long long)(512 / threads) * sm_count(device));
}

// Room for the column sums' parts, or for a part a block where rows fit a block's registers.
size_t norm_ws_bytes(long long rows, int width, int device) {
  long long parts = column_splits(rows, width, device);
  if (backward_shape(width, 2).wpr)
    parts = std::max(parts, std::min(rows, 2ll * sm_count(device)));
  return (size_t)parts * 2 * (size_t)width * sizeof(float);
}

template <typename T>
static int column_join(const NormArgs& a, cudaStream_t st) {
  column_join_kernel<T><<<dim3((unsigned)((a.width + 31) / 32), 2), 1024, 0, st>>>(a);
  FAB_LAUNCH_CHECK();
  return FA_OK;
}

template <typename T>
static int column_sums(NormArgs& a, bool vec, int device, cudaStream_t st) {
  a.splits = column_splits(a.rows, a.width, device);
  const dim3 grid((unsigned)((a.width + 255) / 256), (unsigned)a.splits);
  const bool hats = a.x || a.codes;
  if (hats && vec)
    column_sums_kernel<T, true, true><<<grid, 256, 0, st>>>(a);
  else if (hats)
    column_sums_kernel<T, false, true><<<grid, 256, 0, st>>>(a);
  else if (vec)
    column_sums_kernel<T, true, false><<<grid, 256, 0, st>>>(a);
  else
    column_sums_kernel<T, false, false><<<grid, 256, 0, st>>>(a);
  FAB_LAUNCH_CHECK();
  return column_join<T>(a, st);
}
// Column sums of g alone (a bias's gradient), in the gradient's type.
int bias_grad_impl(const void* g, long long g_row, void* db, int dtype, long long rows, int width,
                   void* ws, size_t ws_bytes, int device, cudaStream_t st) {
  if (ws_bytes < norm_ws_bytes(rows, width, device)) return FA_E_ARG;
  NormArgs a = {};
  a.dy = g;
  a.dy_row = g_row;
  a.rows = rows;
  a.width = width;
  a.db = db;
  a.w32 = dtype == FA_F32;
  a.part = static_cast<float*>(ws);
  const bool vec = whole8(g, g_row, rows, width, item_size(dtype));
  FAB_FOR_TYPE(dtype, T, return column_sums<T>(a, vec, device, st));
}

static int norm_check(const fa_norm* p) {
  if (!p) return FA_E_ARG;
  if (!train_dtype(p->dtype) || (p->weight_dtype != p->dtype && p->weight_dtype != FA_F32))
    return FA_E_DTYPE;
  if (p->rows <= 0 || p->width <= 0 || p->width > (1 << 24) || p->rows > (1ll << 40))
    return FA_E_SHAPE;
  if (!(p->eps >= 0.0)) return FA_E_ARG;
  return FA_OK;
}

static bool at_item(const void* p, int dtype) {
  return reinterpret_cast<size_t>(p) % item_size(dtype) == 0;
}

static NormArgs norm_args(const fa_norm& p) {
  NormArgs a = {};
  a.x = p.x;
  a.x_row = p.x_stride;
  a.res = p.residual;
  a.res_row = p.residual_stride;
  a.w = p.weight;
  a.b = p.bias;
  a.w32 = p.weight_dtype == FA_F32;
  a.w_vec = reinterpret_cast<size_t>(p.weight) % 16 == 0 && reinterpret_cast<size_t>(p.bias) % 16 == 0;
  a.stats = reinterpret_cast<float2*>(p.stats);
  a.codes = static_cast<unsigned char*>(p.codes);
  a.ranges = p.ranges;
  a.rows = p.rows;
  a.width = p.width;
  a.groups = (int)groups8(p.width);
  a.eps = (float)p.eps;
  a.inv_width = 1.f / (float)p.width;
  return a;
}

// Rows of whole units on every lane, with weights of the operands' type that lie so.
static RowKind kind_of(const NormArgs& a, bool vec, int item, RowShape shape) {
  if (!vec) return ODD;
  const bool weights = (!a.w && !a.b) || (a.w_vec && (item == 4 || !a.w32));
  return weights && a.width == 256 * shape.wpr * shape.e ? FULL : VECTORS;
}

// Forward, a block has one row of its own: blocks that stayed and took rows in turn, two
// a multiprocessor's worth of warps, took 342 us where these took 272 (65280 x 4096
// bfloat16, both on the path of VECTORS; FULL takes 211), since all of a block's warps
// load, sum and store at the same time.
template <typename T, RowKind KIND, int E>
static void norm_launch(const NormArgs& a, int wpr, cudaStream_t st) {
  const int rpb = wpr == 1 ? 4 : 1;
  const unsigned threads = 32 * wpr * rpb;
  const unsigned grid = (unsigned)((a.rows + rpb - 1) / rpb);
  if (threads > 256)
    norm_kernel<T, KIND, E, 1024><<<grid, threads, 0, st>>>(a, wpr);
  else
    norm_kernel<T, KIND, E, 256><<<grid, threads, 0, st>>>(a, wpr);
}
template <typename T, int E>
static void norm_launch(const NormArgs& a, int wpr, bool vec, cudaStream_t st) {
  const RowKind kind = kind_of(a, vec, sizeof(T), RowShape{wpr, E});
  if (kind == FULL) norm_launch<T, FULL, E>(a, wpr, st);
  else if (kind == VECTORS) norm_launch<T, VECTORS, E>(a, wpr, st);
  else norm_launch<T, ODD, E>(a, wpr, st);
}

template <typename T>
static int norm_run(const NormArgs& a, bool vec, int device, cudaStream_t st) {
  const RowShape shape = forward_shape(a.width);
  if (shape.wpr && a.rows < 1ll << 31) {
    if (shape.e == 1) norm_launch<T, 1>(a, shape.wpr, vec, st);
    else if (shape.e == 2) norm_launch<T, 2>(a, shape.wpr, vec, st);
    else norm_launch<T, 4>(a, shape.wpr, vec, st);
    FAB_LAUNCH_CHECK();
    return FA_OK;
  }
  const unsigned grid = (unsigned)std::min(a.rows, (long long)sm_count(device) * 8);
  if (vec)
    norm_rows_kernel<T, true><<<grid, 256, 0, st>>>(a);
  else
    norm_rows_kernel<T, false><<<grid, 256, 0, st>>>(a);
  FAB_LAUNCH_CHECK();
  return FA_OK;
}

int norm_impl(const fa_norm* p, void* y, void* sum, int device, cudaStream_t st) {
  if (const int rc = norm_check(p)) return rc;
  if (!p->x || !y || (p->codes && !p->ranges)) return FA_E_ARG;
  NormArgs a = norm_args(*p);
  a.y = y;
  a.sum = sum;
  const int item = item_size(p->dtype);
  for (const void* q : {a.x, a.res, (const void*)y, (const void*)sum})
    if (!at_item(q, p->dtype)) return FA_E_ARG;
  for (const void* q : {a.w, a.b})
    if (!at_item(q, p->weight_dtype)) return FA_E_ARG;
  if (reinterpret_cast<size_t>(a.codes) % 16 || reinterpret_cast<size_t>(a.ranges) % 8 ||
      reinterpret_cast<size_t>(a.stats) % 8)
    return FA_E_ARG;
  const bool vec = whole8(a.x, a.x_row, a.rows, a.width, item) &&
                   (!a.res || whole8(a.res, a.res_row, a.rows, a.width, item)) &&
                   whole8(y, a.width, a.rows, a.width, item) &&
                   (!sum || whole8(sum, a.width, a.rows, a.width, item));
  FAB_DEVICE_SCOPE(device);
  FAB_FOR_TYPE(p->dtype, T, return norm_run<T>(a, vec, device, st));
}

template <typename T, int E, int NT, bool CODES>
static void norm_grad_launch(const NormArgs& a, int wpr, RowKind kind, cudaStream_t st) {
  const unsigned grid = (unsigned)a.splits;
  if (kind == FULL)
    norm_grad_kernel<T, FULL, E, CODES, NT><<<grid, NT, 0, st>>>(a, wpr);
  else if (kind == VECTORS)
    norm_grad_kernel<T, VECTORS, E, CODES, NT><<<grid, NT, 0, st>>>(a, wpr);
  else
    norm_grad_kernel<T, ODD, E, CODES, NT><<<grid, NT, 0, st>>>(a, wpr);
}
template <typename T, int E, int NT>
static int norm_grad_launch(NormArgs& a, int wpr, bool vec, int device, cudaStream_t st) {
  a.splits = backward_blocks(a.rows, NT / 32 / wpr, NT, device);
  const RowKind kind = kind_of(a, vec, sizeof(T), RowShape{wpr, E});
  if (a.codes)
    norm_grad_launch<T, E, NT, true>(a, wpr, kind, st);
  else
    norm_grad_launch<T, E, NT, false>(a, wpr, kind, st);
  FAB_LAUNCH_CHECK();
  return a.dw || a.db ? column_join<T>(a, st) : FA_OK;
}

template <typename T>
static int norm_grad_run(NormArgs& a, bool vec, int device, cudaStream_t st) {
  const RowShape shape = backward_shape(a.width, sizeof(T));
  if constexpr (sizeof(T) == 4)
    if (shape.e == 1 && shape.wpr > 8)
      return norm_grad_launch<T, 1, 512>(a, shape.wpr, vec, device, st);
  if (shape.e == 1) return norm_grad_launch<T, 1, 256>(a, shape.wpr, vec, device, st);
  if (shape.wpr > 8) return norm_grad_launch<T, 2, 512>(a, shape.wpr, vec, device, st);
  if (shape.wpr) return norm_grad_launch<T, 2, 256>(a, shape.wpr, vec, device, st);
  const unsigned grid = (unsigned)std::min(a.rows, (long long)sm_count(device) * 8);
  if (vec)
    norm_grad_rows_kernel<T, true><<<grid, 256, 0, st>>>(a);
  else
    norm_grad_rows_kernel<T, false><<<grid, 256, 0, st>>>(a);
  FAB_LAUNCH_CHECK();
  return a.dw || a.db ? column_sums<T>(a, vec, device, st) : FA_OK;
}

int norm_backward_impl(const fa_norm* p, const void* dy, long long dy_row, const void* ds,
                       long long ds_row, void* dx, void* dw, void* db, void* ws, size_t ws_bytes,
                       int device, cudaStream_t st) {
  if (const int rc = norm_check(p)) return rc;
  if (!p->stats || !dy || !dx || (!p->x && !p->codes) || (p->codes && !p->ranges)) return FA_E_ARG;
  NormArgs a = norm_args(*p);
  a.res = nullptr;
  a.y = dx;
  a.dy = dy;
  a.dy_row = dy_row;
  a.ds = ds;
  a.ds_row = ds_row;
  a.dw = dw;
  a.db = db;
  a.part = static_cast<float*>(ws);
  if (a.codes) a.x = nullptr;
  const int item = item_size(p->dtype);
  for (const void* q : {a.x, dy, ds, (const void*)dx})
    if (!at_item(q, p->dtype)) return FA_E_ARG;
  for (const void* q : {a.w, (const void*)dw, (const void*)db})
    if (!at_item(q, p->weight_dtype)) return FA_E_ARG;
  if (reinterpret_cast<size_t>(a.codes) % 16 || reinterpret_cast<size_t>(a.ranges) % 8 ||
      reinterpret_cast<size_t>(a.stats) % 8 || reinterpret_cast<size_t>(ws) % 16)
    return FA_E_ARG;
  if ((dw || db) && (!ws || ws_bytes < norm_ws_bytes(a.rows, a.width, device))) return FA_E_ARG;
  const bool vec = (!a.x || whole8(a.x, a.x_row, a.rows, a.width, item)) &&
                   whole8(dy, dy_row, a.rows, a.width, item) &&
                   (!ds || whole8(ds, ds_row, a.rows, a.width, item)) &&
                   whole8(dx, a.width, a.rows, a.width, item);
  FAB_DEVICE_SCOPE(device);
  FAB_FOR_TYPE(p->dtype, T, return norm_grad_run<T>(a, vec, device, st));
}

}  // namespace fab
