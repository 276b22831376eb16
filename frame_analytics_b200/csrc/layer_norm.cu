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
// The variance is summed about the mean (not as a difference of squares, which a
// common offset would cancel); all sums are float32.  dw and db are summed in a
// fixed order without atomics, so they are the same bits on every run.
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
  float eps;
  // weight gradients
  float* part;                  // [splits][2][width] partial sums
  void *dw, *db;                // or null
  int splits;
};

// n weights from column c; `none` where there are none.
template <typename T, bool VEC>
__device__ __forceinline__ void weights8(const NormArgs& a, const void* w, int c, int n, float none,
                                         float (&x)[8]) {
  if (!w) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = none;
  } else if (a.w32) {
    const float* p = reinterpret_cast<const float*>(w) + c;
    if (VEC && a.w_vec) load8<float, true>(p, n, x); else load8<float, false>(p, n, x);
  } else {
    const T* p = reinterpret_cast<const T*>(w) + c;
    if (VEC && a.w_vec) load8<T, true>(p, n, x); else load8<T, false>(p, n, x);
  }
}

// s of 8 columns, from the sum that this thread wrote earlier or from the inputs.
template <typename T, bool VEC>
__device__ __forceinline__ void input8(const NormArgs& a, long long row, int c, int n,
                                       float (&x)[8]) {
  load8<T, VEC>(reinterpret_cast<const T*>(a.x) + row * a.x_row + c, n, x);
  if (a.res) {
    float r[8];
    load8<T, VEC>(reinterpret_cast<const T*>(a.res) + row * a.res_row + c, n, r);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = round_to<T>(x[i] + r[i]);
  }
}

// s of 8 columns in the backward pass: kept, or from its codes.
template <typename T, bool VEC>
__device__ __forceinline__ void kept8(const NormArgs& a, long long row, int c, int n,
                                      float (&x)[8]) {
  if (!a.codes) return load8<T, VEC>(reinterpret_cast<const T*>(a.x) + row * a.x_row + c, n, x);
  const long long g = row * a.groups + c / kGroup8;
  const uint2 q = __ldg(reinterpret_cast<const uint2*>(a.codes + row * a.groups * kGroup8 + c));
  decode8<T>(q, range_of(__ldg(reinterpret_cast<const typename RangeBits<T>::type*>(a.ranges) + g),
                         T()), x);
}

// Rows that fit the registers of up to 32 warps: E units of 8 columns a lane, `wpr`
// warps a row, every byte read and written once.
template <typename T, bool VEC, int E, int NT>
__global__ void __launch_bounds__(NT) norm_kernel(const NormArgs a, int wpr) {
  __shared__ float sm[2][32];
  __shared__ __align__(16) Turn8<T> turns[VEC ? 1 : NT / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Turn8<T>* const turn = turns + (VEC ? 0 : warp);
  const int at = warp % wpr, first = warp - at;          // this warp in its row, the row's first
  const long long row = (long long)blockIdx.x * (blockDim.x / 32 / wpr) + warp / wpr;
  const bool in = row < a.rows;
  const int units = a.groups * 8;
  // s stays as it lies in memory and is widened for each of the three passes over it:
  // half the registers of float32 values, so twice the rows under way
  Raw8<T> s[E];
  int n[E];
  {
    Raw8<T> q[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = ((e * wpr + at) * 32 + lane) * 8;
      n[e] = in ? max(0, min(8, a.width - c)) : 0;
      s[e] = fetch8<T, VEC>(reinterpret_cast<const T*>(a.x) + row * a.x_row + c, n[e], turn);
      if (a.res)
        q[e] = fetch8<T, VEC>(reinterpret_cast<const T*>(a.res) + row * a.res_row + c, n[e], turn);
    }
    if (a.res) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float x[8], y[8];
        widen8(s[e], x);
        widen8(q[e], y);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] += y[i];
        s[e] = narrow8(x, T());
      }
    }
  }
  const auto row_sum = [&](float t, int k) {
    t = warp_sum(t);
    if (wpr == 1) return t;
    if (lane == 0) sm[k][warp] = t;
    __syncthreads();
    t = 0.f;
    for (int w = 0; w < wpr; ++w) t += sm[k][first + w];
    return t;
  };
  float t = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    float x[8];
    widen8(s[e], x);
#pragma unroll
    for (int i = 0; i < 8; ++i) t += x[i];
  }
  const float m = row_sum(t, 0) / (float)a.width;
  t = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (VEC && n[e] == 0) continue;
    float x[8];
    widen8(s[e], x);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (VEC || i < n[e]) t = fmaf(x[i] - m, x[i] - m, t);
  }
  const float r = 1.f / sqrtf(row_sum(t, 1) / (float)a.width + a.eps);
  if (a.stats && in && at == 0 && lane == 0) a.stats[row] = make_float2(m, r);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int u = (e * wpr + at) * 32 + lane, c = u * 8;
    float x[8];
    widen8(s[e], x);
    if (a.sum) put8<T, VEC>(reinterpret_cast<T*>(a.sum) + row * a.width + c, n[e], x, turn);
    if (a.codes) {
      Range8 range;
      float lo, hi;
      extent8<VEC>(s[e], n[e], &lo, &hi);
      const uint2 q = encode8<T, VEC>(x, n[e], lo, hi, &range);
      if (in && u < units) {
        reinterpret_cast<uint2*>(a.codes)[row * units + u] = q;
        if ((u & 7) == 0)
          reinterpret_cast<typename RangeBits<T>::type*>(a.ranges)[row * a.groups + u / 8] =
              range_bits(range, T());
      }
    }
    float w[8], b[8];
    weights8<T, VEC>(a, a.w, c, n[e], 1.f, w);
    weights8<T, VEC>(a, a.b, c, n[e], 0.f, b);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fmaf((x[i] - m) * r, w[i], b[i]);
    put8<T, VEC>(reinterpret_cast<T*>(a.y) + row * a.width + c, n[e], x, turn);
  }
}

// The backward pass of such rows: blocks stay and take rows in turn; a lane keeps the
// weight gradients of its columns in registers, the block adds its rows' at the end
// and writes one part.  x, dy and ds stay in registers as they lie in memory.
template <typename T, bool VEC, int E, bool CODES, int NT>
__global__ void __launch_bounds__(NT, 512 / NT) norm_grad_kernel(const NormArgs a, int wpr) {
  __shared__ float2 sm[2][NT / 32];
  __shared__ float join[NT / 32][32 * 9];
  __shared__ __align__(16) Turn8<T> turns[VEC ? 1 : NT / 32];
  typedef typename RangeBits<T>::type Bits;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Turn8<T>* const turn = turns + (VEC ? 0 : warp);
  const int at = warp % wpr, first = warp - at, rpb = NT / 32 / wpr;
  float dw[E][8] = {}, db[E][8] = {};
  // what a row's loads bring; the next row's are under way while this one's sums run
  struct Row {
    Raw8<T> x[E], g[E], s[E];
    uint2 code[E];
    Bits bits[E];
    float2 st;
  };
  const auto load = [&](long long row, Row& o) {
    const bool in = row < a.rows;
    if (!in) row = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int u = (e * wpr + at) * 32 + lane, c = u * 8, n = in ? max(0, min(8, a.width - c)) : 0;
      if constexpr (CODES) {
        o.code[e] = make_uint2(0u, 0u);
        o.bits[e] = Bits();
        if (n) {
          o.code[e] = __ldg(reinterpret_cast<const uint2*>(a.codes) + row * a.groups * 8 + u);
          o.bits[e] = __ldg(reinterpret_cast<const Bits*>(a.ranges) + row * a.groups + u / 8);
        }
      } else {
        o.x[e] = fetch8<T, VEC>(reinterpret_cast<const T*>(a.x) + row * a.x_row + c, n, turn);
      }
      o.g[e] = fetch8<T, VEC>(reinterpret_cast<const T*>(a.dy) + row * a.dy_row + c, n, turn);
      if (a.ds) o.s[e] = fetch8<T, VEC>(reinterpret_cast<const T*>(a.ds) + row * a.ds_row + c, n, turn);
    }
    o.st = in ? __ldg(a.stats + row) : make_float2(0.f, 0.f);
  };
  const long long step = (long long)gridDim.x * rpb;
  int half = 0;
  Row now, next;
  load((long long)blockIdx.x * rpb + warp / wpr, now);
  for (long long row0 = (long long)blockIdx.x * rpb; row0 < a.rows; row0 += step, half ^= 1) {
    const long long row = row0 + warp / wpr;
    const bool in = row < a.rows;
    load(row + step, next);
    const float2 st = now.st;
    float c1 = 0.f, c2 = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = ((e * wpr + at) * 32 + lane) * 8, n = in ? max(0, min(8, a.width - c)) : 0;
      if (VEC && n == 0) continue;
      float x[8], g[8], w[8];
      if constexpr (CODES) decode8<T>(now.code[e], range_of(now.bits[e], T()), x);
      else widen8(now.x[e], x);
      widen8(now.g[e], g);
      weights8<T, VEC>(a, a.w, c, n, 1.f, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float h = VEC || i < n ? (x[i] - st.x) * st.y : 0.f, gw = g[i] * w[i];
        dw[e][i] = fmaf(g[i], h, dw[e][i]);
        db[e][i] += g[i];
        c1 += gw;
        c2 = fmaf(gw, h, c2);
      }
    }
    c1 = warp_sum(c1);
    c2 = warp_sum(c2);
    if (wpr > 1) {
      if (lane == 0) sm[half][warp] = make_float2(c1, c2);
      __syncthreads();          // one a row: the next row's sums have the other half
      c1 = c2 = 0.f;
      for (int w = 0; w < wpr; ++w) {
        c1 += sm[half][first + w].x;
        c2 += sm[half][first + w].y;
      }
    }
    c1 /= (float)a.width;
    c2 /= (float)a.width;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = ((e * wpr + at) * 32 + lane) * 8, n = in ? max(0, min(8, a.width - c)) : 0;
      float x[8], g[8], w[8];
      if constexpr (CODES) decode8<T>(now.code[e], range_of(now.bits[e], T()), x);
      else widen8(now.x[e], x);
      widen8(now.g[e], g);
      weights8<T, VEC>(a, a.w, c, n, 1.f, w);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        x[i] = st.y * (fmaf(g[i], w[i], -c1) - (x[i] - st.x) * st.y * c2);
      if (a.ds) {
        widen8(now.s[e], g);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] += g[i];
      }
      put8<T, VEC>(reinterpret_cast<T*>(a.y) + row * a.width + c, n, x, turn);
    }
    now = next;
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
      for (int i = 0; i < 8; ++i) join[warp][lane * 9 + i] = k ? db[e][i] : dw[e][i];
      __syncthreads();
      for (int j = threadIdx.x; j < wpr * 256; j += NT) {
        const int w = j / 256, l = j % 256, col = (e * wpr + w) * 256 + l;
        float t = 0.f;
        for (int q = 0; q < rpb; ++q) t += join[q * wpr + w][l / 8 * 9 + l % 8];
        if (col < a.width) a.part[((long long)blockIdx.x * 2 + k) * a.width + col] = t;
      }
    }
}

// A block to a row, which it reads again for each of its sums (from the
// second-level cache): for rows that fit no block's registers.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) norm_rows_kernel(const NormArgs a) {
  __shared__ float sm[32];
  const int units = a.groups * 8;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    float t = 0.f, x[8];
    for (int u = threadIdx.x; u < units; u += 256) {
      const int c = u * 8, n = max(0, min(8, a.width - c));
      input8<T, VEC>(a, row, c, n, x);
#pragma unroll
      for (int i = 0; i < 8; ++i) t += x[i];
    }
    const float m = block_sum(t, sm) / (float)a.width;
    t = 0.f;
    for (int u = threadIdx.x; u < units; u += 256) {
      const int c = u * 8, n = max(0, min(8, a.width - c));
      input8<T, VEC>(a, row, c, n, x);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) t += (x[i] - m) * (x[i] - m);
    }
    const float r = 1.f / sqrtf(block_sum(t, sm) / (float)a.width + a.eps);
    if (a.stats && threadIdx.x == 0) a.stats[row] = make_float2(m, r);
    for (int u0 = 0; u0 < units; u0 += 256) {
      const int u = u0 + threadIdx.x, c = u * 8, n = max(0, min(8, a.width - c));
      float w[8], b[8];
      input8<T, VEC>(a, row, c, n, x);
      if (a.sum)
        store8<T, VEC>(reinterpret_cast<T*>(a.sum) + row * a.width + c, n, x);
      if (a.codes) {
        Range8 range;
        float lo, hi;
        extent8<VEC>(x, n, &lo, &hi);
        const uint2 q = encode8<T, VEC>(x, n, lo, hi, &range);
        if (u < units) {
          reinterpret_cast<uint2*>(a.codes)[row * units + u] = q;
          if ((u & 7) == 0)
            reinterpret_cast<typename RangeBits<T>::type*>(a.ranges)[row * a.groups + u / 8] =
                range_bits(range, T());
        }
      }
      weights8<T, VEC>(a, a.w, c, n, 1.f, w);
      weights8<T, VEC>(a, a.b, c, n, 0.f, b);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = fmaf((x[i] - m) * r, w[i], b[i]);
      store8<T, VEC>(reinterpret_cast<T*>(a.y) + row * a.width + c, n, x);
    }
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) norm_grad_rows_kernel(const NormArgs a) {
  __shared__ float sm[32];
  const int units = a.groups * 8;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float2 st = a.stats[row];
    float c1 = 0.f, c2 = 0.f, x[8], g[8], w[8];
    for (int u = threadIdx.x; u < units; u += 256) {
      const int c = u * 8, n = max(0, min(8, a.width - c));
      kept8<T, VEC>(a, row, c, n, x);
      load8<T, VEC>(reinterpret_cast<const T*>(a.dy) + row * a.dy_row + c, n, g);
      weights8<T, VEC>(a, a.w, c, n, 1.f, w);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) {
          c1 += g[i] * w[i];
          c2 += g[i] * w[i] * ((x[i] - st.x) * st.y);
        }
    }
    c1 = block_sum(c1, sm) / (float)a.width;
    c2 = block_sum(c2, sm) / (float)a.width;
    for (int u = threadIdx.x; u < units; u += 256) {
      const int c = u * 8, n = max(0, min(8, a.width - c));
      kept8<T, VEC>(a, row, c, n, x);
      load8<T, VEC>(reinterpret_cast<const T*>(a.dy) + row * a.dy_row + c, n, g);
      weights8<T, VEC>(a, a.w, c, n, 1.f, w);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        x[i] = st.y * (g[i] * w[i] - c1 - (x[i] - st.x) * st.y * c2);
      if (a.ds) {
        load8<T, VEC>(reinterpret_cast<const T*>(a.ds) + row * a.ds_row + c, n, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] += g[i];
      }
      store8<T, VEC>(reinterpret_cast<T*>(a.y) + row * a.width + c, n, x);
    }
  }
}

// Column sums dw, db of one part of the rows: a block has 256 columns, a warp
// every eighth row.  Without codes and x, db alone.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) column_sums_kernel(const NormArgs a) {
  __shared__ float sm[8][32 * 9];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = (blockIdx.x * 32 + lane) * 8, n = max(0, min(8, a.width - c));
  const bool hats = a.x || a.codes;
  float dw[8] = {}, db[8] = {};
  const long long step = (long long)gridDim.y * 8;
#pragma unroll 4
  for (long long row = blockIdx.y * 8ll + warp; row < a.rows; row += step) {
    float g[8], x[8];
    load8<T, VEC>(reinterpret_cast<const T*>(a.dy) + row * a.dy_row + c, n, g);
    if (hats && n) {
      const float2 st = __ldg(a.stats + row);
      kept8<T, VEC>(a, row, c, n, x);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) dw[i] += g[i] * ((x[i] - st.x) * st.y);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) db[i] += g[i];
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) sm[warp][lane * 9 + i] = k ? db[i] : dw[i];
    __syncthreads();
    const int col = blockIdx.x * 256 + threadIdx.x;
    if (col < a.width && (k || hats)) {
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

// Parts of the rows in the column sums: enough blocks for every multiprocessor,
// at least 8 rows to a warp.
static int column_splits(long long rows, int width, int device) {
  const int strips = (width + 255) / 256;
  const long long most = std::max(1ll, (rows + 63) / 64);
  return (int)std::min(most, (long long)std::max(1, sm_count(device) * 6 / strips));
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

size_t norm_ws_bytes(long long rows, int width, int device) {
  const int parts = std::max(column_splits(rows, width, device), 2 * sm_count(device));
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
  if (vec)
    column_sums_kernel<T, true><<<grid, 256, 0, st>>>(a);
  else
    column_sums_kernel<T, false><<<grid, 256, 0, st>>>(a);
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
  return a;
}

template <typename T, int E>
static void norm_launch(const NormArgs& a, int wpr, bool vec, cudaStream_t st) {
  const int rpb = wpr == 1 ? 4 : 1;
  const unsigned grid = (unsigned)((a.rows + rpb - 1) / rpb);
  const unsigned threads = 32 * wpr * rpb;
  if (E == 4 && threads > 512) {
    if (vec)
      norm_kernel<T, true, 4, 1024><<<grid, threads, 0, st>>>(a, wpr);
    else
      norm_kernel<T, false, 4, 1024><<<grid, threads, 0, st>>>(a, wpr);
  } else if (vec) {
    norm_kernel<T, true, E, 512><<<grid, threads, 0, st>>>(a, wpr);
  } else {
    norm_kernel<T, false, E, 512><<<grid, threads, 0, st>>>(a, wpr);
  }
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

template <typename T, int E, int NT>
static int norm_grad_launch(NormArgs& a, int wpr, bool vec, int device, cudaStream_t st) {
  a.splits = backward_blocks(a.rows, NT / 32 / wpr, NT, device);
  const unsigned grid = (unsigned)a.splits;
  if (a.codes && vec)
    norm_grad_kernel<T, true, E, true, NT><<<grid, NT, 0, st>>>(a, wpr);
  else if (a.codes)
    norm_grad_kernel<T, false, E, true, NT><<<grid, NT, 0, st>>>(a, wpr);
  else if (vec)
    norm_grad_kernel<T, true, E, false, NT><<<grid, NT, 0, st>>>(a, wpr);
  else
    norm_grad_kernel<T, false, E, false, NT><<<grid, NT, 0, st>>>(a, wpr);
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
