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
template <typename T>
__device__ __forceinline__ void weights8(const void* w, int w32, int c, int n, float none,
                                         float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = none;
    if (w && i < n)
      x[i] = w32 ? __ldg(reinterpret_cast<const float*>(w) + c + i)
                 : Ld<T>::f(ldro(reinterpret_cast<const T*>(w) + c + i));
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
        const uint2 q = encode8<T>(x, n, &range);
        if (u < units) {
          reinterpret_cast<uint2*>(a.codes)[row * units + u] = q;
          if ((u & 7) == 0)
            reinterpret_cast<typename RangeBits<T>::type*>(a.ranges)[row * a.groups + u / 8] =
                range_bits(range, T());
        }
      }
      weights8<T>(a.w, a.w32, c, n, 1.f, w);
      weights8<T>(a.b, a.w32, c, n, 0.f, b);
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
      weights8<T>(a.w, a.w32, c, n, 1.f, w);
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
      weights8<T>(a.w, a.w32, c, n, 1.f, w);
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
__global__ void __launch_bounds__(256) column_join_kernel(const NormArgs a) {
  __shared__ float sm[8][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
  void* const out = blockIdx.y ? a.db : a.dw;
  if (!out) return;
  float t = 0.f;
  if (col < a.width)
    for (int i = warp; i < a.splits; i += 8)
      t += a.part[((long long)i * 2 + blockIdx.y) * a.width + col];
  sm[warp][lane] = t;
  __syncthreads();
  if (warp || col >= a.width) return;
  t = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) t += sm[w][lane];
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

size_t norm_ws_bytes(long long rows, int width, int device) {
  return (size_t)column_splits(rows, width, device) * 2 * (size_t)width * sizeof(float);
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
  column_join_kernel<T><<<dim3((unsigned)((a.width + 31) / 32), 2), 256, 0, st>>>(a);
  FAB_LAUNCH_CHECK();
  return FA_OK;
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
  a.stats = reinterpret_cast<float2*>(p.stats);
  a.codes = static_cast<unsigned char*>(p.codes);
  a.ranges = p.ranges;
  a.rows = p.rows;
  a.width = p.width;
  a.groups = (int)groups8(p.width);
  a.eps = (float)p.eps;
  return a;
}

template <typename T>
static int norm_run(const NormArgs& a, bool vec, int device, cudaStream_t st) {
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

template <typename T>
static int norm_grad_run(NormArgs& a, bool vec, int device, cudaStream_t st) {
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
