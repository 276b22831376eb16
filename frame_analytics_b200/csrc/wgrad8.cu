// Weight gradient of a product y = x W^T from the packed copy of x (keep8.cuh):
//   dW[m, k] = sum over rows t of dy[t, m] x^[t, k],   db[m] = sum over t of dy[t, m],
// where x^ are the values that the codes stand for.
#include <algorithm>

#include "keep8.cuh"

namespace fab {

int bias_grad_impl(const void* g, long long g_row, void* db, int dtype, long long rows, int width,
                   void* ws, size_t ws_bytes, int device, cudaStream_t st);
size_t norm_ws_bytes(long long rows, int width, int device);

struct WgradArgs {
  const void* dy;
  long long dy_row;
  const unsigned char* codes;
  const void* ranges;
  long long rows;
  int inputs, outputs, groups;
  void* dw;                     // [outputs][inputs]
};

constexpr int kWgTile = 64;     // rows and columns of a block's part of dW
constexpr int kWgRows = 16;     // rows t at a time

// One block to a 64 x 64 tile in float32 on the ordinary lanes.
template <typename T>
__global__ void __launch_bounds__(256) wgrad_lanes_kernel(const WgradArgs a) {
  __shared__ float sa[kWgRows][kWgTile + 4], sb[kWgRows][kWgTile + 4];
  const int m0 = blockIdx.y * kWgTile, k0 = blockIdx.x * kWgTile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (long long t0 = 0; t0 < a.rows; t0 += kWgRows) {
    __syncthreads();
    for (int i = threadIdx.x; i < kWgRows * kWgTile; i += 256) {
      const int t = i / kWgTile, m = i % kWgTile;
      float v = 0.f;
      if (t0 + t < a.rows && m0 + m < a.outputs)
        v = Ld<T>::f(ldro(reinterpret_cast<const T*>(a.dy) + (t0 + t) * a.dy_row + m0 + m));
      sa[t][m] = v;
    }
    if (threadIdx.x < kWgRows * 8) {
      const int t = threadIdx.x / 8, u = threadIdx.x % 8;
      float x[8] = {};
      if (t0 + t < a.rows) {
        const long long g = (t0 + t) * a.groups + k0 / kGroup8;
        decode8<T>(__ldg(reinterpret_cast<const uint2*>(a.codes) + g * 8 + u),
                   range_of(__ldg(reinterpret_cast<const typename RangeBits<T>::type*>(a.ranges) + g),
                            T()), x);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) sb[t][u * 8 + i] = x[i];
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < kWgRows; ++t) {
      float p[4], q[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[i] = sa[t][ty * 4 + i];
        q[i] = sb[t][tx * 4 + i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(p[i], q[j], acc[i][j]);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int m = m0 + ty * 4 + i, k = k0 + tx * 4 + j;
      if (m < a.outputs && k < a.inputs)
        reinterpret_cast<T*>(a.dw)[(long long)m * a.inputs + k] = St<T>::v(acc[i][j]);
    }
}

size_t wgrad8_ws_bytes(long long rows, int inputs, int outputs, int dtype, int device) {
  (void)inputs;
  (void)dtype;
  return norm_ws_bytes(rows, outputs, device);
}

int wgrad8_impl(const void* dy, long long dy_row, const void* codes, const void* ranges, int dtype,
                long long rows, int inputs, int outputs, void* dw, void* db, void* ws,
                size_t ws_bytes, int device, cudaStream_t st) {
  if (!train_dtype(dtype)) return FA_E_DTYPE;
  if (rows <= 0 || inputs <= 0 || outputs <= 0 || rows > (1ll << 40) || inputs > (1 << 22) ||
      outputs > (1 << 22))
    return FA_E_SHAPE;
  const int item = item_size(dtype);
  if (!dy || (dw && (!codes || !ranges)) || reinterpret_cast<size_t>(dy) % item ||
      reinterpret_cast<size_t>(dw) % item || reinterpret_cast<size_t>(db) % item ||
      reinterpret_cast<size_t>(codes) % 16 || reinterpret_cast<size_t>(ranges) % 8 || !ws ||
      reinterpret_cast<size_t>(ws) % 16 ||
      ws_bytes < wgrad8_ws_bytes(rows, inputs, outputs, dtype, device))
    return FA_E_ARG;
  FAB_DEVICE_SCOPE(device);
  if (db)
    if (const int rc = bias_grad_impl(dy, dy_row, db, dtype, rows, outputs, ws, ws_bytes, device, st))
      return rc;
  if (!dw) return FA_OK;
  WgradArgs a;
  a.dy = dy;
  a.dy_row = dy_row;
  a.codes = static_cast<const unsigned char*>(codes);
  a.ranges = ranges;
  a.rows = rows;
  a.inputs = inputs;
  a.outputs = outputs;
  a.groups = (int)groups8(inputs);
  a.dw = dw;
  const dim3 grid((unsigned)((inputs + kWgTile - 1) / kWgTile),
                  (unsigned)((outputs + kWgTile - 1) / kWgTile));
  if (grid.y > 65535u) return FA_E_SHAPE;
  FAB_FOR_TYPE(dtype, T, wgrad_lanes_kernel<T><<<grid, 256, 0, st>>>(a));
  FAB_LAUNCH_CHECK();
  return FA_OK;
}

}  // namespace fab
