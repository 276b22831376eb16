// Orthogonalised updates: Newton-Schulz steps on a matrix over its Frobenius
// norm, and the optimiser step built on them.
//
//   X <- X / |X|_F  (a zero matrix stays zero),   then `steps` times
//   A = X X^T  (rows <= cols)  or  X^T X,   B = b A + c A^2,
//   X <- a X + B X             or  a X + X B,
// which maps every singular value s to s (a + b s^2 + c s^4).
//
// The optimiser step on a weight W with gradient G and momentum M:
//   M <- mu M + G,  U = G + mu M (Nesterov) or M,
//   W <- (1 - lr wd) W - lr scale O(U).
#include "train.cuh"

#include <algorithm>

namespace fab {

constexpr int kMats = 64;          // matrices of one launch sequence
constexpr int kNormBlocks = 32;    // partial sums of squares of one matrix

struct NsMat {
  const void* src;   // x, or the gradient
  void* dst;         // out, or the weight
  float* mom;        // momentum, or null
  long long x_off, a_off;  // offsets of X[2] and of A, B in floats
  long long src_row, dst_row;  // row strides
  int rows, cols;
  float step;                  // W <- decay W - step O
};

struct NsArgs {
  NsMat m[kMats];
  float* ws;
  double* part;      // [kMats][kNormBlocks]
  float mu;
  int nesterov;
  float decay;
};

__device__ __forceinline__ float nan_f() { return __int_as_float(0x7fffffff); }

// Updates the momentum and sums the squares of the update.
template <typename T>
__global__ void __launch_bounds__(256) ns_norm_kernel(const __grid_constant__ NsArgs a) {
  __shared__ double sm[32];
  const NsMat& m = a.m[blockIdx.y];
  const long long n = (long long)m.rows * m.cols;
  const T* src = reinterpret_cast<const T*>(m.src);
  double ss = 0;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += 256ll * gridDim.x) {
    const long long r = i / m.cols, c = i - r * m.cols;
    float u = Ld<T>::f(src[r * m.src_row + c]);
    if (m.mom) {
      const float v = fmaf(a.mu, m.mom[i], u);
      m.mom[i] = v;
      u = a.nesterov ? fmaf(a.mu, v, u) : v;
    }
    ss += (double)u * u;
  }
  ss = block_sum(ss, sm);
  if (threadIdx.x == 0) a.part[blockIdx.y * kNormBlocks + blockIdx.x] = ss;
}

template <typename T>
__global__ void __launch_bounds__(256) ns_pack_kernel(const __grid_constant__ NsArgs a) {
  const NsMat& m = a.m[blockIdx.y];
  const long long n = (long long)m.rows * m.cols;
  const T* src = reinterpret_cast<const T*>(m.src);
  double ss = 0;
  for (int i = 0; i < kNormBlocks; ++i) ss += a.part[blockIdx.y * kNormBlocks + i];
  const bool finite = ss <= 1.7e308;
  const double inv = ss > 0 ? 1.0 / sqrt(ss) : 0.0;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += 256ll * gridDim.x) {
    const long long r = i / m.cols, c = i - r * m.cols;
    float u = Ld<T>::f(src[r * m.src_row + c]);
    if (m.mom) {
      const float v = m.mom[i];
      u = a.nesterov ? fmaf(a.mu, v, u) : v;
    }
    a.ws[m.x_off + i] = finite ? (float)(u * inv) : nan_f();
  }
}

enum { NS_GRAM, NS_SQUARE, NS_APPLY, NS_FINAL };

// 64 x 64 outputs of one matrix; D[i][j] = sum_k P(i, k) Q(k, j).
template <int MODE, typename T>
__global__ void __launch_bounds__(256) ns_product_kernel(const __grid_constant__ NsArgs a, int cur,
                                                         float ca, float cb, float cc) {
  __shared__ float sp[16][65], sq[16][65];
  const NsMat& m = a.m[blockIdx.y];
  const bool tall = m.rows > m.cols;
  const int s = min(m.rows, m.cols);
  const long long n = (long long)m.rows * m.cols;
  const float* X = a.ws + m.x_off + cur * n;
  float* X2 = a.ws + m.x_off + (1 - cur) * n;
  float* A = a.ws + m.a_off;
  float* B = A + (long long)s * s;
  const int M = MODE <= NS_SQUARE ? s : m.rows, N = MODE <= NS_SQUARE ? s : m.cols;
  const int K = MODE == NS_GRAM ? max(m.rows, m.cols) : s;
  const int tn = (N + 63) / 64, tiles = ((M + 63) / 64) * tn;
  const float *P, *Q;
  long long pi, pk, qk, qj;  // strides
  if (MODE == NS_GRAM) {
    P = Q = X;
    pi = qj = tall ? 1 : m.cols;
    pk = qk = tall ? m.cols : 1;
  } else if (MODE == NS_SQUARE) {
    P = Q = A;
    pi = qk = s;
    pk = qj = 1;
  } else {
    P = tall ? X : B;
    Q = tall ? B : X;
    pi = tall ? m.cols : s;
    qk = tall ? s : m.cols;
    pk = qj = 1;
  }
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  for (int t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int i0 = t / tn * 64, j0 = t % tn * 64;
    float acc[4][4] = {};
    for (int k0 = 0; k0 < K; k0 += 16) {
      for (int e = threadIdx.x; e < 1024; e += 256) {
        const int kk = e & 15, ii = e >> 4;
        sp[kk][ii] = i0 + ii < M && k0 + kk < K ? P[(i0 + ii) * pi + (k0 + kk) * pk] : 0.f;
        sq[kk][ii] = j0 + ii < N && k0 + kk < K ? Q[(j0 + ii) * qj + (k0 + kk) * qk] : 0.f;
      }
      __syncthreads();
#pragma unroll
      for (int kk = 0; kk < 16; ++kk)
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int v = 0; v < 4; ++v)
            acc[u][v] = fmaf(sp[kk][ty + 16 * u], sq[kk][tx + 16 * v], acc[u][v]);
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int i = i0 + ty + 16 * u, j = j0 + tx + 16 * v;
        if (i >= M || j >= N) continue;
        const long long o = (long long)i * N + j;
        const float d = acc[u][v];
        if (MODE == NS_GRAM) A[o] = d;
        else if (MODE == NS_SQUARE) B[o] = fmaf(cb, A[o], cc * d);
        else if (MODE == NS_APPLY) X2[o] = fmaf(ca, X[o], d);
        else {
          const float y = fmaf(ca, X[o], d);
          T* w = reinterpret_cast<T*>(m.dst) + i * m.dst_row + j;
          *w = St<T>::v(m.mom ? fmaf(a.decay, Ld<T>::f(*w), -m.step * y) : y);
        }
      }
  }
}

static long long ns_floats(int rows, int cols) {
  const long long s = std::min(rows, cols);
  return 2ll * rows * cols + 2 * s * s;
}

static constexpr size_t kNsHead = sizeof(double) * kMats * kNormBlocks;

size_t ns_ws_bytes(const fa_matrix* m, int count, int dtype) {
  (void)dtype;
  long long most = 0;
  for (int i = 0; i < count; i += kMats) {
    long long f = 0;
    for (int j = i; j < std::min(count, i + kMats); ++j) f += ns_floats(m[j].rows, m[j].cols);
    most = std::max(most, f);
  }
  return kNsHead + 4 * (size_t)most;
}

template <typename T>
static int ns_run(NsArgs& a, int count, const double* coef, int steps, int device,
                  cudaStream_t st) {
  const unsigned y = (unsigned)count;
  int tiles = 1;
  for (int i = 0; i < count; ++i)
    tiles = std::max(tiles, ((a.m[i].rows + 63) / 64) * ((a.m[i].cols + 63) / 64));
  const unsigned gx = (unsigned)std::min(tiles, std::max(1, sm_count(device) * 8 / count));
  ns_norm_kernel<T><<<dim3(kNormBlocks, y), 256, 0, st>>>(a);
  ns_pack_kernel<T><<<dim3(kNormBlocks, y), 256, 0, st>>>(a);
  for (int k = 0; k < steps; ++k) {
    const float ca = (float)coef[3 * k], cb = (float)coef[3 * k + 1], cc = (float)coef[3 * k + 2];
    ns_product_kernel<NS_GRAM, T><<<dim3(gx, y), 256, 0, st>>>(a, k & 1, ca, cb, cc);
    ns_product_kernel<NS_SQUARE, T><<<dim3(gx, y), 256, 0, st>>>(a, k & 1, ca, cb, cc);
    if (k + 1 < steps)
      ns_product_kernel<NS_APPLY, T><<<dim3(gx, y), 256, 0, st>>>(a, k & 1, ca, cb, cc);
    else
      ns_product_kernel<NS_FINAL, T><<<dim3(gx, y), 256, 0, st>>>(a, k & 1, ca, cb, cc);
  }
  FAB_LAUNCH_CHECK();
  return FA_OK;
}

// Everything about a call that can be refused before the device is touched.
int ns_check(const fa_matrix* m, int count, int dtype, bool update) {
  if (!m || count <= 0) return FA_E_ARG;
  if (dtype != FA_F16 && dtype != FA_BF16 && dtype != FA_F32) return FA_E_DTYPE;
  for (int i = 0; i < count; ++i) {
    if (!m[i].src || !m[i].dst || (update && !m[i].momentum)) return FA_E_ARG;
    if (m[i].rows <= 0 || m[i].cols <= 0) return FA_E_SHAPE;
    if (m[i].src_row_stride < m[i].cols || m[i].dst_row_stride < m[i].cols) return FA_E_SHAPE;
  }
  return FA_OK;
}

int ns_impl(const fa_matrix* mats, int count, int dtype, const double* coef, int steps,
            bool update, double mu, int nesterov, double decay, void* ws, size_t ws_bytes,
            int device, cudaStream_t st) {
  if (!coef || !ws) return FA_E_ARG;
  if (steps < 1) return FA_E_SHAPE;
  for (int i0 = 0; i0 < count; i0 += kMats) {
    const int n = std::min(kMats, count - i0);
    NsArgs a{};
    a.part = reinterpret_cast<double*>(ws);
    a.ws = reinterpret_cast<float*>(static_cast<char*>(ws) + kNsHead);
    a.mu = (float)mu;
    a.nesterov = nesterov;
    a.decay = (float)decay;
    long long off = 0;
    for (int i = 0; i < n; ++i) {
      const fa_matrix& f = mats[i0 + i];
      NsMat& m = a.m[i];
      m.src = f.src;
      m.dst = f.dst;
      m.mom = update ? f.momentum : nullptr;
      m.rows = f.rows;
      m.cols = f.cols;
      m.src_row = f.src_row_stride;
      m.dst_row = f.dst_row_stride;
      m.step = (float)f.step;
      m.x_off = off;
      m.a_off = off + 2ll * f.rows * f.cols;
      off += ns_floats(f.rows, f.cols);
    }
    if (ws_bytes < kNsHead + 4 * (size_t)off) return FA_E_ARG;
    int rc;
    switch (dtype) {
      case FA_F16: rc = ns_run<f16_t>(a, n, coef, steps, device, st); break;
      case FA_BF16: rc = ns_run<bf16_t>(a, n, coef, steps, device, st); break;
      default: rc = ns_run<float>(a, n, coef, steps, device, st); break;
    }
    if (rc) return rc;
  }
  return FA_OK;
}

}  // namespace fab
