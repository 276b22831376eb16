// Activations in 8 bits: packing, unpacking, and the activation function whose
// backward pass reads its packed input.  keep8.cuh has the format.
//
//   gelu(x) = x Phi(x),             d = Phi(x) + x phi(x)
//   or      x (1 + tanh u) / 2,     u = sqrt(2/pi) (x + 0.044715 x^3)
//
// Each kernel reads its operands once and writes its outputs once; 8 lanes hold
// a group of 64, so a group's range costs three shuffles.
#include <algorithm>

#include "keep8.cuh"

namespace fab {

// Rows of `width` values, walked in units of 8: a row has 8 units a group.
struct Rows8 {
  const void* x;        // values, or the gradient
  long long x_row;      // elements between rows
  void* y;              // values out
  long long y_row;
  unsigned char* codes;
  void* ranges;
  long long units;      // rows x per_row
  long long per_row;    // units of a row
  int width;
  int tanh_form;
};

enum { OP_PACK, OP_UNPACK, OP_GELU, OP_GELU_PACK, OP_GELU_GRAD };

__device__ __forceinline__ float gelu_value(float x, int tanh_form) {
  if (tanh_form) {
    const float u = 0.7978845608028654f * (x + 0.044715f * x * x * x);
    return 0.5f * x * (1.f + tanhf(u));
  }
  return x * normcdff(x);
}
__device__ __forceinline__ float gelu_slope(float x, int tanh_form) {
  if (tanh_form) {
    const float u = 0.7978845608028654f * (x + 0.044715f * x * x * x);
    const float t = tanhf(u);
    return 0.5f * (1.f + t) + 0.5f * x * (1.f - t * t) * 0.7978845608028654f *
                                  (1.f + 3.f * 0.044715f * x * x);
  }
  return normcdff(x) + x * (0.3989422804014327f * expf(-0.5f * x * x));
}

template <typename T, int OP, bool VEC>
__global__ void __launch_bounds__(256) rows8_kernel(const Rows8 a) {
  typedef typename RangeBits<T>::type Bits;
  // whole warps stay together: a row is a multiple of 8 units, a warp's 32 may span rows
  for (long long u0 = (long long)blockIdx.x * 256; u0 < a.units; u0 += (long long)gridDim.x * 256) {
    const long long u = u0 + threadIdx.x;
    const bool in = u < a.units;
    const long long row = in ? u / a.per_row : 0;
    const long long unit = in ? u - row * a.per_row : 0;
    const long long c = unit * 8;
    const int n = in ? (int)max(0ll, min(8ll, a.width - c)) : 0;
    uint2* const code = reinterpret_cast<uint2*>(a.codes) + u;
    Bits* const bits = reinterpret_cast<Bits*>(a.ranges) + u / 8;
    const T* const xp = reinterpret_cast<const T*>(a.x) + row * a.x_row + c;
    T* const yp = reinterpret_cast<T*>(a.y) + row * a.y_row + c;
    float x[8];
    if constexpr (OP == OP_PACK || OP == OP_GELU || OP == OP_GELU_PACK) {
      load8<T, VEC>(xp, n, x);
      if constexpr (OP != OP_GELU) {
        Range8 r;
        const uint2 q = encode8<T>(x, n, &r);
        if (in) {
          *code = q;
          if ((u & 7) == 0) *bits = range_bits(r, T());
        }
      }
      if constexpr (OP != OP_PACK) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = gelu_value(x[i], a.tanh_form);
        store8<T, VEC>(yp, n, x);
      }
    } else if (in) {
      decode8<T>(*code, range_of(*bits, T()), x);
      if constexpr (OP == OP_GELU_GRAD) {
        float g[8];
        load8<T, VEC>(xp, n, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = g[i] * gelu_slope(x[i], a.tanh_form);
      }
      store8<T, VEC>(yp, n, x);
    }
  }
}

template <typename T, int OP>
static int rows8_run(const Rows8& a, bool vec, int device, cudaStream_t st) {
  const long long blocks = std::min((a.units + 255) / 256, (long long)sm_count(device) * 32);
  if (vec)
    rows8_kernel<T, OP, true><<<(unsigned)blocks, 256, 0, st>>>(a);
  else
    rows8_kernel<T, OP, false><<<(unsigned)blocks, 256, 0, st>>>(a);
  FAB_LAUNCH_CHECK();
  return FA_OK;
}

// One of the five passes; null codes where the pass has none.
static int rows8(int op, const void* x, long long x_row, void* y, long long y_row,
                 const void* codes, const void* ranges, int dtype, long long rows, int width,
                 int tanh_form, int device, cudaStream_t st) {
  if (!train_dtype(dtype)) return FA_E_DTYPE;
  if (rows <= 0 || width <= 0) return FA_E_SHAPE;
  const bool coded = op != OP_GELU;
  const int item = item_size(dtype);
  if ((op != OP_UNPACK && !x) || (op != OP_PACK && !y) || (coded && (!codes || !ranges)))
    return FA_E_ARG;
  if (reinterpret_cast<size_t>(x) % item || reinterpret_cast<size_t>(y) % item ||
      reinterpret_cast<size_t>(codes) % 16 || reinterpret_cast<size_t>(ranges) % 8)
    return FA_E_ARG;
  Rows8 a;
  a.x = x;
  a.x_row = x_row;
  a.y = y;
  a.y_row = y_row;
  a.codes = static_cast<unsigned char*>(const_cast<void*>(codes));
  a.ranges = const_cast<void*>(ranges);
  a.per_row = groups8(width) * 8;
  if (rows > (1ll << 62) / a.per_row) return FA_E_SHAPE;
  a.units = rows * a.per_row;
  a.width = width;
  a.tanh_form = tanh_form;
  const bool vec = (!x || whole8(x, x_row, rows, width, item)) &&
                   (!y || whole8(y, y_row, rows, width, item));
  FAB_DEVICE_SCOPE(device);
  FAB_FOR_TYPE(dtype, T, switch (op) {
    case OP_PACK: return rows8_run<T, OP_PACK>(a, vec, device, st);
    case OP_UNPACK: return rows8_run<T, OP_UNPACK>(a, vec, device, st);
    case OP_GELU: return rows8_run<T, OP_GELU>(a, vec, device, st);
    case OP_GELU_PACK: return rows8_run<T, OP_GELU_PACK>(a, vec, device, st);
    default: return rows8_run<T, OP_GELU_GRAD>(a, vec, device, st);
  });
}

int pack8_impl(const void* x, long long x_row, void* codes, void* ranges, int dtype,
               long long rows, int width, int device, cudaStream_t st) {
  return rows8(OP_PACK, x, x_row, nullptr, 0, codes, ranges, dtype, rows, width, 0, device, st);
}
int unpack8_impl(const void* codes, const void* ranges, void* y, long long y_row, int dtype,
                 long long rows, int width, int device, cudaStream_t st) {
  return rows8(OP_UNPACK, nullptr, 0, y, y_row, codes, ranges, dtype, rows, width, 0, device, st);
}
int gelu8_impl(const void* x, long long x_row, void* y, void* codes, void* ranges, int tanh_form,
               int dtype, long long rows, int width, int device, cudaStream_t st) {
  return rows8(codes ? OP_GELU_PACK : OP_GELU, x, x_row, y, width, codes, ranges, dtype, rows,
               width, tanh_form, device, st);
}
int gelu8_backward_impl(const void* g, long long g_row, const void* codes, const void* ranges,
                        void* dx, int tanh_form, int dtype, long long rows, int width, int device,
                        cudaStream_t st) {
  return rows8(OP_GELU_GRAD, g, g_row, dx, width, codes, ranges, dtype, rows, width, tanh_form,
               device, st);
}

}  // namespace fab
