// Activations in 8 bits: packing, unpacking, and the activation function whose
// backward pass reads its packed input.  keep8.cuh has the format.
//
//   gelu(x) = x Phi(x),             d = Phi(x) + x phi(x)
//   or      x (1 + tanh u) / 2,     u = sqrt(2/pi) (x + 0.044715 x^3)
//
// Each kernel reads its operands once and writes its outputs once; 8 lanes hold
// a group of 64, so a group's range costs three shuffles.  Measured on one B200, 65280 x
// 4096 bfloat16: packing 128 us and unpacking 130 us (0.98 and 0.96 of the copy rate),
// gelu with packing 229 us and its gradient 238 us (0.90 and 0.87), the tanh form 213 and
// 211 us (0.97).  float32 gelu is bound by normcdff and expf (0.5 of the copy rate), rows
// that are not whole vectors by their loads and stores of single values (0.35 to 0.55).
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
  long long per_row;    // units of a row; 0 where the rows join to one long one
  unsigned inv;         // 1 / per_row, see rows8
  int shift;
  int width;
};

enum { OP_PACK, OP_UNPACK, OP_GELU, OP_GELU_PACK, OP_GELU_GRAD };

__device__ __forceinline__ float2 exp2_fast(float2 v) {
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(v.x));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(v.y));
  return v;
}
__device__ __forceinline__ float2 over(float2 v) {  // 1 / v
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(v.x));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(v.y));
  return v;
}
constexpr float kTanhIn = 0.7978845608028654f;   // sqrt(2 / pi)
constexpr float kCube = 0.044715f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kBell = 0.3989422804014327f;     // 1 / sqrt(2 pi)
constexpr float kLog2Bell = -1.3257480647361593f;

// Results of 16 bits.  The upper tail of the normal distribution is Q(a) = F(a) exp(-a^2 / 2),
// a >= 0; returned is F(a) = t (c0 + ... + c6 t^6), t = 1 / (1 + 0.36 a).  The seven numbers
// make the largest RELATIVE error over 0 <= a <= 14 least (a linear program over 3000
// points, in float64): 8.7e-7, 1.1e-6 with float32's roundings, a 450th of float16's half
// step.  Relative, since far out a value or a slope is nothing but this tail: one that is
// right to 1e-7 absolutely (Abramowitz and Stegun's 7.1.26) leaves no digit of a slope at
// -6.  normcdff and expf take three times the instructions, which bound these kernels.
struct Tail {
  float2 t, p;                  // F = t p
};
// `s`: a factor of p.
__device__ __forceinline__ Tail tail_factor(float2 a, float s) {
  const float2 t = over(__ffma2_rn(a, both(0.36f), both(1.f)));
  float2 p = __ffma2_rn(t, both(s * 0.0470595174f), both(s * -0.179774687f));
  p = __ffma2_rn(p, t, both(s * 0.180965707f));
  p = __ffma2_rn(p, t, both(s * 0.0265429329f));
  p = __ffma2_rn(p, t, both(s * 0.139720857f));
  p = __ffma2_rn(p, t, both(s * 0.141772315f));
  p = __ffma2_rn(p, t, both(s * 0.143713057f));
  return {t, p};
}

// (1 + tanh u) / 2 = 1 / (1 + exp(-2 u)); `sq` is x^2, held where x^3 would overflow.
__device__ __forceinline__ float tanh_exp(float x, float sq) {
  return expf(-x * fmaf(sq, 2.f * kTanhIn * kCube, 2.f * kTanhIn));
}
__device__ __forceinline__ float tanh_factor(float x, float sq) {
  return 1.f / (1.f + tanh_exp(x, sq));
}
// f = (1 + tanh u) / 2 and f (1 - f), the latter without the rounding of an f near one
// (which x u' then enlarges: 1.8e-7 of a slope's size instead of 7e-8): 1 - f = exp(-2 u) f.
__device__ __forceinline__ float2 tanh_pair(float x, float sq) {
  const float e = fminf(tanh_exp(x, sq), 1e38f), f = 1.f / (1.f + e);
  return make_float2(f, f * (e * f));
}
__device__ __forceinline__ float2 tanh_factor_fast(float2 x, float2 sq) {
  const float2 u = __ffma2_rn(sq, both(-2.f * kTanhIn * kLog2e * kCube), both(-2.f * kTanhIn * kLog2e));
  return over(__fadd2_rn(both(1.f), exp2_fast(__fmul2_rn(x, u))));
}
__device__ __forceinline__ float2 square(float2 x) {
  const float2 s = __fmul2_rn(x, x);
  return make_float2(fminf(s.x, 1e12f), fminf(s.y, 1e12f));
}

// `FAST`: for results of 16 bits.  Below -64 the value is zero; an infinity or a NaN
// passes as such.
template <bool TANH, bool FAST>
__device__ __forceinline__ float2 gelu_value(float2 x) {
  if constexpr (TANH) {
    const float2 sq = square(x);
    const float2 m = make_float2(max_nan(x.x, -64.f), max_nan(x.y, -64.f));
    if constexpr (FAST) return __fmul2_rn(m, tanh_factor_fast(x, sq));
    return make_float2(m.x * tanh_factor(x.x, sq.x), m.y * tanh_factor(x.y, sq.y));
  } else if constexpr (FAST) {
    // x Phi(x) = max(x, 0) - a Q(a), a = |x|, Q the upper tail
    const float2 a = make_float2(min_nan(fabsf(x.x), 64.f), min_nan(fabsf(x.y), 64.f));
    const float2 c = __fmul2_rn(a, both(-0.5f * kLog2e));
    const Tail f = tail_factor(a, 1.f);
    const float2 q = __fmul2_rn(__fmul2_rn(f.t, f.p), exp2_fast(__fmul2_rn(c, a)));
    return make_float2(fmaf(-a.x, q.x, max_nan(x.x, 0.f)), fmaf(-a.y, q.y, max_nan(x.y, 0.f)));
  } else {
    return make_float2(max_nan(x.x, -64.f) * normcdff(x.x), max_nan(x.y, -64.f) * normcdff(x.y));
  }
}
template <bool TANH, bool FAST>
__device__ __forceinline__ float2 gelu_slope(float2 x) {
  if constexpr (TANH) {
    const float2 sq = square(x);
    float2 f, g;                // f + x f (1 - f) 2 u'
    if constexpr (FAST) {
      f = tanh_factor_fast(x, sq);
      g = __ffma2_rn(f, make_float2(-f.x, -f.y), f);
    } else {
      const float2 a = tanh_pair(x.x, sq.x), b = tanh_pair(x.y, sq.y);
      f = make_float2(a.x, b.x);
      g = make_float2(a.y, b.y);
    }
    const float2 u = __ffma2_rn(sq, both(6.f * kTanhIn * kCube), both(2.f * kTanhIn));
    return __ffma2_rn(__fmul2_rn(x, g), u, f);
  } else if constexpr (FAST) {
    // with a = |x| and v = a phi(a) - Q(a) = (a - t p / bell) bell exp(-a^2 / 2): 1 + v, or
    // below zero -v, so that nothing is taken from a one there
    const unsigned sx = __float_as_uint(x.x), sy = __float_as_uint(x.y);
    const float2 a = make_float2(fabsf(x.x), fabsf(x.y));
    const float2 e = exp2_fast(__ffma2_rn(__fmul2_rn(x, both(-0.5f * kLog2e)), x, both(kLog2Bell)));
    const Tail f = tail_factor(a, -1.f / kBell);
    const float2 v = __fmul2_rn(__ffma2_rn(f.t, f.p, a), e);
    const float2 one = make_float2(__uint_as_float(0x3f800000u & ~(unsigned)((int)sx >> 31)),
                                   __uint_as_float(0x3f800000u & ~(unsigned)((int)sy >> 31)));
    return __fadd2_rn(make_float2(__uint_as_float(__float_as_uint(v.x) ^ (sx & 0x80000000u)),
                                  __uint_as_float(__float_as_uint(v.y) ^ (sy & 0x80000000u))), one);
  } else {
    return make_float2(normcdff(x.x) + x.x * (kBell * expf(-0.5f * x.x * x.x)),
                       normcdff(x.y) + x.y * (kBell * expf(-0.5f * x.y * x.y)));
  }
}

// A thread has kUnits units at a time, whose loads are all under way before the first
// is used.  WHOLE: rows that join to one long one, and all of the block's units in it:
// addresses are one base each, which leaves the kernels to their bytes (65280 x 4096
// bfloat16: packing 143 -> 128 us, gelu 264 -> 221 us).  Otherwise a row's place takes
// one multiplication (`inv`).
constexpr int kUnits = 4;

template <typename T, int OP, bool VEC, bool TANH, bool WHOLE>
__device__ __forceinline__ void rows8_units(const Rows8& a, long long u0, Turn8<T>* turn) {
  typedef typename RangeBits<T>::type Bits;
  constexpr bool FAST = sizeof(T) == 2;
  constexpr bool READS = OP == OP_UNPACK || OP == OP_GELU_GRAD;   // codes
  const long long u1 = u0 + threadIdx.x;
  uint2* const codes = reinterpret_cast<uint2*>(a.codes) + u1;
  Bits* const ranges = reinterpret_cast<Bits*>(a.ranges) + u1 / 8;
  const T* const x0 = reinterpret_cast<const T*>(a.x) + (WHOLE ? u1 * 8 : 0);
  T* const y0 = reinterpret_cast<T*>(a.y) + (WHOLE ? u1 * 8 : 0);
  Raw8<T> raw[kUnits];
  uint2 code[kUnits];
  Bits bits[kUnits];
  int n[kUnits];
  long long at[kUnits];         // of this unit in y
#pragma unroll
  for (int k = 0; k < kUnits; ++k) {
    const long long u = u1 + k * 256;
    const bool in = WHOLE || u < a.units;
    const T* from = x0 + k * 2048;
    n[k] = 8;
    at[k] = k * 2048;
    if constexpr (!WHOLE) {
      n[k] = 0;
      at[k] = 0;
      from = x0;
      if (in) {
        long long row = 0, c = u * 8;
        n[k] = 8;
        if (a.per_row) {
          row = a.units <= 0x7fffffffll ? (long long)(__umulhi((unsigned)u, a.inv) >> a.shift)
                                        : u / a.per_row;
          c = (u - row * a.per_row) * 8;
          n[k] = (int)max(0ll, min(8ll, a.width - c));
        }
        at[k] = row * a.y_row + c;
        from = x0 + row * a.x_row + c;
      }
    }
    if constexpr (READS) {
      code[k] = in ? __ldg(codes + k * 256) : make_uint2(0u, 0u);
      bits[k] = in ? __ldg(ranges + k * 32) : Bits();
    }
    if constexpr (OP != OP_UNPACK) raw[k] = fetch8<T, VEC>(from, n[k], turn);
  }
#pragma unroll
  for (int k = 0; k < kUnits; ++k) {
    const bool in = WHOLE || u1 + k * 256 < a.units;
    F8 x;
    if constexpr (READS) {
      x = decode8<T>(code[k], range_of(bits[k], T()));
    } else {
      x = widen8(raw[k]);
    }
    if constexpr (OP == OP_PACK || OP == OP_GELU_PACK) {
      Range8 r;
      float lo, hi;
      extent8<VEC>(raw[k], n[k], &lo, &hi);
      const uint2 q = encode8<T, VEC>(x, n[k], lo, hi, &r);
      if (in) {
        codes[k * 256] = q;
        if ((threadIdx.x & 7) == 0) ranges[k * 32] = range_bits(r, T());
      }
    }
    if constexpr (OP == OP_GELU || OP == OP_GELU_PACK) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x.v[i] = gelu_value<TANH, FAST>(x.v[i]);
    }
    if constexpr (OP == OP_GELU_GRAD) {
      const F8 g = widen8(raw[k]);
#pragma unroll
      for (int i = 0; i < 4; ++i) x.v[i] = __fmul2_rn(g.v[i], gelu_slope<TANH, FAST>(x.v[i]));
    }
    if constexpr (OP != OP_PACK) store8<T, VEC>(y0 + at[k], n[k], x, turn);
  }
}

template <typename T, int OP, bool VEC, bool TANH>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 4 : 3) rows8_kernel(const Rows8 a) {
  __shared__ __align__(16) Turn8<T> turns[VEC ? 1 : 8];
  Turn8<T>* const turn = turns + (VEC ? 0 : threadIdx.x / 32);
  // whole warps stay together: a row is a multiple of 8 units, a warp's 32 may span rows
  const long long step = (long long)gridDim.x * (256 * kUnits);
  for (long long u0 = (long long)blockIdx.x * (256 * kUnits); u0 < a.units; u0 += step) {
    if (VEC && a.per_row == 0 && u0 + 256 * kUnits <= a.units)
      rows8_units<T, OP, VEC, TANH, VEC>(a, u0, turn);
    else
      rows8_units<T, OP, VEC, TANH, false>(a, u0, turn);
  }
}

template <typename T, int OP, bool TANH>
static int rows8_run(const Rows8& a, bool vec, int device, cudaStream_t st) {
  // 4 blocks a multiprocessor run at once (3 of float32).  Up to 16 times as many share the
  // units, so that a slow one holds up little at the end: 65280 x 4096 bfloat16, packing and
  // unpacking 145 and 137 us with 8 blocks a multiprocessor, 137 and 135 with 16, 127 and 129
  // with 64, 129 and 125 without a limit; gelu's gradient 236, 234, 236 and 240.
  const long long blocks =
      std::min((a.units + 256 * kUnits - 1) / (256 * kUnits), (long long)sm_count(device) * 64);
  if (vec)
    rows8_kernel<T, OP, true, TANH><<<(unsigned)blocks, 256, 0, st>>>(a);
  else
    rows8_kernel<T, OP, false, TANH><<<(unsigned)blocks, 256, 0, st>>>(a);
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
  // u / per_row for u < 2^31: with 2^s >= per_row, (u ceil(2^(31 + s) / per_row)) >> (31 + s)
  a.shift = 0;
  while ((1ll << a.shift) < a.per_row) ++a.shift;
  a.inv = (unsigned)(((1ull << (31 + a.shift)) + a.per_row - 1) / a.per_row);
  a.shift -= 1;                 // the high word is 32 of the 31 + s
  const bool vec = (!x || whole8(x, x_row, rows, width, item)) &&
                   (!y || whole8(y, y_row, rows, width, item));
  if (width % kGroup8 == 0 && (!x || rows == 1 || x_row == width) &&
      (!y || rows == 1 || y_row == width))
    a.per_row = 0;
  FAB_DEVICE_SCOPE(device);
  FAB_FOR_TYPE(dtype, T, switch (op) {
    case OP_PACK: return rows8_run<T, OP_PACK, false>(a, vec, device, st);
    case OP_UNPACK: return rows8_run<T, OP_UNPACK, false>(a, vec, device, st);
    case OP_GELU:
      return tanh_form ? rows8_run<T, OP_GELU, true>(a, vec, device, st)
                       : rows8_run<T, OP_GELU, false>(a, vec, device, st);
    case OP_GELU_PACK:
      return tanh_form ? rows8_run<T, OP_GELU_PACK, true>(a, vec, device, st)
                       : rows8_run<T, OP_GELU_PACK, false>(a, vec, device, st);
    default:
      return tanh_form ? rows8_run<T, OP_GELU_GRAD, true>(a, vec, device, st)
                       : rows8_run<T, OP_GELU_GRAD, false>(a, vec, device, st);
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
