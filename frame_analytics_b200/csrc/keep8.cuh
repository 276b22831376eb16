// Activations in 8 bits: the format, and what the kernels that write or read it
// share.
//
// A row of `width` values is cut into groups of 64 (the last may be short).  A
// group holds its lowest value lo, a power of two s and a code of 8 bits for
// each value:
//   d = fl32(max - lo),  s = 2^e,  e the smallest integer >= -126 with d <= 255 s,
//   q = rint(fl32(x - lo) / s),   and stands for   fl_T(fl32(q s + lo)).
// The difference is rounded once, the division by s is exact, so the codes follow
// from the values alone, whatever computes them.  |value - x| is at most s / 2,
// which is below d / 255 (or 2^-127), and the step of T.  A group whose d is not
// finite (an infinity, a NaN, a spread past float32's range) has a NaN for s and
// stands for NaNs.  A code that would stand for more than T's largest number is
// one lower.
//
// Lowest values instead of a symmetric range: a row with a common offset keeps
// its precision, and one-sided activations use all 256 codes.  A power of two:
// the code of a value does not depend on how a division was rounded, and q s is
// exact in bfloat16 and float16 operands of the tensor cores.  64 values: the
// 4 bytes of a group (8 in float32) are 6 % of its 64 codes.
//
// In memory: codes [rows][64 G] bytes, G = ceil(width / 64), those past the width
// zero; ranges [rows][G]: for 16-bit types a word with lo in the low half and s as
// bfloat16 (exact) in the high half, for float32 the pair (lo, s).
#pragma once

#include "train.cuh"

namespace fab {

constexpr int kGroup8 = 64;
constexpr float kMagic8 = 8388608.f;  // 2^23: the low byte of 2^23 + q is q

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The least float32 that rounds past T's largest finite number.
template <typename T> struct Over;
template <> struct Over<float> {
  static __device__ __forceinline__ float v() { return __uint_as_float(0x7f800000u); }
};
template <> struct Over<f16_t> {
  static __device__ __forceinline__ float v() { return 65520.f; }
};
template <> struct Over<bf16_t> {
  static __device__ __forceinline__ float v() { return __uint_as_float(0x7f7f8000u); }
};

// A value rounded to T, as float32.
template <typename T>
__device__ __forceinline__ float round_to(float f) {
  return Ld<T>::f(St<T>::v(f));
}

// The range of one group.
struct Range8 {
  float lo, s;
};
template <typename T> struct RangeBits { typedef unsigned type; };
template <> struct RangeBits<float> { typedef float2 type; };

__device__ __forceinline__ float2 range_bits(const Range8& r, float) {
  return make_float2(r.lo, r.s);
}
template <typename T>
__device__ __forceinline__ unsigned range_bits(const Range8& r, T) {
  return (unsigned)St<T>::v(r.lo).bits | (__float_as_uint(r.s) & 0xffff0000u);
}
__device__ __forceinline__ Range8 range_of(float2 b, float) { return {b.x, b.y}; }
template <typename T>
__device__ __forceinline__ Range8 range_of(unsigned b, T) {
  T lo;
  lo.bits = (unsigned short)(b & 0xffffu);
  return {Ld<T>::f(lo), __uint_as_float(b & 0xffff0000u)};
}

// Range and codes of a group spread over 8 neighbouring lanes, 8 values a lane of
// which the first n exist.  Every lane of the warp takes part.
template <typename T>
__device__ __forceinline__ uint2 encode8(const float (&x)[8], int n, Range8* r) {
  float a = __uint_as_float(0x7f800000u), b = __uint_as_float(0xff800000u);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) {
      a = min_nan(a, x[i]);
      b = max_nan(b, x[i]);
    }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    a = min_nan(a, __shfl_xor_sync(0xffffffffu, a, o));
    b = max_nan(b, __shfl_xor_sync(0xffffffffu, b, o));
  }
  const float d = b - a;
  const unsigned u = __float_as_uint(d);
  r->lo = a;
  if (!(d < __uint_as_float(0x7f800000u))) {
    r->s = __uint_as_float(0x7fc00000u);
    return make_uint2(0u, 0u);
  }
  // 255 is 1.9921875 x 2^7
  const int e = max((int)(u >> 23) - 7 + (int)((u & 0x7fffffu) > 0x7f0000u), 1);
  r->s = __uint_as_float((unsigned)e << 23);
  const float inv = __uint_as_float((unsigned)(254 - e) << 23);
  float top = kMagic8 + 255.f;
  const float high = fmaf(d, inv, kMagic8);
  if (fmaf(high - kMagic8, r->s, a) >= Over<T>::v()) top = high - 1.f;
  unsigned q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    q[i] = i < n ? __float_as_uint(fminf(fmaf(x[i] - a, inv, kMagic8), top)) : 0u;
  uint2 c;
  c.x = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
  c.y = __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410);
  return c;
}

// The 8 values that codes stand for, rounded to T.
template <typename T>
__device__ __forceinline__ void decode8(uint2 c, const Range8& r, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const unsigned w = i < 4 ? c.x : c.y;
    const float q = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 | (i & 3))) - kMagic8;
    x[i] = round_to<T>(fmaf(q, r.s, r.lo));
  }
}

// ---------------------------------------------------------------------------
// 8 values of a row
// ---------------------------------------------------------------------------

// The first n of 8 values at p; VEC: n is 8 or 0 and p is 16-byte aligned.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, int n, float (&x)[8]) {
  if constexpr (VEC) {
    if (n) {
      if constexpr (sizeof(T) == 4) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(p));
        const float4 b = __ldg(reinterpret_cast<const float4*>(p) + 1);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
      } else {
        const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
        const unsigned w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          T v;
          v.bits = (unsigned short)(w[i / 2] >> (16 * (i & 1)));
          x[i] = Ld<T>::f(v);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = i < n ? Ld<T>::f(ldro(p + i)) : 0.f;
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, int n, const float (&x)[8]) {
  if constexpr (VEC) {
    if (!n) return;
    if constexpr (sizeof(T) == 4) {
      reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
      reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
      unsigned w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = (unsigned)St<T>::v(x[2 * i]).bits | ((unsigned)St<T>::v(x[2 * i + 1]).bits << 16);
      *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = St<T>::v(x[i]);
  }
}

// 8 values as they lie in memory: loaded early, widened where they are used.
template <typename T> struct Raw8 {
  uint4 v;
};
template <> struct Raw8<float> {
  float4 a, b;
};
template <typename T, bool VEC>
__device__ __forceinline__ Raw8<T> raw8(const T* p, int n) {
  Raw8<T> r;
  if constexpr (sizeof(T) == 4) {
    r.a = r.b = make_float4(0.f, 0.f, 0.f, 0.f);
    if constexpr (VEC) {
      if (n) {
        r.a = __ldg(reinterpret_cast<const float4*>(p));
        r.b = __ldg(reinterpret_cast<const float4*>(p) + 1);
      }
    } else {
      float x[8];
      load8<T, false>(p, n, x);
      r.a = make_float4(x[0], x[1], x[2], x[3]);
      r.b = make_float4(x[4], x[5], x[6], x[7]);
    }
  } else {
    r.v = make_uint4(0u, 0u, 0u, 0u);
    if constexpr (VEC) {
      if (n) r.v = __ldg(reinterpret_cast<const uint4*>(p));
    } else {
      unsigned w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[i] = 2 * i < n ? (unsigned)ldro(p + 2 * i).bits : 0u;
        if (2 * i + 1 < n) w[i] |= (unsigned)ldro(p + 2 * i + 1).bits << 16;
      }
      r.v = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  return r;
}
__device__ __forceinline__ void widen8(const Raw8<float>& r, float (&x)[8]) {
  x[0] = r.a.x; x[1] = r.a.y; x[2] = r.a.z; x[3] = r.a.w;
  x[4] = r.b.x; x[5] = r.b.y; x[6] = r.b.z; x[7] = r.b.w;
}
template <typename T>
__device__ __forceinline__ void widen8(const Raw8<T>& r, float (&x)[8]) {
  const unsigned w[4] = {r.v.x, r.v.y, r.v.z, r.v.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    T v;
    v.bits = (unsigned short)(w[i / 2] >> (16 * (i & 1)));
    x[i] = Ld<T>::f(v);
  }
}

// Whether rows at p are whole aligned vectors of 8.
static inline bool whole8(const void* p, long long row_stride, long long rows, int width,
                          int item) {
  return width % 8 == 0 && reinterpret_cast<size_t>(p) % 16 == 0 &&
         (rows <= 1 || row_stride * item % 16 == 0);
}

static inline long long groups8(int width) { return ((long long)width + kGroup8 - 1) / kGroup8; }
static inline int item_size(int dtype) { return dtype == FA_F32 ? 4 : 2; }
static inline bool train_dtype(int dtype) {
  return dtype == FA_F16 || dtype == FA_BF16 || dtype == FA_F32;
}

// FN<T>(args...) for the type of a dtype code.
#define FAB_FOR_TYPE(DTYPE, T, ...)                         \
  do {                                                      \
    if ((DTYPE) == FA_F32) { typedef float T; __VA_ARGS__; } \
    else if ((DTYPE) == FA_F16) { typedef f16_t T; __VA_ARGS__; } \
    else { typedef bf16_t T; __VA_ARGS__; }                 \
  } while (0)

}  // namespace fab
