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

// Lowest and highest of the first n of 8 values; VEC: n is 8 or 0.  A NaN among them
// is both.
template <bool VEC>
__device__ __forceinline__ void extent8(const float (&x)[8], int n, float* lo, float* hi) {
  *lo = __uint_as_float(0x7f800000u);
  *hi = __uint_as_float(0xff800000u);
  if (VEC && n == 0) return;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (VEC || i < n) {
      *lo = min_nan(*lo, x[i]);
      *hi = max_nan(*hi, x[i]);
    }
}

// Range and codes of a group spread over 8 neighbouring lanes, 8 values a lane of
// which the first n exist and span [lo, hi].  Every lane of the warp takes part.
template <typename T, bool VEC>
__device__ __forceinline__ uint2 encode8(const float (&x)[8], int n, float lo, float hi,
                                         Range8* r) {
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  const float d = hi - lo;
  const unsigned u = __float_as_uint(d);
  r->lo = lo;
  if (!(d < __uint_as_float(0x7f800000u))) {
    r->s = __uint_as_float(0x7fc00000u);
    return make_uint2(0u, 0u);
  }
  // 255 is 1.9921875 x 2^7
  const int e = max((int)(u >> 23) - 7 + (int)((u & 0x7fffffu) > 0x7f0000u), 1);
  r->s = __uint_as_float((unsigned)e << 23);
  const float inv = __uint_as_float((unsigned)(254 - e) << 23);
  float q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i] = fmaf(x[i] - lo, inv, kMagic8);
  const float high = fmaf(d, inv, kMagic8);
  if (fmaf(high - kMagic8, r->s, lo) >= Over<T>::v()) {
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = fminf(q[i], high - 1.f);
  }
  if (!VEC || n == 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i >= n) q[i] = kMagic8;
  }
  uint2 c;
#define FAB_LOW2(I) __byte_perm(__float_as_uint(q[I]), __float_as_uint(q[I + 1]), 0x0040)
  c.x = __byte_perm(FAB_LOW2(0), FAB_LOW2(2), 0x5410);
  c.y = __byte_perm(FAB_LOW2(4), FAB_LOW2(6), 0x5410);
#undef FAB_LOW2
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

// The extent of 8 values as they lie: two 16-bit values an instruction.
template <bool VEC>
__device__ __forceinline__ void extent8(const Raw8<float>& r, int n, float* lo, float* hi) {
  float x[8];
  widen8(r, x);
  extent8<VEC>(x, n, lo, hi);
}
template <bool VEC, typename T>
__device__ __forceinline__ void extent8(const Raw8<T>& r, int n, float* lo, float* hi) {
  if (!VEC && n != 8) {
    float x[8];
    widen8(r, x);
    extent8<false>(x, n, lo, hi);
    return;
  }
  *lo = __uint_as_float(0x7f800000u);
  *hi = __uint_as_float(0xff800000u);
  if (n == 0) return;
  unsigned a = r.v.x, b = r.v.x;
#define FAB_EXTENT(W)                                                                    \
  if constexpr (std::is_same<T, bf16_t>::value) {                                        \
    asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(a) : "r"(a), "r"(W));                        \
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(b) : "r"(b), "r"(W));                        \
  } else {                                                                               \
    asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(a) : "r"(a), "r"(W));                         \
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(b) : "r"(b), "r"(W));                         \
  }
  FAB_EXTENT(r.v.y)
  FAB_EXTENT(r.v.z)
  FAB_EXTENT(r.v.w)
#undef FAB_EXTENT
  T l, h;
  l.bits = (unsigned short)a;
  h.bits = (unsigned short)(a >> 16);
  *lo = min_nan(Ld<T>::f(l), Ld<T>::f(h));
  l.bits = (unsigned short)b;
  h.bits = (unsigned short)(b >> 16);
  *hi = max_nan(Ld<T>::f(l), Ld<T>::f(h));
}

// 8 values rounded to T, as they lie.
__device__ __forceinline__ Raw8<float> narrow8(const float (&x)[8], float) {
  Raw8<float> r;
  r.a = make_float4(x[0], x[1], x[2], x[3]);
  r.b = make_float4(x[4], x[5], x[6], x[7]);
  return r;
}
template <typename T>
__device__ __forceinline__ Raw8<T> narrow8(const float (&x)[8], T) {
  unsigned w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = (unsigned)St<T>::v(x[2 * i]).bits | ((unsigned)St<T>::v(x[2 * i + 1]).bits << 16);
  Raw8<T> r;
  r.v = make_uint4(w[0], w[1], w[2], w[3]);
  return r;
}
template <typename T>
__device__ __forceinline__ void put8(T* p, const Raw8<T>& r) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = r.a;
    reinterpret_cast<float4*>(p)[1] = r.b;
  } else {
    *reinterpret_cast<uint4*>(p) = r.v;
  }
}

// Rows that are not whole aligned vectors: a warp's 256 values go through shared
// memory, so that neighbouring lanes touch neighbouring addresses (a lane's 8 values
// with 8 loads or stores of its own touch 16 sectors an instruction, 2 bytes of each).
// `p` is the lane's place, of which the first n values exist.
template <typename T>
struct Turn8 {
  T v[256];
};
template <typename T>
__device__ __forceinline__ Raw8<T> gather8(const T* p, int n, Turn8<T>* t) {
  const int lane = threadIdx.x & 31;
  const unsigned long long at = reinterpret_cast<unsigned long long>(p);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int s = i * 4 + (lane >> 3), j = lane & 7;
    const T* const q = reinterpret_cast<const T*>(__shfl_sync(0xffffffffu, at, s)) + j;
    T v = T();
    if (j < __shfl_sync(0xffffffffu, n, s)) v = ldro(q);
    t->v[i * 32 + lane] = v;
  }
  __syncwarp();
  Raw8<T> r;
  if constexpr (sizeof(T) == 4) {
    r.a = reinterpret_cast<const float4*>(t->v + lane * 8)[0];
    r.b = reinterpret_cast<const float4*>(t->v + lane * 8)[1];
  } else {
    r.v = *reinterpret_cast<const uint4*>(t->v + lane * 8);
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void scatter8(T* p, int n, const Raw8<T>& r, Turn8<T>* t) {
  const int lane = threadIdx.x & 31;
  const unsigned long long at = reinterpret_cast<unsigned long long>(p);
  __syncwarp();
  put8<T>(t->v + lane * 8, r);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int s = i * 4 + (lane >> 3), j = lane & 7;
    T* const q = reinterpret_cast<T*>(__shfl_sync(0xffffffffu, at, s)) + j;
    if (j < __shfl_sync(0xffffffffu, n, s)) *q = t->v[i * 32 + lane];
  }
}
// Either way of loading and storing; every lane of the warp takes part.
template <typename T, bool VEC>
__device__ __forceinline__ Raw8<T> fetch8(const T* p, int n, Turn8<T>* t) {
  if constexpr (VEC) return raw8<T, true>(p, n); else return gather8<T>(p, n, t);
}
template <typename T, bool VEC>
__device__ __forceinline__ void put8(T* p, int n, const float (&x)[8], Turn8<T>* t) {
  if constexpr (VEC) {
    if (n) put8<T>(p, narrow8(x, T()));
  } else {
    scatter8<T>(p, n, narrow8(x, T()), t);
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
