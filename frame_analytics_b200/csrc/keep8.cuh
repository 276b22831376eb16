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

// ---------------------------------------------------------------------------
// 8 values of a row
// ---------------------------------------------------------------------------

// As float32 pairs: the arithmetic on them takes two values an instruction.
struct F8 {
  float2 v[4];
  __device__ __forceinline__ float at(int i) const { return i & 1 ? v[i / 2].y : v[i / 2].x; }
};
__device__ __forceinline__ float2 both(float f) { return make_float2(f, f); }
// Values from the n-th on become `f`.
__device__ __forceinline__ void fill_from(F8& x, int n, float f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (2 * i >= n) x.v[i].x = f;
    if (2 * i + 1 >= n) x.v[i].y = f;
  }
}
__device__ __forceinline__ float sum8(const F8& x) {
  const float2 s = __fadd2_rn(__fadd2_rn(x.v[0], x.v[1]), __fadd2_rn(x.v[2], x.v[3]));
  return s.x + s.y;
}

// As they lie in memory: loaded early, widened where they are used.
template <typename T> struct Raw8 {
  uint4 v;
};
template <> struct Raw8<float> {
  float4 a, b;
};

__device__ __forceinline__ F8 widen8(const Raw8<float>& r) {
  F8 x;
  x.v[0] = make_float2(r.a.x, r.a.y);
  x.v[1] = make_float2(r.a.z, r.a.w);
  x.v[2] = make_float2(r.b.x, r.b.y);
  x.v[3] = make_float2(r.b.z, r.b.w);
  return x;
}
__device__ __forceinline__ float2 widen2(unsigned w, bf16_t) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float2 widen2(unsigned w, f16_t) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <typename T>
__device__ __forceinline__ F8 widen8(const Raw8<T>& r) {
  F8 x;
  x.v[0] = widen2(r.v.x, T());
  x.v[1] = widen2(r.v.y, T());
  x.v[2] = widen2(r.v.z, T());
  x.v[3] = widen2(r.v.w, T());
  return x;
}

// Two values rounded to T, the first in the low half.
__device__ __forceinline__ unsigned narrow2(float2 v, bf16_t) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
  return *reinterpret_cast<const unsigned*>(&h);
}
__device__ __forceinline__ unsigned narrow2(float2 v, f16_t) {
  const __half2 h = __floats2half2_rn(v.x, v.y);
  return *reinterpret_cast<const unsigned*>(&h);
}
__device__ __forceinline__ Raw8<float> narrow8(const F8& x, float) {
  Raw8<float> r;
  r.a = make_float4(x.v[0].x, x.v[0].y, x.v[1].x, x.v[1].y);
  r.b = make_float4(x.v[2].x, x.v[2].y, x.v[3].x, x.v[3].y);
  return r;
}
template <typename T>
__device__ __forceinline__ Raw8<T> narrow8(const F8& x, T) {
  Raw8<T> r;
  r.v = make_uint4(narrow2(x.v[0], T()), narrow2(x.v[1], T()), narrow2(x.v[2], T()),
                   narrow2(x.v[3], T()));
  return r;
}
// Rounded to T and back.
__device__ __forceinline__ void round8(F8&, float) {}
template <typename T>
__device__ __forceinline__ void round8(F8& x, T) {
#pragma unroll
  for (int i = 0; i < 4; ++i) x.v[i] = widen2(narrow2(x.v[i], T()), T());
}

template <typename T>
__device__ __forceinline__ Raw8<T> zero8() {
  Raw8<T> r;
  if constexpr (sizeof(T) == 4) r.a = r.b = make_float4(0.f, 0.f, 0.f, 0.f);
  else r.v = make_uint4(0u, 0u, 0u, 0u);
  return r;
}
// A whole aligned vector.
template <typename T>
__device__ __forceinline__ Raw8<T> get8(const T* p) {
  Raw8<T> r;
  if constexpr (sizeof(T) == 4) {
    r.a = __ldg(reinterpret_cast<const float4*>(p));
    r.b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  } else {
    r.v = __ldg(reinterpret_cast<const uint4*>(p));
  }
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
// The first n of 8 values one by one, zeros behind them.
template <typename T>
__device__ __forceinline__ F8 few8(const T* p, int n) {
  F8 x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x.v[i].x = 2 * i < n ? Ld<T>::f(ldro(p + 2 * i)) : 0.f;
    x.v[i].y = 2 * i + 1 < n ? Ld<T>::f(ldro(p + 2 * i + 1)) : 0.f;
  }
  return x;
}

// Rows that are not whole aligned vectors: a warp's 256 values go through shared
// memory, so that neighbouring lanes touch neighbouring addresses (a lane's 8 values
// with 8 loads or stores of its own touch 16 sectors an instruction, 2 bytes of each).
// `p` is the lane's place, of which the first n values exist.
template <typename T>
struct Turn8 {
  T v[256];
};
// Whether the warp's values follow one another from lane 0's place; then how many.  Lanes
// whose values are fewer than 8 come last: rows padded to whole groups lie 8 values a lane
// too, but with gaps between them.
template <typename T>
__device__ __forceinline__ bool one_run(const T* p, int n, const T** first, int* count) {
  const unsigned long long at = reinterpret_cast<unsigned long long>(p);
  *first = reinterpret_cast<const T*>(__shfl_sync(0xffffffffu, at, 0));
  *count = __reduce_add_sync(0xffffffffu, n);
  const unsigned any = __ballot_sync(0xffffffffu, n > 0), all = __ballot_sync(0xffffffffu, n == 8);
  return (any & (any + 1u)) == 0u && ((any ^ all) & (any >> 1)) == 0u &&
         __all_sync(0xffffffffu, n == 0 || p == *first + (threadIdx.x & 31) * 8);
}
template <typename T>
__device__ __forceinline__ Raw8<T> gather8(const T* p, int n, Turn8<T>* t) {
  const int lane = threadIdx.x & 31;
  const T* first;
  int count;
  const bool run = one_run(p, n, &first, &count);
  __syncwarp();
  if (run) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      T v = T();
      if (i * 32 + lane < count) v = ldro(first + i * 32 + lane);
      t->v[i * 32 + lane] = v;
    }
  } else {
    const unsigned long long at = reinterpret_cast<unsigned long long>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int s = i * 4 + (lane >> 3), j = lane & 7;
      const T* const q = reinterpret_cast<const T*>(__shfl_sync(0xffffffffu, at, s)) + j;
      T v = T();
      if (j < __shfl_sync(0xffffffffu, n, s)) v = ldro(q);
      t->v[i * 32 + lane] = v;
    }
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
  const T* first;
  int count;
  const bool run = one_run<T>(p, n, &first, &count);
  __syncwarp();
  put8<T>(t->v + lane * 8, r);
  __syncwarp();
  if (run) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i * 32 + lane < count) const_cast<T*>(first)[i * 32 + lane] = t->v[i * 32 + lane];
  } else {
    const unsigned long long at = reinterpret_cast<unsigned long long>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int s = i * 4 + (lane >> 3), j = lane & 7;
      T* const q = reinterpret_cast<T*>(__shfl_sync(0xffffffffu, at, s)) + j;
      if (j < __shfl_sync(0xffffffffu, n, s)) *q = t->v[i * 32 + lane];
    }
  }
}
// Loads and stores of either kind; every lane of the warp takes part.  VEC: n is 8 or 0
// and p is 16-byte aligned.
template <typename T, bool VEC>
__device__ __forceinline__ Raw8<T> fetch8(const T* p, int n, Turn8<T>* t) {
  if constexpr (VEC) return n ? get8<T>(p) : zero8<T>();
  else return gather8<T>(p, n, t);
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, int n, const F8& x, Turn8<T>* t) {
  if constexpr (VEC) {
    if (n) put8<T>(p, narrow8(x, T()));
  } else {
    scatter8<T>(p, n, narrow8(x, T()), t);
  }
}

// ---------------------------------------------------------------------------
// groups
// ---------------------------------------------------------------------------

// Lowest and highest of the first n of 8 values; VEC: n is 8 or 0.  A NaN among them
// is both.
template <bool VEC>
__device__ __forceinline__ void extent8(const F8& x, int n, float* lo, float* hi) {
  *lo = __uint_as_float(0x7f800000u);
  *hi = __uint_as_float(0xff800000u);
  if (VEC && n == 0) return;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (VEC || i < n) {
      *lo = min_nan(*lo, x.at(i));
      *hi = max_nan(*hi, x.at(i));
    }
}
// The same of values as they lie: two 16-bit values an instruction.
template <bool VEC>
__device__ __forceinline__ void extent8(const Raw8<float>& r, int n, float* lo, float* hi) {
  extent8<VEC>(widen8(r), n, lo, hi);
}
__device__ __forceinline__ unsigned min2(unsigned a, unsigned b, bf16_t) {
  asm("min.NaN.bf16x2 %0, %0, %1;" : "+r"(a) : "r"(b));
  return a;
}
__device__ __forceinline__ unsigned max2(unsigned a, unsigned b, bf16_t) {
  asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(a) : "r"(b));
  return a;
}
__device__ __forceinline__ unsigned min2(unsigned a, unsigned b, f16_t) {
  asm("min.NaN.f16x2 %0, %0, %1;" : "+r"(a) : "r"(b));
  return a;
}
__device__ __forceinline__ unsigned max2(unsigned a, unsigned b, f16_t) {
  asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(a) : "r"(b));
  return a;
}
template <bool VEC, typename T>
__device__ __forceinline__ void extent8(const Raw8<T>& r, int n, float* lo, float* hi) {
  if (!VEC && n != 8) return extent8<false>(widen8(r), n, lo, hi);
  *lo = __uint_as_float(0x7f800000u);
  *hi = __uint_as_float(0xff800000u);
  if (n == 0) return;
  const float2 a = widen2(min2(min2(r.v.x, r.v.y, T()), min2(r.v.z, r.v.w, T()), T()), T());
  const float2 b = widen2(max2(max2(r.v.x, r.v.y, T()), max2(r.v.z, r.v.w, T()), T()), T());
  *lo = min_nan(a.x, a.y);
  *hi = max_nan(b.x, b.y);
}

// Range and codes of a group spread over 8 neighbouring lanes, 8 values a lane of
// which the first n exist and span [lo, hi].  Every lane of the warp takes part.
template <typename T, bool VEC>
__device__ __forceinline__ uint2 encode8(const F8& x, int n, float lo, float hi, Range8* r) {
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
  F8 q;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    q.v[i] = __ffma2_rn(__fadd2_rn(x.v[i], both(-lo)), both(inv), both(kMagic8));
  const float high = fmaf(d, inv, kMagic8);
  if (fmaf(high - kMagic8, r->s, lo) >= Over<T>::v()) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      q.v[i] = make_float2(fminf(q.v[i].x, high - 1.f), fminf(q.v[i].y, high - 1.f));
  }
  if (!VEC || n == 0) fill_from(q, n, kMagic8);
  unsigned h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    h[i] = __byte_perm(__float_as_uint(q.v[i].x), __float_as_uint(q.v[i].y), 0x0040);
  return make_uint2(__byte_perm(h[0], h[1], 0x5410), __byte_perm(h[2], h[3], 0x5410));
}

// The 8 values that codes stand for, rounded to T.
template <typename T>
__device__ __forceinline__ F8 decode8(uint2 c, const Range8& r) {
  F8 x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned w = i < 2 ? c.x : c.y, k = (i & 1) * 2;
    const float2 q = make_float2(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 | k)),
                                 __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7441 | k)));
    x.v[i] = __ffma2_rn(__fadd2_rn(q, both(-kMagic8)), both(r.s), both(r.lo));
  }
  round8(x, T());
  return x;
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
