// Pieces shared by the training-step operators (query/key norm, orthogonalised
// updates).
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace fab {

// Rounding stores, the counterparts of Ld<T>.
template <typename T> struct St;
template <> struct St<float> {
  static __device__ __forceinline__ float v(float f) { return f; }
};
template <> struct St<f16_t> {
  static __device__ __forceinline__ f16_t v(float f) {
    f16_t o;
    o.bits = __half_as_ushort(__float2half_rn(f));
    return o;
  }
};
template <> struct St<bf16_t> {
  static __device__ __forceinline__ bf16_t v(float f) {
    bf16_t o;
    o.bits = __bfloat16_as_ushort(__float2bfloat16_rn(f));
    return o;
  }
};

// A vector register type of so many bytes.
template <int BYTES> struct RawOf;
template <> struct RawOf<16> { typedef uint4 type; };
template <> struct RawOf<8> { typedef uint2 type; };

}  // namespace fab
