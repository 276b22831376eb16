// Tensor-core pieces shared by the product kernels (sm_100a): TMA boxes, operand
// descriptors, tcgen05 products, single blocks or pairs, and tensor memory.
#pragma once

#include <cuda.h>

#include "mbar.cuh"

namespace fab {

constexpr int kBox = 64 * 128;     // bytes of a 64 x 64 box of 16-bit values

// PAIR: `bar` may be the other block's of the pair.
template <bool PAIR>
__device__ __forceinline__ void tma_box(unsigned dst, const CUtensorMap* map, int x, int y, int z,
                                        unsigned bar) {
  if constexpr (PAIR)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::"
        "bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(dst),
        "l"(reinterpret_cast<unsigned long long>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(dst),
        "l"(reinterpret_cast<unsigned long long>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}

// Shared-memory operand descriptor, 128-byte swizzle.  Rows along K (K-major):
// 128-byte rows, 8-row groups 1024 bytes apart.  Rows along the other axis
// (MN-major): 64-element blocks kBox apart, groups of 8 K rows 1024 bytes apart.
__device__ __forceinline__ unsigned long long operand(unsigned addr) {
  return (unsigned long long)((addr & 0x3ffffu) >> 4) |
         ((unsigned long long)(kBox >> 4) << 16) | ((unsigned long long)(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}

template <bool PAIR>
__device__ __forceinline__ void mma_f16(unsigned d, unsigned long long a, unsigned long long b,
                                        unsigned idesc, bool add) {
  if constexpr (PAIR)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((unsigned)add)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((unsigned)add)
        : "memory");
}
// Arrives when the products issued so far are complete; PAIR: in both blocks.
template <bool PAIR>
__device__ __forceinline__ void mma_commit(unsigned long long* bar) {
  if constexpr (PAIR)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
        "[%0], %1;\n" ::"r"(smem_u32(bar)), "h"((unsigned short)3)
        : "memory");
  else
    asm volatile(
        "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(
            smem_u32(bar))
        : "memory");
}
// The same shared address in the pair's first block, which issues the products.
__device__ __forceinline__ unsigned in_leader(unsigned addr) {
  unsigned r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;\n" : "=r"(r) : "r"(addr));
  return r;
}
template <bool PAIR>
__device__ __forceinline__ void arrive_leader(unsigned long long* bar) {
  if constexpr (PAIR)
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(
                     in_leader(smem_u32(bar)))
                 : "memory");
  else
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(smem_u32(bar)) : "memory");
}
// mbar_try for a barrier at which threads of the pair's other block arrive, too: what is
// acquired is then the whole cluster's.
template <bool PAIR>
__device__ __forceinline__ bool mbar_try_pair(unsigned a, unsigned parity) {
  if constexpr (!PAIR) return mbar_try(a, parity);
  unsigned done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(done)
      : "r"(a), "r"(parity)
      : "memory");
  return done != 0;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;\n" ::
                   : "memory");
}

// 32 accumulator columns of this thread's row.
__device__ __forceinline__ void tmem_load32(unsigned addr, float (&v)[32]) {
  unsigned* u = reinterpret_cast<unsigned*>(v);
  __syncwarp();
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
      "%30, %31}, [%32];\n"
      "tcgen05.wait::ld.sync.aligned;\n"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]),
        "=r"(u[7]), "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]),
        "=r"(u[14]), "=r"(u[15]), "=r"(u[16]), "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]),
        "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]), "=r"(u[25]), "=r"(u[26]), "=r"(u[27]),
        "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(addr)
      : "memory");
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                  const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn encode_tiled() {
  static const EncodeTiledFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) !=
            cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeTiledFn>(f);
  }();
  return fn;
}
// A tensor map in three dimensions, in the 128-byte swizzle; outside arrives as zeros.
static bool encode_map(CUtensorMap* map, CUtensorMapDataType type, const void* p,
                       const cuuint64_t (&dim)[3], const cuuint64_t (&stride)[2],
                       const cuuint32_t (&box)[3]) {
  const EncodeTiledFn fn = encode_tiled();
  if (!fn) return false;
  const cuuint32_t one[3] = {1, 1, 1};
  const auto encode = [&] {
    return fn(map, type, 3, const_cast<void*>(p), dim, stride, box, one,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  };
  if (encode()) return true;
  // The driver's call wants a context, which a thread that has launched nothing yet does
  // not have (autograd's, in the first backward pass); setting its device gives it one.
  int device;
  return cudaGetDevice(&device) == cudaSuccess && cudaSetDevice(device) == cudaSuccess && encode();
}

}  // namespace fab
