// Weight gradient of a product y = x W^T from the packed copy of x (keep8.cuh):
//   dW[m, k] = sum over rows t of dy[t, m] x^[t, k],   db[m] = sum over t of dy[t, m],
// where x^ are the values that the codes stand for.
//
// 16-bit types: tensor-core products of 256 x 256 tiles over pairs of blocks
// (tcgen05, cta_group::2), persistent, accumulators double-buffered in tensor
// memory.  dy arrives by TMA as it lies (its rows are the sum's axis: MN-major),
// the codes by TMA as bytes; eight warps turn a stage's codes into operand values
// in shared memory, in the layout that TMA would have written, while the tensor
// cores work on the stages before it.  Every value q s + lo is rounded once, as
// unpacking rounds it.  Where the tiles are fewer than the pairs of blocks, the
// rows are cut into parts whose float32 sums are joined in order.
#include <algorithm>
#include <atomic>

#include "keep8.cuh"
#include "tensor.cuh"

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
      uint2 q = make_uint2(0u, 0u);
      typename RangeBits<T>::type bits = {};
      if (t0 + t < a.rows) {
        const long long g = (t0 + t) * a.groups + k0 / kGroup8;
        q = __ldg(reinterpret_cast<const uint2*>(a.codes) + g * 8 + u);
        bits = __ldg(reinterpret_cast<const typename RangeBits<T>::type*>(a.ranges) + g);
      }
      const F8 x = decode8<T>(q, range_of(bits, T()));
#pragma unroll
      for (int i = 0; i < 8; ++i) sb[t][u * 8 + i] = x.at(i);
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

// ---------------------------------------------------------------------------
// 16-bit products on the tensor cores
// ---------------------------------------------------------------------------

constexpr int kTile = 256;      // rows and columns of a pair's tile
constexpr int kDepth = 64;      // of the sum's axis, a stage
constexpr int kHalf = 2 * kBox; // bytes of one block's 128 x 64 of an operand
constexpr int kRaw = kDepth * 128;  // bytes of a stage's codes
constexpr int kRanges = kDepth * 8; // and of their ranges, two groups a row
constexpr int kTurn = 4096;     // a warp's 32 x 64 of the result
constexpr int kPartFloats = 128 * 256;  // of one block's part of a tile

// D[m][n] = sum over k of A[m][k] B[n][k].
struct ProductArgs {
  CUtensorMap a, b, d;          // b: of the codes where they are packed
  int m, n, kb;                 // kb: stages of the whole sum
  int a_mn, b_mn;               // the operand lies with k as its rows
  int tiles_m, tiles_n, parts;
  const unsigned* ranges;
  long long rows;
  int groups;
  void* out;                    // [m][n]
  const void* bias;             // [n] or null
  int tma_out, bias_vec;
  float* part;
  unsigned* err;
};

template <bool PACKED>
struct Product {
  // Stages of the operands, and of the codes, which the writers read ahead of them.
  static constexpr int kStages = PACKED ? 5 : 6, kC = PACKED ? 4 : 0;
  static constexpr int kWriters = PACKED ? 8 : 0;   // warps that unpack
  static constexpr int kEpi = PACKED ? 4 : 8;       // warps of the epilogue
  static constexpr int kThreads = 128 + 32 * (kWriters + kEpi);
  static constexpr int kBAt = kStages * kHalf;      // offsets in shared memory
  static constexpr int kTurnAt = 2 * kBAt;
  static constexpr int kCodesAt = kTurnAt + kEpi * kTurn;
  static constexpr int kRangesAt = kCodesAt + kC * kRaw;
  static constexpr int kSmem = kRangesAt + kC * kRanges + 1024;
};

struct Work {
  int i0, j0, kb0, kb1, item;
};
// Items are numbered part by part; inside a part eight rows of tiles are walked
// column by column, so the tiles at work share operand panels in the L2 cache.
__device__ __forceinline__ bool work_of(const ProductArgs& a, int item, Work* w) {
  const int tiles = a.tiles_m * a.tiles_n;
  if (item >= tiles * a.parts) return false;
  const int part = item / tiles, tile = item - part * tiles;
  const int band = tile / (8 * a.tiles_n), in = tile - band * 8 * a.tiles_n;
  const int high = min(8, a.tiles_m - band * 8);
  w->i0 = (band * 8 + in % high) * kTile;
  w->j0 = in / high * kTile;
  w->kb0 = (int)((long long)a.kb * part / a.parts);
  w->kb1 = (int)((long long)a.kb * (part + 1) / a.parts);
  w->item = item;
  return true;
}

// Bounded waits that sleep.  Sixteen warps wait here at a time, and each poll of a
// barrier holds up the others' (a poll of a phase that was complete took 260 cycles
// when the waiting warps polled in a loop), so a poll may suspend its warp until the
// phase completes, or up to 2 ms.  The error word, in host memory, is looked at once in
// 16 such polls.
__device__ __forceinline__ bool mbar_sleep(unsigned a, unsigned parity) {
  unsigned done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n"
      " selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(done)
      : "r"(a), "r"(parity), "r"(2000000u)
      : "memory");
  return done != 0;
}
// Whether a phase is complete, without waiting.
__device__ __forceinline__ bool mbar_peek(unsigned long long* bar, unsigned parity) {
  unsigned done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return done != 0;
}
static __device__ __noinline__ void stage_wait_slow(unsigned a, unsigned parity, unsigned* err) {
  const unsigned long long t0 = globaltimer_ns();
  unsigned long long next = 1000000ull;
  for (unsigned i = 1;; ++i) {
    if (mbar_sleep(a, parity)) return;
    const unsigned long long t = globaltimer_ns() - t0;
    if ((i & 15u) != 0u || t < next) continue;
    next = t + 1000000ull;
    if (t > kWaitLimitNs || (err && *reinterpret_cast<volatile unsigned*>(err) != 0u)) {
      if (err) {
        *reinterpret_cast<volatile unsigned*>(err) = (unsigned)FA_E_TIMEOUT;
        __threadfence_system();
      }
      return;
    }
  }
}
__device__ __forceinline__ void stage_wait(unsigned long long* bar, unsigned parity,
                                           unsigned* err) {
  const unsigned a = smem_u32(bar);
  if (!mbar_sleep(a, parity)) stage_wait_slow(a, parity, err);
}

// A phase that the other block of the pair may complete.
__device__ __forceinline__ void wait_pair(unsigned long long* bar, unsigned parity, unsigned* err) {
  stage_wait(bar, parity, err);
  asm volatile("fence.acq_rel.cluster;\n" ::: "memory");
}

// A warp has written its share of a stage, here or in the other block of the pair.
// What it wrote is in its own block's shared memory and fence.proxy.async has handed
// it to the tensor cores; nothing else has to be ordered, and a release to the whole
// cluster here, a memory barrier of over a thousand cycles a stage, bounded the kernel
// (258 against 160 us for 16320 rows, 1024 x 4096).
__device__ __forceinline__ void arrive_written(unsigned long long* bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];\n" ::"r"(in_leader(smem_u32(bar)))
               : "memory");
}

// One lane polls, the others wait at the warp's barrier.
__device__ __forceinline__ void warp_wait(unsigned long long* bar, unsigned parity, unsigned* err) {
  if ((threadIdx.x & 31) == 0) stage_wait(bar, parity, err);
  __syncwarp();
}

// 16 codes to 16 operand values, two to a word.  The low bytes of 2^23 + q and of
// 1024 + q are q, and q has 8 bits: bfloat16 holds it exactly, as the high half of
// a float32.
template <typename T>
__device__ __forceinline__ void operands16(uint4 c, unsigned bits, uint4* out) {
  const unsigned in[4] = {c.x, c.y, c.z, c.w};
  unsigned o[8];
  const Range8 r = range_of(bits, T());
  if constexpr (std::is_same<T, bf16_t>::value) {
    const unsigned lo2 = __byte_perm(bits, 0u, 0x1010), s2 = __byte_perm(bits, 0u, 0x3232);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const unsigned w = in[i / 2], k = (i & 1) * 2;
      const float q0 = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 | k)) - kMagic8;
      const float q1 = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 | (k + 1))) - kMagic8;
      const unsigned q = __byte_perm(__float_as_uint(q0), __float_as_uint(q1), 0x7632);
      asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(o[i]) : "r"(q), "r"(s2), "r"(lo2));
    }
  } else if (r.s >= 5.9604644775390625e-8f) {  // 2^-24: float16 holds s
    const unsigned lo2 = __byte_perm(bits, 0u, 0x1010);
    const unsigned sh = __half_as_ushort(__float2half_rn(r.s)), s2 = sh | (sh << 16);
    const unsigned less = 0xe400e400u;  // -1024
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      unsigned q = __byte_perm(in[i / 2], 0x64646464u, i & 1 ? 0x4342 : 0x4140);
      asm("add.rn.f16x2 %0, %1, %2;" : "=r"(q) : "r"(q), "r"(less));
      asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(o[i]) : "r"(q), "r"(s2), "r"(lo2));
    }
  } else {  // spreads below 2^-16, and groups that are not finite
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      unsigned h[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float q = (float)((in[i / 2] >> (16 * (i & 1) + 8 * j)) & 255u);
        h[j] = St<T>::v(fmaf(q, r.s, r.lo)).bits;
      }
      o[i] = h[0] | (h[1] << 16);
    }
  }
  out[0] = make_uint4(o[0], o[1], o[2], o[3]);
  out[1] = make_uint4(o[4], o[5], o[6], o[7]);
}

template <typename T>
__device__ __forceinline__ unsigned pair_bits(float a, float b) {
  return narrow2(make_float2(a, b), T());
}

// A warp's 32 rows x 64 columns of the result, at (i, j), a row a lane; `turn` is
// 4 KB of shared memory of its own, rows of 128 bytes in the 128-byte swizzle.
template <typename T>
__device__ __forceinline__ void put_result(const ProductArgs& a, int i, int j, float (&v)[64],
                                           char* turn) {
  const int lane = threadIdx.x & 31;
  if (a.bias) {
    const T* b = reinterpret_cast<const T*>(a.bias) + j;
    if (a.bias_vec && j + 64 <= a.n) {
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const F8 x = widen8(get8<T>(b + 8 * q));
#pragma unroll
        for (int c = 0; c < 8; ++c) v[8 * q + c] += x.at(c);
      }
    } else {
#pragma unroll
      for (int c = 0; c < 64; ++c)
        if (j + c < a.n) v[c] += Ld<T>::f(ldro(b + c));
    }
  }
  // the buffer's last store has been read out of it
  asm volatile("cp.async.bulk.wait_group.read 0;\n" ::: "memory");
  __syncwarp();
#pragma unroll
  for (int q = 0; q < 8; ++q)
    *reinterpret_cast<uint4*>(turn + lane * 128 + (q ^ (lane & 7)) * 16) =
        make_uint4(pair_bits<T>(v[8 * q], v[8 * q + 1]), pair_bits<T>(v[8 * q + 2], v[8 * q + 3]),
                   pair_bits<T>(v[8 * q + 4], v[8 * q + 5]), pair_bits<T>(v[8 * q + 6], v[8 * q + 7]));
  if (a.tma_out) {
    fence_async_smem();
    __syncwarp();
    if (lane == 0) {
      asm volatile(
          "cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];\n"
          "cp.async.bulk.commit_group;\n" ::"l"(reinterpret_cast<unsigned long long>(&a.d)),
          "r"(j), "r"(i), "r"(0), "r"(smem_u32(turn))
          : "memory");
    }
  } else {
    __syncwarp();
    T* const out = reinterpret_cast<T*>(a.out);
    for (int r = 0; r < min(32, a.m - i); ++r) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = lane + 32 * h;
        if (j + c < a.n)
          out[(long long)(i + r) * a.n + j + c] = *reinterpret_cast<const T*>(
              turn + r * 128 + ((c / 8) ^ (r & 7)) * 16 + c % 8 * 2);
      }
    }
    __syncwarp();
  }
}

template <typename T, bool PACKED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Product<PACKED>::kThreads, 1)
    product_kernel(const __grid_constant__ ProductArgs a) {
  typedef Product<PACKED> P;
  constexpr int S = P::kStages, SC = PACKED ? P::kC : 1;
  extern __shared__ char smem_raw[];
  const unsigned smem0 = (smem_u32(smem_raw) + 1023u) & ~1023u;
  char* const smem = smem_raw + (smem0 - smem_u32(smem_raw));
  __shared__ unsigned long long full[S], empty[S], c_full[SC], c_empty[SC], tm_full[2],
      tm_empty[2], drain;
  __shared__ unsigned tmem_base;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = blockIdx.x & 1;
  const int first = blockIdx.x >> 1, step = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      // the copies' bytes, and a team of four writers in either block
      mbar_init(&full[i], 1 + (PACKED ? P::kWriters : 0));
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < SC; ++i) {
      mbar_init(&c_full[i], 1 + 32);  // the codes' copy, and a warp's copies of ranges
      mbar_init(&c_empty[i], PACKED ? P::kWriters / 2 : 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tm_full[i], 1);
      mbar_init(&tm_empty[i], 2 * P::kEpi);
    }
    mbar_init(&drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    fence_async_smem();
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(
                     smem_u32(&tmem_base))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n");
  }
  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
  __syncthreads();
  cluster_sync();
  asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
  const unsigned tmem = tmem_base;
  Work t;

  if (warp == 0) {
    if (lane == 0) {
      unsigned n = 0;
      for (int item = first; work_of(a, item, &t); item += step) {
        const int ia = t.i0 + rank * 128, jb = t.j0 + rank * 128;
        for (int kb = t.kb0; kb < t.kb1; ++kb, ++n) {
          const int s = n % S;
          if (n >= (unsigned)S) stage_wait(&empty[s], (n / S - 1) & 1, a.err);
          // both blocks' copies count on the first block's barrier
          const unsigned bar = in_leader(smem_u32(&full[s]));
          if (rank == 0) mbar_expect_tx(&full[s], 2 * (PACKED ? 1 : 2) * kHalf);
#pragma unroll
          for (int i = 0; i < 2; ++i)
            tma_box<true>(smem0 + s * kHalf + i * kBox, &a.a, a.a_mn ? ia + 64 * i : kb * kDepth,
                          a.a_mn ? kb * kDepth : ia + 64 * i, 0, bar);
          if constexpr (!PACKED) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
              tma_box<true>(smem0 + P::kBAt + s * kHalf + i * kBox, &a.b,
                            a.b_mn ? jb + 64 * i : kb * kDepth, a.b_mn ? kb * kDepth : jb + 64 * i,
                            0, bar);
          }
        }
      }
      // copies still in flight land before the block ends
      for (unsigned i = n > (unsigned)S ? n - S : 0; rank == 0 && i < n; ++i)
        stage_wait(&full[i % S], (i / S) & 1, a.err);
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      // float32 sums; both operands float16 or both bfloat16; 256 x 256 over the pair
      const unsigned kind = std::is_same<T, bf16_t>::value ? (1u << 7) | (1u << 10) : 0u;
      const unsigned idesc = (1u << 4) | kind | ((unsigned)a.a_mn << 15) |
                             ((unsigned)a.b_mn << 16) | ((unsigned)(kTile / 8) << 17) |
                             ((unsigned)(kTile / 16) << 24);
      // 16 of k further: 2 groups of 8 rows, or 32 bytes along a row
      const unsigned as = (a.a_mn ? 2048u : 32u) >> 4, bs = (a.b_mn ? 2048u : 32u) >> 4;
      unsigned n = 0, tile = 0;
      for (int item = first; work_of(a, item, &t); item += step, ++tile) {
        const int buf = tile & 1;
        if (tile >= 2) wait_pair(&tm_empty[buf], (tile / 2 - 1) & 1, a.err);
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        bool ready = false;
        for (int kb = t.kb0; kb < t.kb1; ++kb, ++n) {
          const int s = n % S;
          if (!ready) stage_wait(&full[s], (n / S) & 1, a.err);
          asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
          const unsigned long long p = operand(smem0 + s * kHalf),
                                   q = operand(smem0 + P::kBAt + s * kHalf);
#pragma unroll
          for (int k = 0; k < kDepth / 16; ++k) {
            mma_f16<true>(tmem + buf * 256, p + k * as, q + k * bs, idesc, kb > t.kb0 || k > 0);
            // the next stage is asked for while this one's products run: few are queued,
            // and a poll takes longer than the last of them
            if (k == 1) ready = kb + 1 < t.kb1 && mbar_peek(&full[(n + 1) % S], ((n + 1) / S) & 1);
          }
          mma_commit<true>(&empty[s]);
        }
        mma_commit<true>(&tm_full[buf]);
      }
      // products still in flight end before tensor memory is given back
      mma_commit<true>(&drain);
      stage_wait(&drain, 0, a.err);
    }
  } else if (PACKED && warp == 3) {
    // codes of a stage, and their ranges: 4 words a lane, zeros (operands of zero)
    // behind the last row
    unsigned n = 0;
    for (int item = first; work_of(a, item, &t); item += step) {
      const int jb = t.j0 + rank * 128, g = jb / kGroup8 + (lane & 1);
      for (int kb = t.kb0; kb < t.kb1; ++kb, ++n) {
        const int s = n % SC;
        if (n >= (unsigned)SC) warp_wait(&c_empty[s], (n / SC - 1) & 1, a.err);
        if (lane == 0) {
          mbar_expect_tx(&c_full[s], kRaw);
          tma_box<false>(smem0 + P::kCodesAt + s * kRaw, &a.b, jb, kb * kDepth, 0,
                         smem_u32(&c_full[s]));
        }
        const unsigned to = smem0 + P::kRangesAt + s * kRanges + lane * 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const long long r = (long long)kb * kDepth + 16 * i + (lane >> 1);
          const bool in = g < a.groups && r < a.rows;
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(to + 128 * i),
                       "l"(a.ranges + (in ? r * a.groups + g : 0)), "r"(in ? 4 : 0)
                       : "memory");
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];\n" ::"r"(
                         smem_u32(&c_full[s]))
                     : "memory");
      }
    }
    asm volatile("cp.async.wait_all;\n" ::: "memory");
    for (unsigned i = n > (unsigned)SC ? n - SC : 0; i < n; ++i)
      warp_wait(&c_full[i % SC], (i / SC) & 1, a.err);
  } else if (PACKED && warp >= 4 && warp < 4 + P::kWriters) {
    // Two teams of four warps take the stages in turn, so that one team's loads and
    // barriers run beside the other's arithmetic.  A thread has 16 columns of four of
    // a stage's 64 rows.
    const int team = (warp - 4) >> 2, id = threadIdx.x & 127, row = id >> 3, seg = id & 7;
    const int odd = seg >> 2, u = (seg & 3) * 2;
    unsigned n = 0;
    for (int item = first; work_of(a, item, &t); item += step) {
      for (int kb = t.kb0; kb < t.kb1; ++kb, ++n) {
        if ((int)(n & 1) != team) continue;
        const int s = n % S, c = n % SC;
        warp_wait(&c_full[c], (n / SC) & 1, a.err);
        const char* const codes = smem + P::kCodesAt + c * kRaw + seg * 16;
        const unsigned* const ranges =
            reinterpret_cast<const unsigned*>(smem + P::kRangesAt + c * kRanges) + odd;
        uint4 q[4];
        unsigned bits[4];
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          q[h] = *reinterpret_cast<const uint4*>(codes + (row + 16 * h) * 128);
          bits[h] = ranges[(row + 16 * h) * 2];
        }
        if (n >= (unsigned)S) warp_wait(&empty[s], (n / S - 1) & 1, a.err);
        // Only now: the codes of stage n + 5 then follow this stage's phase, so that the
        // other team, whose that stage is, cannot take an older phase for it.
        __syncwarp();
        if (lane == 0) arrive_leader<false>(&c_empty[c]);
        char* const stage = smem + P::kBAt + s * kHalf + odd * kBox;
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const int r = row + 16 * h;
          uint4 o[2];
          operands16<T>(q[h], bits[h], o);
          // blocks of 64 columns; 128-byte rows whose 16-byte units are xor-ed with the
          // row; the two halves of a row's columns take turns at the banks
          char* const to = stage + r * 128;
          *reinterpret_cast<uint4*>(to + (((u + odd) ^ (r & 7)) << 4)) = odd ? o[1] : o[0];
          *reinterpret_cast<uint4*>(to + (((u + 1 - odd) ^ (r & 7)) << 4)) = odd ? o[0] : o[1];
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) arrive_written(&full[s]);
      }
    }
  } else if (warp >= 4 + P::kWriters) {
    const int w = warp & 3, h = (warp - 4 - P::kWriters) >> 2;
    constexpr int kCols = kTile * 4 / P::kEpi;  // columns of a warp
    char* const turn = smem + P::kTurnAt + (warp - 4 - P::kWriters) * kTurn;
    unsigned tile = 0;
    for (int item = first; work_of(a, item, &t); item += step, ++tile) {
      const int buf = tile & 1;
      if (lane == 0) wait_pair(&tm_full[buf], (tile / 2) & 1, a.err);
      __syncwarp();
      asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
      const int i = t.i0 + rank * 128 + 32 * w;
#pragma unroll 1
      for (int c = h * kCols; c < (h + 1) * kCols; c += 64) {
        float v[64];
#pragma unroll
        for (int q = 0; q < 2; ++q)
          tmem_load32(tmem + buf * 256 + c + 32 * q + ((unsigned)(32 * w) << 16),
                      *reinterpret_cast<float(*)[32]>(v + 32 * q));
        if (c + 64 == (h + 1) * kCols) {
          __syncwarp();
          asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
          if (lane == 0) arrive_leader<true>(&tm_empty[buf]);
        }
        if (PACKED && a.parts > 1) {
          // [item][block][columns / 4][128 rows] of four columns each
          float4* const to = reinterpret_cast<float4*>(
              a.part + ((long long)t.item * 2 + rank) * kPartFloats) + c / 4 * 128 + 32 * w + lane;
#pragma unroll
          for (int q = 0; q < 16; ++q)
            to[q * 128] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
        } else if (i < a.m && t.j0 + c < a.n) {
          put_result<T>(a, i, t.j0 + c, v, turn);
        }
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;\n" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
  __syncthreads();
  cluster_sync();  // neither block's memory is in use any more
  // The first block has issued its last commit, which arrives at the second
  // block's barriers too: that block stays until it has.
  if (rank == 1 && threadIdx.x == 32) stage_wait(&drain, 0, a.err);
  if (warp == 2) {
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;\n" ::"r"(tmem));
  }
}

// The parts of a tile added in order: a thread has 16 columns of a row.
template <typename T>
__global__ void __launch_bounds__(128) join_parts_kernel(const __grid_constant__ ProductArgs a) {
  const int tiles = a.tiles_m * a.tiles_n;
  const int tile = blockIdx.x >> 5, rank = (blockIdx.x >> 4) & 1, c = (blockIdx.x & 15) * 16;
  Work t;
  work_of(a, tile, &t);
  const int i = t.i0 + rank * 128 + threadIdx.x, j = t.j0 + c;
  if (i >= a.m || j >= a.n) return;
  float v[16] = {};
  for (int p = 0; p < a.parts; ++p) {
    const float4* const from = reinterpret_cast<const float4*>(
        a.part + ((long long)(p * tiles + tile) * 2 + rank) * kPartFloats) + c / 4 * 128 + threadIdx.x;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float4 f = from[q * 128];
      v[4 * q] += f.x;
      v[4 * q + 1] += f.y;
      v[4 * q + 2] += f.z;
      v[4 * q + 3] += f.w;
    }
  }
  T* const out = reinterpret_cast<T*>(a.out) + (long long)i * a.n + j;
  if (a.tma_out && j + 16 <= a.n) {
#pragma unroll
    for (int q = 0; q < 2; ++q)
      reinterpret_cast<uint4*>(out)[q] =
          make_uint4(pair_bits<T>(v[8 * q], v[8 * q + 1]), pair_bits<T>(v[8 * q + 2], v[8 * q + 3]),
                     pair_bits<T>(v[8 * q + 4], v[8 * q + 5]), pair_bits<T>(v[8 * q + 6], v[8 * q + 7]));
  } else {
#pragma unroll
    for (int q = 0; q < 16; ++q)
      if (j + q < a.n) out[q] = St<T>::v(v[q]);
  }
}

// Rows at a pitch of whole 16 bytes, for TMA.
template <typename T>
__global__ void __launch_bounds__(256) pitch_kernel(const T* x, long long x_row, T* y, int pitch,
                                                    long long rows, int width) {
  const long long n = rows * pitch;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
    const long long r = i / pitch;
    const int c = (int)(i - r * pitch);
    T v = T();
    if (c < width) v = ldro(x + r * x_row + c);
    y[i] = v;
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

// A tile's sum over 2^27 rows takes under a second, and a wait for it two at most.
constexpr long long kMaxRows = 1ll << 27;
constexpr int kMaxSide = (1 << 22) - 64;  // 65535 tiles of 64

static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

// [rows][pitch bytes] of 16-bit values, boxes of 64 x `high` in the 128-byte
// swizzle; or of bytes, boxes of 128 x 64 as they lie.  Outside arrives as zeros.
static bool box_map(CUtensorMap* map, const void* p, long long rows, long long cols,
                    long long pitch, bool bytes, int high) {
  EncodeTiledFn fn = encode_tiled();
  if (!fn) return false;
  const cuuint64_t dim[3] = {(cuuint64_t)cols, (cuuint64_t)rows, 1};
  const cuuint64_t stride[2] = {(cuuint64_t)pitch, (cuuint64_t)(pitch * rows)};
  const cuuint32_t box[3] = {bytes ? 128u : 64u, (cuuint32_t)high, 1}, one[3] = {1, 1, 1};
  return fn(map, bytes ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 3,
            const_cast<void*>(p), dim, stride, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
            bytes ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static int tiles_of(long long n) { return (int)((n + kTile - 1) / kTile); }

// Parts of the sum's axis: the number whose waves take the least time, at 0.4 us a
// stage of a pair, 3 us a tile's end, and the parts' trip through memory.
static int parts_of(int tiles, int kb, int pairs) {
  int best = 1;
  double least = 0;
  for (int p = 1; p <= 32 && p <= kb; ++p) {
    const double waves = (double)((tiles * (long long)p + pairs - 1) / pairs);
    double us = waves * (0.4 * ((kb + p - 1) / p) + 3.0);
    if (p > 1) us += 4.0 + tiles * (double)p * 2 * kPartFloats * 4 * 2 / 4e6;
    if (p == 1 || us < least) {
      least = us;
      best = p;
    }
  }
  return best;
}

// Pairs of blocks that run at once.
static int resident_pairs(int device) {
  constexpr int MAXD = 64;
  static std::atomic<int> known[MAXD];
  if (device < 0 && cudaGetDevice(&device) != cudaSuccess) device = MAXD;
  if (device < MAXD && known[device].load() > 0) return known[device].load();
  int n = 0;
  const ScopedDevice scope(device < MAXD ? device : -1);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(sm_count(device) / 2 * 2));
  cfg.blockDim = dim3(Product<true>::kThreads);
  cfg.dynamicSmemBytes = Product<true>::kSmem;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = 2;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (cudaFuncSetAttribute(product_kernel<bf16_t, true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           Product<true>::kSmem) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, product_kernel<bf16_t, true>, &cfg) != cudaSuccess || n < 1) {
    cudaGetLastError();
    n = std::max(1, sm_count(device) / 2);
  }
  if (device < MAXD) known[device].store(n);
  return n;
}

// What one call of the weight gradient takes from its workspace.
struct WgradPlan {
  int pitch;                    // of the copy of dy, in values (0: no copy)
  int parts, pairs;
  size_t copy, part, bytes;     // offsets and size
};
static WgradPlan wgrad_plan(long long rows, int inputs, int outputs, int dtype, int device) {
  WgradPlan p = {};
  p.bytes = up256(norm_ws_bytes(rows, outputs, device));
  if (dtype == FA_F32) return p;
  p.copy = p.bytes;
  p.pitch = (outputs + 7) / 8 * 8;
  p.bytes += up256((size_t)rows * p.pitch * 2);
  const int tiles = tiles_of(inputs) * tiles_of(outputs);
  p.pairs = resident_pairs(device);
  p.parts = parts_of(tiles, (int)((rows + kDepth - 1) / kDepth), p.pairs);
  p.part = p.bytes;
  if (p.parts > 1) p.bytes += (size_t)tiles * p.parts * 2 * kPartFloats * sizeof(float);
  return p;
}

size_t wgrad8_ws_bytes(long long rows, int inputs, int outputs, int dtype, int device) {
  return wgrad_plan(rows, inputs, outputs, dtype, device).bytes;
}

template <typename T, bool PACKED>
static int product_run(const ProductArgs& a, int pairs, cudaStream_t st) {
  constexpr int smem = Product<PACKED>::kSmem;
  FAB_TRY(cudaFuncSetAttribute(product_kernel<T, PACKED>,
                               cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  const int items = a.tiles_m * a.tiles_n * a.parts;
  product_kernel<T, PACKED><<<2 * std::min(items, pairs), Product<PACKED>::kThreads, smem, st>>>(a);
  FAB_LAUNCH_CHECK();
  return FA_OK;
}

template <typename T>
static int wgrad_run(const void* dy, long long dy_row, const void* codes, const void* ranges,
                     long long rows, int inputs, int outputs, void* dw, char* ws,
                     const WgradPlan& plan, int device, cudaStream_t st) {
  // TMA reads rows at a pitch of whole 16 bytes that do not overlap
  if (reinterpret_cast<size_t>(dy) % 16 || (rows > 1 && (dy_row % 8 || dy_row < outputs))) {
    T* const copy = reinterpret_cast<T*>(ws + plan.copy);
    const long long blocks = std::min((rows * plan.pitch + 255) / 256, (long long)sm_count(device) * 16);
    pitch_kernel<T><<<(unsigned)blocks, 256, 0, st>>>(static_cast<const T*>(dy), dy_row, copy,
                                                      plan.pitch, rows, outputs);
    FAB_LAUNCH_CHECK();
    dy = copy;
    dy_row = plan.pitch;
  }
  if (rows == 1) dy_row = plan.pitch;
  ProductArgs a = {};
  const long long groups = groups8(inputs);
  if (!box_map(&a.a, dy, rows, outputs, dy_row * 2, false, 64) ||
      !box_map(&a.b, codes, rows, groups * kGroup8, groups * kGroup8, true, kDepth))
    return FA_E_INTERNAL;
  a.tma_out = inputs % 8 == 0 && reinterpret_cast<size_t>(dw) % 16 == 0;
  if (a.tma_out && !box_map(&a.d, dw, outputs, inputs, inputs * 2ll, false, 32)) return FA_E_INTERNAL;
  a.m = outputs;
  a.n = inputs;
  a.kb = (int)((rows + kDepth - 1) / kDepth);
  a.a_mn = a.b_mn = 1;
  a.tiles_m = tiles_of(outputs);
  a.tiles_n = tiles_of(inputs);
  a.parts = plan.parts;
  a.ranges = static_cast<const unsigned*>(ranges);
  a.rows = rows;
  a.groups = (int)groups;
  a.out = dw;
  a.part = reinterpret_cast<float*>(ws + plan.part);
  a.err = wait_error_word();
  if (const int rc = product_run<T, true>(a, plan.pairs, st)) return rc;
  if (a.parts > 1) {
    join_parts_kernel<T><<<(unsigned)(a.tiles_m * a.tiles_n * 32), 128, 0, st>>>(a);
    FAB_LAUNCH_CHECK();
  }
  return FA_OK;
}

int wgrad8_impl(const void* dy, long long dy_row, const void* codes, const void* ranges, int dtype,
                long long rows, int inputs, int outputs, void* dw, void* db, void* ws,
                size_t ws_bytes, int device, cudaStream_t st) {
  if (!train_dtype(dtype)) return FA_E_DTYPE;
  if (rows <= 0 || inputs <= 0 || outputs <= 0 || rows > kMaxRows || inputs > kMaxSide ||
      outputs > kMaxSide)
    return FA_E_SHAPE;
  const int item = item_size(dtype);
  if (!dy || (dw && (!codes || !ranges)) || reinterpret_cast<size_t>(dy) % item ||
      reinterpret_cast<size_t>(dw) % item || reinterpret_cast<size_t>(db) % item ||
      reinterpret_cast<size_t>(codes) % 16 || reinterpret_cast<size_t>(ranges) % 8 || !ws ||
      reinterpret_cast<size_t>(ws) % 256)
    return FA_E_ARG;
  const WgradPlan plan = wgrad_plan(rows, inputs, outputs, dtype, device);
  if (ws_bytes < plan.bytes) return FA_E_ARG;
  FAB_DEVICE_SCOPE(device);
  if (db)
    if (const int rc = bias_grad_impl(dy, dy_row, db, dtype, rows, outputs, ws, ws_bytes, device, st))
      return rc;
  if (!dw) return FA_OK;
  if (dtype == FA_F16)
    return wgrad_run<f16_t>(dy, dy_row, codes, ranges, rows, inputs, outputs, dw,
                            static_cast<char*>(ws), plan, device, st);
  if (dtype == FA_BF16)
    return wgrad_run<bf16_t>(dy, dy_row, codes, ranges, rows, inputs, outputs, dw,
                             static_cast<char*>(ws), plan, device, st);
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
  wgrad_lanes_kernel<float><<<grid, 256, 0, st>>>(a);
  FAB_LAUNCH_CHECK();
  return FA_OK;
}

}  // namespace fab
