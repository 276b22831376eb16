// A product that keeps its operand packed (keep8.cuh):
//   y = x W^T + b,   dx = dy W,
//   dW[m, k] = sum over rows t of dy[t, m] x^[t, k],   db[m] = sum over t of dy[t, m],
// where x^ are the values that the codes stand for.  All sums are float32 and rounded
// once, also where an axis is cut into parts.
//
// dW in 16-bit types: tensor-core products of 256 inputs x 256 outputs over pairs of blocks
// (tcgen05, cta_group::2), persistent.  dy arrives by TMA as it lies (its rows are the
// sum's axis: MN-major) and is the products' second operand in shared memory.  The
// codes arrive by TMA as bytes; eight warps turn them, transposed on the way out of
// shared memory, into the first operand in TENSOR MEMORY (a lane an input, two rows t a
// word), while the tensor cores work on the stages before.  So the unpacked values
// never pass through shared memory, whose bytes bound these products: with them there
// a stage of 64 rows took 1000 cycles against 670 with both operands from TMA.  Every
// value q s + lo is rounded once, as unpacking rounds it.  Where the tiles are fewer
// than the pairs of blocks, the rows are cut into parts whose float32 sums are joined
// in order.  y and dx: the same tiles, both operands by TMA.  float32: on the ordinary
// lanes.
//
// Measured on one B200 at 16320 rows, 1024 inputs, 4096 outputs, bfloat16: y 109 us, dx
// 98 us, dW 115 us (1.2 to 1.4 PFLOP/s; torch's products 99, 94 and 90 us), packing 11
// us, db 26 us.  y and dx are bound by operand bytes out of the second-level cache (11.3
// TB/s; the tensor pipe 72 % active at 8192 x 4096 x 4096, 189 us), dW by the products
// themselves (685 cycles for 256 x 256 x 64) and by 64 tiles for 74 pairs of blocks.
#include <algorithm>
#include <atomic>

#include "keep8.cuh"
#include "tensor.cuh"

namespace fab {

int bias_grad_impl(const void* g, long long g_row, void* db, int dtype, long long rows, int width,
                   void* ws, size_t ws_bytes, int device, cudaStream_t st);
size_t norm_ws_bytes(long long rows, int width, int device);
int pack8_impl(const void* x, long long x_row, void* codes, void* ranges, int dtype,
               long long rows, int width, int device, cudaStream_t st);

// ---------------------------------------------------------------------------
// float32
// ---------------------------------------------------------------------------

// All three products in float32, on the ordinary lanes (two products an instruction):
// the tensor cores would round the operands.  D[m][n] = sum over k of A B, 128 x 128 a
// block, 8 x 8 a thread, 16 of k a stage; the next stage is on its way while this one's
// products run.  Few tiles: k is cut into parts, whose sums are joined in order.  After
// every 32768 terms the sum goes to its place in the result, so that a long one's roundings
// do not add up.
// Bound by the products: 16320 rows, 1024 x 1024, y 0.68, dx 0.63, dW 0.84 ms, 41 to 54
// TFLOP/s.
constexpr int kLaneTile = 128, kLaneDepth = 16;
constexpr long long kLongest = 32768;  // terms of a sum

struct LaneArgs {
  const float *a, *b;           // or codes
  long long a_row, b_row;
  const unsigned char* codes;
  const float2* ranges;
  long long k, per_part;        // whole stages a part
  int m, n, groups, parts;
  const float* bias;            // [n] or null
  float* d;                     // [parts][m][n]
  int a_vec, b_vec;             // rows are whole aligned vectors of four
};

// How an operand lies: its tile's axis as rows with k along them, k as rows, or packed
// rows k.
enum LaneOperand { ALONG_K, ROWS_K, CODES_K };

// 4 values of a row from column c, those past the n-th zero.
__device__ __forceinline__ float4 four(const float* p, long long c, long long n, int vec) {
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (vec && c + 4 <= n) return __ldg(reinterpret_cast<const float4*>(p + c));
  if (c < n) v.x = __ldg(p + c);
  if (c + 1 < n) v.y = __ldg(p + c + 1);
  if (c + 2 < n) v.z = __ldg(p + c + 2);
  if (c + 3 < n) v.w = __ldg(p + c + 3);
  return v;
}

// LONG: some part is longer than 32768.
template <LaneOperand A, LaneOperand B, bool LONG>
__global__ void __launch_bounds__(256, 2) lanes_kernel(const LaneArgs a) {
  constexpr int P = kLaneTile + 4;  // pitch: transposed stores meet two at a bank, not eight
  __shared__ __align__(16) float sa[2][kLaneDepth][P], sb[2][kLaneDepth][P];
  const int m0 = blockIdx.x * kLaneTile, n0 = blockIdx.y * kLaneTile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const long long k0 = blockIdx.z * a.per_part, k1 = min(a.k, k0 + a.per_part);
  // this thread's share of a stage: two vectors of four, or 8 codes
  const int rk = threadIdx.x >> 5, ck = (threadIdx.x & 31) * 4;   // k rows rk, rk + 8
  const int rt = threadIdx.x >> 2, ct = (threadIdx.x & 3) * 4;    // tile rows rt, rt + 64
  const int rc = threadIdx.x >> 4, uc = threadIdx.x & 15;         // codes: k row, unit
  float4 na[2], nb[2];
  uint2 nq;
  float2 nr;
  const auto share = [&](LaneOperand how, const float* p, long long row, int i0, int size, int vec,
                         long long k, float4 (&to)[2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      to[h] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (how == ROWS_K) {
        if (k + rk + 8 * h < k1) to[h] = four(p + (k + rk + 8 * h) * row, i0 + ck, size, vec);
      } else if (i0 + rt + 64 * h < size) {
        to[h] = four(p + (i0 + rt + 64 * h) * row, k + ct, k1, vec);
      }
    }
  };
  const auto fetch = [&](long long k) {
    share(A, a.a, a.a_row, m0, a.m, a.a_vec, k, na);
    if constexpr (B != CODES_K) {
      share(B, a.b, a.b_row, n0, a.n, a.b_vec, k, nb);
    } else {
      const int g = n0 / kGroup8 + (uc >> 3);
      nq = make_uint2(0u, 0u);
      nr = make_float2(0.f, 0.f);
      if (k + rc < k1 && g < a.groups) {
        const long long at = (k + rc) * a.groups + g;
        nq = __ldg(reinterpret_cast<const uint2*>(a.codes) + at * 8 + (uc & 7));
        nr = __ldg(a.ranges + at);
      }
    }
  };
  const auto lay = [&](LaneOperand how, float (*to)[P], const float4 (&v)[2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (how == ROWS_K) {
        *reinterpret_cast<float4*>(&to[rk + 8 * h][ck]) = v[h];
      } else {
        to[ct][rt + 64 * h] = v[h].x;
        to[ct + 1][rt + 64 * h] = v[h].y;
        to[ct + 2][rt + 64 * h] = v[h].z;
        to[ct + 3][rt + 64 * h] = v[h].w;
      }
    }
  };
  const auto put = [&](int half) {
    lay(A, sa[half], na);
    if constexpr (B != CODES_K)
      lay(B, sb[half], nb);
    else
      put8<float>(&sb[half][rc][uc * 8], narrow8(decode8<float>(nq, range_of(nr, 0.f)), 0.f));
  };
  float2 acc[8][4];
  fetch(k0);
  put(0);
  int half = 0;
  long long k = k0;
  do {
    const long long c0 = k, c1 = LONG ? min(k1, c0 + kLongest) : k1;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = both(0.f);
    for (; k < c1; k += kLaneDepth, half ^= 1) {
      __syncthreads();
      fetch(k + kLaneDepth);
#pragma unroll
      for (int r = 0; r < kLaneDepth; ++r) {
        // rows ty * 4 + 0..3 and 64 on, columns tx * 4 + 0..3 and 64 on
        const float4 p0 = *reinterpret_cast<const float4*>(&sa[half][r][ty * 4]),
                     p1 = *reinterpret_cast<const float4*>(&sa[half][r][64 + ty * 4]),
                     q0 = *reinterpret_cast<const float4*>(&sb[half][r][tx * 4]),
                     q1 = *reinterpret_cast<const float4*>(&sb[half][r][64 + tx * 4]);
        const float p[8] = {p0.x, p0.y, p0.z, p0.w, p1.x, p1.y, p1.z, p1.w};
        const float2 q[4] = {{q0.x, q0.y}, {q0.z, q0.w}, {q1.x, q1.y}, {q1.z, q1.w}};
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] = __ffma2_rn(both(p[i]), q[j], acc[i][j]);
      }
      if (k + kLaneDepth < k1) put(half ^ 1);
    }
    // what is there is the sum before
    float* const out = a.d + (long long)blockIdx.z * a.m * a.n;
    const float* const bias = a.parts == 1 && c1 == k1 ? a.bias : nullptr;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int m = m0 + (i >> 2) * 64 + ty * 4 + (i & 3);
      if (m >= a.m) continue;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int n = n0 + (j >> 2) * 64 + tx * 4 + (j & 3);
        float v = j & 1 ? acc[i][j / 2].y : acc[i][j / 2].x;
        if (n < a.n) {
          if (LONG && c0 > k0) v += out[(long long)m * a.n + n];
          out[(long long)m * a.n + n] = bias ? v + __ldg(bias + n) : v;
        }
      }
    }
  } while (LONG && k < k1);
}
__global__ void __launch_bounds__(256) join_lanes_kernel(const float* part, float* d, int parts,
                                                         long long size, const float* bias, int n) {
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < size; i += gridDim.x * 256ll) {
    float t = 0.f;
    for (int p = 0; p < parts; ++p) t += part[p * size + i];
    d[i] = bias ? t + __ldg(bias + i % n) : t;
  }
}

// ---------------------------------------------------------------------------
// 16-bit products on the tensor cores
// ---------------------------------------------------------------------------

constexpr int kTile = 256;      // inputs and outputs of a pair's tile
constexpr int kDepth = 64;      // rows t a stage
constexpr int kHalf = 2 * kBox; // bytes of one block's 128 outputs of a stage
constexpr int kRaw = kDepth * 128;  // bytes of a stage's codes
constexpr int kRanges = kDepth * 8; // and of their ranges, two groups a row
// Stages of operands and of codes, which run ahead of them.  Even numbers: the two
// teams of writers take turns, and each then sees every phase of its stages.
constexpr int kStages = 8, kCodeStages = 8;
constexpr int kWriters = 8;     // warps that unpack, and write the sums out
constexpr int kWgThreads = 128 + 32 * kWriters;
constexpr int kCodesAt = kStages * kHalf;           // offsets in shared memory
constexpr int kRangesAt = kCodesAt + kCodeStages * kRaw;
constexpr int kWgSmem = kRangesAt + kCodeStages * kRanges + 1024;
constexpr int kOperandAt = 256; // columns of tensor memory: the sums', then 32 a stage
constexpr int kPartFloats = 128 * 256;  // of one block's part of a tile
// The tensor cores add to a sum with truncation, up to 2^-24 of it for each 16 terms and
// always towards zero.  A sum of more than 32768 terms is therefore taken in chunks of
// so many, each at most 6e-5 of it short on average (a quarter of float16's half step),
// and the chunks are added with rounding, in a slab of float32 that a pair of blocks keeps
// for all of its tiles (or a part its own): the workspace does not grow with the sum.
constexpr int kChunk = 512;     // stages

// dW[n][m] = sum over t of x^[t][m] dy[t][n].
struct ProductArgs {
  CUtensorMap codes, dy;
  int m, n, kb;                 // inputs, outputs, stages of the whole sum
  int tiles_m, tiles_n, parts;
  const unsigned* ranges;
  long long rows;
  int groups;
  void* out;
  float* part;                  // a slab of 256 x 256 a part, or (one part) a pair of blocks
  unsigned* err;
};

struct Work {
  int i0, j0, kb0, kb1, item;
};
// ROWS of a tile.  Items are numbered part by part; inside a part eight rows of tiles are walked
// column by column, so the tiles at work share operand panels in the L2 cache.
template <int ROWS = kTile, typename Args>
__device__ __forceinline__ bool work_of(const Args& a, int item, Work* w) {
  const int tiles = a.tiles_m * a.tiles_n;
  if (item >= tiles * a.parts) return false;
  const int part = item / tiles, tile = item - part * tiles;
  const int band = tile / (8 * a.tiles_n), in = tile - band * 8 * a.tiles_n;
  const int high = min(8, a.tiles_m - band * 8);
  w->i0 = (band * 8 + in % high) * ROWS;
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
// 16 such polls, and once in a millisecond.
// PAIR: threads of the pair's other block arrive at the barrier, too, so that what is
// acquired is the whole cluster's.
template <bool PAIR>
__device__ __forceinline__ bool mbar_sleep(unsigned a, unsigned parity) {
  unsigned done;
  if constexpr (PAIR)
    asm volatile(
        "{\n .reg .pred p;\n"
        " mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n"
        " selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(done)
        : "r"(a), "r"(parity), "r"(2000000u)
        : "memory");
  else
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
      "{\n .reg .pred p;\n"
      " mbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return done != 0;
}
template <bool PAIR>
static __device__ __noinline__ void stage_wait_slow(unsigned a, unsigned parity, unsigned* err,
                                                    unsigned long long limit_ns) {
  const unsigned long long t0 = globaltimer_ns();
  unsigned long long next = 1000000ull;
  for (unsigned i = 1;; ++i) {
    if (mbar_sleep<PAIR>(a, parity)) return;
    const unsigned long long t = globaltimer_ns() - t0;
    if ((i & 15u) != 0u || t < next) continue;
    next = t + 1000000ull;
    if (t > limit_ns || (err && *reinterpret_cast<volatile unsigned*>(err) != 0u)) {
      if (err) {
        *reinterpret_cast<volatile unsigned*>(err) = (unsigned)FA_E_TIMEOUT;
        __threadfence_system();
      }
      return;
    }
  }
}
template <bool PAIR = false>
__device__ __forceinline__ void stage_wait(unsigned long long* bar, unsigned parity,
                                           unsigned* err) {
  const unsigned a = smem_u32(bar);
  if (!mbar_sleep<PAIR>(a, parity)) stage_wait_slow<PAIR>(a, parity, err, kWaitLimitNs);
}

// A warp has written its share of a stage into its own block's tensor memory, and the
// first block's thread that waits for it issues a product that reads both blocks'.  What
// orders the two is tcgen05's own chain: the stores' wait, the fence before the arrival,
// the fence behind the wait; between them the arrival and the wait have to be of the
// cluster's scope, as the blocks are two, but nothing else is handed over, so the arrival
// releases nothing (dW of 16320 rows, 1024 x 4096 bfloat16, 115 us; 226 with a release,
// which waits for all of the warp's memory operations).
__device__ __forceinline__ void arrive_written(unsigned long long* bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(
                   in_leader(smem_u32(bar)))
               : "memory");
}

// One lane polls, the others wait at the warp's barrier.
__device__ __forceinline__ void warp_wait(unsigned long long* bar, unsigned parity, unsigned* err) {
  if ((threadIdx.x & 31) == 0) stage_wait(bar, parity, err);
  __syncwarp();
}

// Steps and lowest values of four rows t, two to a word.
struct Range4 {
  unsigned s[2], lo[2];
};
template <typename T>
__device__ __forceinline__ Range4 range4(uint4 b) {
  Range4 r;
  r.lo[0] = __byte_perm(b.x, b.y, 0x5410);
  r.lo[1] = __byte_perm(b.z, b.w, 0x5410);
  r.s[0] = __byte_perm(b.x, b.y, 0x7632);
  r.s[1] = __byte_perm(b.z, b.w, 0x7632);
  if constexpr (std::is_same<T, f16_t>::value) {  // from bfloat16
#pragma unroll
    for (int i = 0; i < 2; ++i) r.s[i] = narrow2(widen2(r.s[i], bf16_t()), f16_t());
  }
  return r;
}
// Whether float16 holds every step: not of spreads below 2^-16, of rows behind the last
// (zero), or of groups that are not finite (NaN).
__device__ __forceinline__ bool held_in_half(uint4 b) {
  const float s[4] = {range_of(b.x, f16_t()).s, range_of(b.y, f16_t()).s,
                      range_of(b.z, f16_t()).s, range_of(b.w, f16_t()).s};
  bool held = true;
#pragma unroll
  for (int i = 0; i < 4; ++i) held = held && s[i] >= 5.9604644775390625e-8f;  // 2^-24
  return held;
}
// Codes k and k + 1 of a word to two operand values.  The low bytes of 2^23 + q and of
// 1024 + q are q, and q has 8 bits: bfloat16 holds it exactly, as the high half of a
// float32.
__device__ __forceinline__ unsigned operand2(unsigned w, int k, unsigned s, unsigned lo, bf16_t) {
  const float2 q = __fadd2_rn(
      make_float2(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 | k)),
                  __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 | (k + 1)))),
      both(-kMagic8));
  unsigned o = __byte_perm(__float_as_uint(q.x), __float_as_uint(q.y), 0x7632);
  asm("fma.rn.bf16x2 %0, %0, %1, %2;" : "+r"(o) : "r"(s), "r"(lo));
  return o;
}
__device__ __forceinline__ unsigned operand2(unsigned w, int k, unsigned s, unsigned lo, f16_t) {
  unsigned o = __byte_perm(w, 0x64646464u, k ? 0x4342 : 0x4140);
  asm("add.rn.f16x2 %0, %0, %1;" : "+r"(o) : "r"(0xe400e400u));  // -1024
  asm("fma.rn.f16x2 %0, %0, %1, %2;" : "+r"(o) : "r"(s), "r"(lo));
  return o;
}
// The same from the ranges themselves, where float16 does not hold a step.
__device__ __forceinline__ unsigned operand2_wide(unsigned w, int k, unsigned b0, unsigned b1) {
  const Range8 r0 = range_of(b0, f16_t()), r1 = range_of(b1, f16_t());
  const float q0 = (float)((w >> (8 * k)) & 255u), q1 = (float)((w >> (8 * k + 8)) & 255u);
  return narrow2(make_float2(fmaf(q0, r0.s, r0.lo), fmaf(q1, r1.s, r1.lo)), f16_t());
}

// 16 x 16 bytes transposed, twice: a lane gets, for rows t = 4 (lane % 4) ... + 3 of
// either, the codes of inputs lane / 4 (o[0], o[2]) and lane / 4 + 8 (o[1], o[3]).
__device__ __forceinline__ void codes16x2(unsigned addr, unsigned (&o)[4]) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0, %1, %2, %3}, [%4];\n"
               : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3])
               : "r"(addr)
               : "memory");
}
// 16 lanes x 32 columns of tensor memory, in the same arrangement.
__device__ __forceinline__ void tmem_store16(unsigned addr, const unsigned (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15, %16};\n" ::"r"(addr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
// D (256 x 256 over the pair) += A (tensor memory) B (shared memory)
__device__ __forceinline__ void mma_from_tmem(unsigned d, unsigned a, unsigned long long b,
                                              unsigned idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((unsigned)add)
      : "memory");
}

// CHUNKS: some part is longer than a chunk (the writers' sums then end a part's stages
// more than once, which costs 5 % where it is not needed).
template <typename T, bool CHUNKS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kWgThreads, 1)
    wgrad_kernel(const __grid_constant__ ProductArgs a) {
  constexpr int S = kStages, SC = kCodeStages;
  extern __shared__ char smem_raw[];
  const unsigned smem0 = (smem_u32(smem_raw) + 1023u) & ~1023u;
  char* const smem = smem_raw + (smem0 - smem_u32(smem_raw));
  __shared__ unsigned long long full[S], empty[S], c_full[SC], c_empty[SC], tm_full, tm_empty,
      drain;
  __shared__ unsigned tmem_base;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = blockIdx.x & 1;
  const int first = blockIdx.x >> 1, step = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&full[i], 1 + kWriters);  // the copies' bytes, a team of writers in either block
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < SC; ++i) {
      mbar_init(&c_full[i], 1 + 32);      // the codes' copy, and a warp's copies of ranges
      mbar_init(&c_empty[i], kWriters / 2);
    }
    mbar_init(&tm_full, 1);
    mbar_init(&tm_empty, 2 * kWriters);
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
        const int jb = t.j0 + rank * 128;
        for (int kb = t.kb0; kb < t.kb1; ++kb, ++n) {
          const int s = n % S;
          if (n >= (unsigned)S) stage_wait(&empty[s], (n / S - 1) & 1, a.err);
          // both blocks' copies count on the first block's barrier
          const unsigned bar = in_leader(smem_u32(&full[s]));
          if (rank == 0) mbar_expect_tx(&full[s], 2 * kHalf);
#pragma unroll
          for (int i = 0; i < 2; ++i)
            tma_box<true>(smem0 + s * kHalf + i * kBox, &a.dy, jb + 64 * i, kb * kDepth, 0, bar);
        }
      }
      // copies still in flight land before the block ends
      for (unsigned i = n > (unsigned)S ? n - S : 0; rank == 0 && i < n; ++i)
        stage_wait(&full[i % S], (i / S) & 1, a.err);
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      // float32 sums; both operands float16 or both bfloat16; 256 x 256 over the pair;
      // the second operand with t as its rows
      const unsigned kind = std::is_same<T, bf16_t>::value ? (1u << 7) | (1u << 10) : 0u;
      const unsigned idesc = (1u << 4) | kind | (1u << 16) | ((unsigned)(kTile / 8) << 17) |
                             ((unsigned)(kTile / 16) << 24);
      unsigned n = 0, tile = 0;
      for (int item = first; work_of(a, item, &t); item += step)
        for (int c0 = t.kb0, c1; c0 < t.kb1; c0 = c1, ++tile) {
          c1 = CHUNKS ? min(t.kb1, c0 + kChunk) : t.kb1;
          if (tile >= 1) stage_wait<true>(&tm_empty, (tile - 1) & 1, a.err);
          asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
          bool ready = false;
          for (int kb = c0; kb < c1; ++kb, ++n) {
            const int s = n % S;
            if (!ready) stage_wait<true>(&full[s], (n / S) & 1, a.err);
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
            const unsigned p = tmem + kOperandAt + s * 32;
            const unsigned long long q = operand(smem0 + s * kHalf);
#pragma unroll
            for (int k = 0; k < kDepth / 16; ++k) {
              mma_from_tmem(tmem, p + 8 * k, q + k * (2048u >> 4), idesc, kb > c0 || k > 0);
              // the next stage is asked for while this one's products run: few are queued,
              // and a poll takes longer than the last of them
              if (k == 1) ready = kb + 1 < c1 && mbar_peek(&full[(n + 1) % S], ((n + 1) / S) & 1);
            }
            mma_commit<true>(&empty[s]);
          }
          mma_commit<true>(&tm_full);
        }
      // products still in flight end before tensor memory is given back
      mma_commit<true>(&drain);
      stage_wait(&drain, 0, a.err);
    }
  } else if (warp == 2) {
    if (lane == 0) {  // codes
      unsigned n = 0;
      for (int item = first; work_of(a, item, &t); item += step)
        for (int kb = t.kb0; kb < t.kb1; ++kb, ++n) {
          const int s = n % SC;
          if (n >= (unsigned)SC) stage_wait(&c_empty[s], (n / SC - 1) & 1, a.err);
          mbar_expect_tx(&c_full[s], kRaw);
          tma_box<false>(smem0 + kCodesAt + s * kRaw, &a.codes, t.i0 + rank * 128, kb * kDepth, 0,
                         smem_u32(&c_full[s]));
        }
      for (unsigned i = n > (unsigned)SC ? n - SC : 0; i < n; ++i)
        stage_wait(&c_full[i % SC], (i / SC) & 1, a.err);
    }
    __syncwarp();
  } else if (warp == 3) {
    // ranges, a group's 64 rows after another's: 4 words a lane, zeros (operands of
    // zero) behind the last row
    unsigned n = 0;
    for (int item = first; work_of(a, item, &t); item += step) {
      const int g = (t.i0 + rank * 128) / kGroup8 + (lane & 1);
      const bool in = g < a.groups;
      long long r = (long long)t.kb0 * kDepth + (lane >> 1);
      const unsigned* from = a.ranges + (in ? r * a.groups + g : 0);
      const long long apart = in ? 16ll * a.groups : 0;
      for (int kb = t.kb0; kb < t.kb1; ++kb, ++n, r += kDepth, from += 4 * apart) {
        const int s = n % SC;
        if (n >= (unsigned)SC) warp_wait(&c_empty[s], (n / SC - 1) & 1, a.err);
        const unsigned to =
            smem0 + kRangesAt + s * kRanges + ((lane & 1) * kDepth + (lane >> 1)) * 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool here = in && r + 16 * i < a.rows;
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(to + 64 * i),
                       "l"(here ? from + i * apart : a.ranges), "r"(here ? 4 : 0)
                       : "memory");
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];\n" ::"r"(
                         smem_u32(&c_full[s]))
                     : "memory");
      }
    }
    asm volatile("cp.async.wait_all;\n" ::: "memory");
  } else if (warp >= 4) {
    // Two teams of four warps take the stages in turn, so that one team's loads and
    // barriers run beside the other's arithmetic.  A warp has 32 inputs, the lanes of
    // tensor memory that it may touch, and all 64 rows of a stage.
    const int team = (warp - 4) >> 2, w = warp & 3;
    unsigned n = 0, tile = 0;
    for (int item = first; work_of(a, item, &t); item += step)
      for (int c0 = t.kb0, c1; c0 < t.kb1; c0 = c1, ++tile) {
        c1 = CHUNKS ? min(t.kb1, c0 + kChunk) : t.kb1;
        for (int kb = c0; kb < c1; ++kb, ++n) {
          if ((int)(n & 1) != team) continue;
          const int s = n % S, c = n % SC;
          warp_wait(&c_full[c], (n / SC) & 1, a.err);
          const uint4* const ranges =
              reinterpret_cast<const uint4*>(smem + kRangesAt + c * kRanges) +
              (w >> 1) * (kDepth / 4) + (lane & 3);
          Range4 r[4];
          bool held = true;
#pragma unroll
          for (int b = 0; b < 4; ++b) {  // 16 rows each, four of them this lane's
            const uint4 bits = ranges[4 * b];
            r[b] = range4<T>(bits);
            if constexpr (std::is_same<T, f16_t>::value) held = held && held_in_half(bits);
          }
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            unsigned v[16];
#pragma unroll
            for (int bb = 0; bb < 2; ++bb) {
              // rows of 128 bytes whose 16-byte units are xor-ed with the row
              const int row = 32 * bb + lane;
              unsigned q[4];
              codes16x2(smem0 + kCodesAt + c * kRaw + row * 128 +
                            (((2 * w + half) ^ (row & 7)) << 4),
                        q);
#pragma unroll
              for (int i = 0; i < 8; ++i) {  // block of 16 rows, input, pair of rows
                const int b = i >> 2, in = (i >> 1) & 1, k = i & 1;
                const Range4& g = r[2 * bb + b];
                v[8 * bb + i] = operand2(q[2 * b + in], 2 * k, g.s[k], g.lo[k], T());
              }
              if constexpr (std::is_same<T, f16_t>::value) {
                if (!held) {
#pragma unroll
                  for (int i = 0; i < 8; ++i) {
                    const int b = i >> 2, in = (i >> 1) & 1, k = i & 1;
                    const uint4 bits = ranges[4 * (2 * bb + b)];
                    v[8 * bb + i] = operand2_wide(q[2 * b + in], 2 * k, k ? bits.z : bits.x,
                                                  k ? bits.w : bits.y);
                  }
                }
              }
            }
            if (half == 0) {
              if (n >= (unsigned)S) warp_wait(&empty[s], (n / S - 1) & 1, a.err);
              asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
            }
            tmem_store16(tmem + kOperandAt + s * 32 + ((unsigned)(32 * w + 16 * half) << 16), v);
          }
          asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
          asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            arrive_written(&full[s]);
            arrive_leader<false>(&c_empty[c]);
          }
        }
        // the tile's sums: a lane an input, this team's half of the outputs
        if (lane == 0) stage_wait(&tm_full, tile & 1, a.err);
        __syncwarp();
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        const int i = t.i0 + rank * 128 + 32 * w + lane;
#pragma unroll 1
        for (int c = team * 128; c < team * 128 + 128; c += 32) {
          float v[32];
          tmem_load32(tmem + c + ((unsigned)(32 * w) << 16), v);
          if (c + 32 == team * 128 + 128) {
            __syncwarp();
            asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
            if (lane == 0) arrive_leader<true>(&tm_empty);
          }
          // [slab][block][outputs][128 inputs]
          const long long slab = a.parts > 1 ? t.item : first;
          float* const to = a.part + (slab * 2 + rank) * kPartFloats + c * 128 + 32 * w + lane;
          if (CHUNKS && c0 > t.kb0) {
#pragma unroll
            for (int q = 0; q < 32; ++q) v[q] += to[q * 128];
          }
          if (a.parts > 1 || (CHUNKS && c1 < t.kb1)) {
#pragma unroll
            for (int q = 0; q < 32; ++q) to[q * 128] = v[q];
          } else if (i < a.m) {
            T* const to = reinterpret_cast<T*>(a.out) + (long long)(t.j0 + c) * a.m + i;
#pragma unroll
            for (int q = 0; q < 32; ++q)
              if (t.j0 + c + q < a.n) to[(long long)q * a.m] = St<T>::v(v[q]);
          }
        }
      }
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

// The parts of a tile added in order: a block has 16 outputs of 128 inputs.
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
    const float* const from =
        a.part + ((long long)(p * tiles + tile) * 2 + rank) * kPartFloats + c * 128 + threadIdx.x;
#pragma unroll
    for (int q = 0; q < 16; ++q) v[q] += from[q * 128];
  }
  T* const out = reinterpret_cast<T*>(a.out) + (long long)j * a.m + i;
#pragma unroll
  for (int q = 0; q < 16; ++q)
    if (j + q < a.n) out[(long long)q * a.m] = St<T>::v(v[q]);
}

// ---------------------------------------------------------------------------
// y = x W^T + bias and dx = dy W, 16-bit types
// ---------------------------------------------------------------------------

// D[m][n] = sum over k of A[m][k] B[n][k] (+ bias[n]): A with k along its rows, B so or
// with k as its rows (b_mn).  Both operands by TMA, eight warps that write the result.  A
// pair of blocks has 256 x 256 of it, with two accumulators in turn, so that one is
// written while the other is summed; or (TALL) 512 x 256, which takes three quarters of
// the operand bytes a product, but all of tensor memory, so that writing shows.  Operand
// bytes out of the second-level cache bound these products.
constexpr int kPlainThreads = 128 + 32 * kWriters;
constexpr int kTurn = 4096;     // bytes of a warp's 32 x 64 of the result
constexpr int kTurnAt = 12 * kHalf;  // 6 stages of 2 x 128 rows of operands, or 4 of 3
constexpr int kPlainSmem = kTurnAt + kWriters * kTurn + 1024;

struct PlainArgs {
  CUtensorMap a, b, d;
  int m, n, kb;                 // kb: stages of the whole sum
  int b_mn;
  int tiles_m, tiles_n, parts;
  void* out;                    // [m][n]
  const void* bias;             // [n] or null
  int tma_out, bias_vec;
  float* part;                  // as in ProductArgs
  unsigned* err;
};

// The biases of a warp's 128 columns from j, four a lane, fetched while the tile's sum is
// still running; and added to the 64 values of the columns' half `g`.
template <typename T>
__device__ __forceinline__ uint2 fetch_bias(const PlainArgs& a, int j) {
  j += 4 * (threadIdx.x & 31);
  const T* const b = reinterpret_cast<const T*>(a.bias) + j;
  if (a.bias_vec && j + 4 <= a.n) return __ldg(reinterpret_cast<const uint2*>(b));
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = j + i < a.n ? Ld<T>::f(ldro(b + i)) : 0.f;
  return make_uint2(narrow2(make_float2(v[0], v[1]), T()), narrow2(make_float2(v[2], v[3]), T()));
}
template <typename T>
__device__ __forceinline__ void add_bias(uint2 bias, int g, float (&v)[64]) {
#pragma unroll
  for (int q = 0; q < 16; ++q) {
    const float2 x = widen2(__shfl_sync(0xffffffffu, bias.x, 16 * g + q), T()),
                 y = widen2(__shfl_sync(0xffffffffu, bias.y, 16 * g + q), T());
    v[4 * q] += x.x;
    v[4 * q + 1] += x.y;
    v[4 * q + 2] += y.x;
    v[4 * q + 3] += y.y;
  }
}
// A warp's 32 rows x 64 columns of the result at (i, j), a row a lane.  `turn` is 4 KB of
// shared memory of the warp's own: rows of 128 bytes in the 128-byte swizzle, whose copy
// to memory is under way when this returns.  (Rows of 64 bytes, two buffers in turn: 47
// against 45 us for 18944 rows, 512 -> 2048 bfloat16.)
template <typename T>
__device__ __forceinline__ void put_result(const PlainArgs& a, int i, int j, const float (&v)[64],
                                           char* turn) {
  const int lane = threadIdx.x & 31;
  unsigned o[32];
#pragma unroll
  for (int q = 0; q < 32; ++q) o[q] = narrow2(make_float2(v[2 * q], v[2 * q + 1]), T());
  // the buffer's last copy has been read out of it
  if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;\n" ::: "memory");
  __syncwarp();
#pragma unroll
  for (int q = 0; q < 8; ++q)
    *reinterpret_cast<uint4*>(turn + lane * 128 + ((q ^ lane) & 7) * 16) =
        make_uint4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
  if (a.tma_out) {
    fence_async_smem();
    __syncwarp();
    if (lane == 0)
      asm volatile(
          "cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];\n"
          "cp.async.bulk.commit_group;\n" ::"l"(reinterpret_cast<unsigned long long>(&a.d)),
          "r"(j), "r"(i), "r"(0), "r"(smem_u32(turn))
          : "memory");
  } else {
    __syncwarp();
    T* const out = reinterpret_cast<T*>(a.out) + (long long)i * a.n + j + lane;
    for (int r = 0; r < min(32, a.m - i); ++r) {
#pragma unroll
      for (int c = 0; c < 64; c += 32)
        if (j + lane + c < a.n)
          out[(long long)r * a.n + c] = *reinterpret_cast<const T*>(
              turn + r * 128 + ((((lane + c) >> 3) ^ r) & 7) * 16 + (lane & 7) * 2);
    }
    __syncwarp();
  }
}

// A wait for a phase that nothing completes, with nothing in flight: the error word is all
// that running out of time leaves.
__global__ void stage_wait_selftest_kernel(unsigned* err, unsigned long long limit_ns) {
  __shared__ __align__(8) unsigned long long bar;
  if (threadIdx.x == 0) {
    mbar_init(&bar, 1);
    fence_async_smem();
    stage_wait_slow<false>(smem_u32(&bar), 0u, err, limit_ns);
    stage_wait_slow<true>(smem_u32(&bar), 0u, err, limit_ns);
  }
}

template <typename T, bool TALL>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPlainThreads, 1)
    product_kernel(const __grid_constant__ PlainArgs a) {
  constexpr int R = TALL ? 2 : 1;              // blocks of 128 rows of A in either block
  constexpr int S = TALL ? 4 : 6, kStage = (R + 1) * kHalf, ROWS = R * kTile;
  extern __shared__ char smem_raw[];
  const unsigned smem0 = (smem_u32(smem_raw) + 1023u) & ~1023u;
  char* const smem = smem_raw + (smem0 - smem_u32(smem_raw));
  __shared__ unsigned long long full[S], empty[S], tm_full[2], tm_empty[2], drain;
  __shared__ unsigned tmem_base;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = blockIdx.x & 1;
  const int first = blockIdx.x >> 1, step = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tm_full[i], 1);
      mbar_init(&tm_empty[i], 2 * kWriters);
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
      for (int item = first; work_of<ROWS>(a, item, &t); item += step) {
        const int ia = t.i0 + rank * 128, jb = t.j0 + rank * 128;
        for (int kb = t.kb0; kb < t.kb1; ++kb, ++n) {
          const int s = n % S;
          if (n >= (unsigned)S) stage_wait(&empty[s], (n / S - 1) & 1, a.err);
          // both blocks' copies count on the first block's barrier
          const unsigned bar = in_leader(smem_u32(&full[s])), to = smem0 + s * kStage;
          if (rank == 0) mbar_expect_tx(&full[s], 2 * kStage);
#pragma unroll
          for (int i = 0; i < 2 * R; ++i)
            tma_box<true>(to + i * kBox, &a.a, kb * kDepth, ia + (i >> 1) * 256 + (i & 1) * 64, 0,
                          bar);
#pragma unroll
          for (int i = 0; i < 2; ++i)
            tma_box<true>(to + R * kHalf + i * kBox, &a.b, a.b_mn ? jb + 64 * i : kb * kDepth,
                          a.b_mn ? kb * kDepth : jb + 64 * i, 0, bar);
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
      const unsigned idesc = (1u << 4) | kind | ((unsigned)a.b_mn << 16) |
                             ((unsigned)(kTile / 8) << 17) | ((unsigned)(kTile / 16) << 24);
      // 16 of k further: 32 bytes along a row, or 2 groups of 8 rows
      const unsigned bs = (a.b_mn ? 2048u : 32u) >> 4;
      unsigned n = 0, tile = 0;
      for (int item = first; work_of<ROWS>(a, item, &t); item += step)
        for (int c0 = t.kb0; c0 < t.kb1; c0 += kChunk, ++tile) {
          const int c1 = min(t.kb1, c0 + kChunk);
          const unsigned d = TALL ? tmem : tmem + (tile & 1) * 256;
          if (TALL && tile >= 1) stage_wait<true>(&tm_empty[0], (tile - 1) & 1, a.err);
          if (!TALL && tile >= 2) stage_wait<true>(&tm_empty[tile & 1], (tile / 2 - 1) & 1, a.err);
          asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
          bool ready = false;
          for (int kb = c0; kb < c1; ++kb, ++n) {
            const int s = n % S;
            if (!ready) stage_wait<true>(&full[s], (n / S) & 1, a.err);
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
            const unsigned long long p = operand(smem0 + s * kStage),
                                     q = operand(smem0 + s * kStage + R * kHalf);
#pragma unroll
            for (int k = 0; k < kDepth / 16; ++k) {
#pragma unroll
              for (int r = 0; r < R; ++r)
                mma_f16<true>(d + r * 256, p + r * (kHalf >> 4) + k * (32u >> 4), q + k * bs, idesc,
                              kb > c0 || k > 0);
              if (k == 1) ready = kb + 1 < c1 && mbar_peek(&full[(n + 1) % S], ((n + 1) / S) & 1);
            }
            mma_commit<true>(&empty[s]);
          }
          mma_commit<true>(&tm_full[TALL ? 0 : tile & 1]);
        }
      // products still in flight end before tensor memory is given back
      mma_commit<true>(&drain);
      stage_wait(&drain, 0, a.err);
    }
  } else if (warp >= 4) {
    const int w = warp & 3, h = (warp - 4) >> 2;
    char* const turn = smem + kTurnAt + (warp - 4) * kTurn;
    unsigned tile = 0;
    for (int item = first; work_of<ROWS>(a, item, &t); item += step)
      for (int c0 = t.kb0; c0 < t.kb1; c0 += kChunk, ++tile) {
        const int buf = TALL ? 0 : tile & 1, c1 = min(t.kb1, c0 + kChunk);
        const uint2 bias = a.bias ? fetch_bias<T>(a, t.j0 + h * 128) : make_uint2(0u, 0u);
        if (lane == 0) stage_wait(&tm_full[buf], (TALL ? tile : tile / 2) & 1, a.err);
        __syncwarp();
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
#pragma unroll 1
        for (int g = 0; g < 2 * R; ++g) {
          const int c = h * 128 + (g & 1) * 64, i = t.i0 + (g >> 1) * 256 + rank * 128 + 32 * w;
          float v[64];
#pragma unroll
          for (int q = 0; q < 2; ++q)
            tmem_load32(tmem + (buf + (g >> 1)) * 256 + c + 32 * q + ((unsigned)(32 * w) << 16),
                        *reinterpret_cast<float(*)[32]>(v + 32 * q));
          if (g + 1 == 2 * R) {
            __syncwarp();
            asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
            if (lane == 0) arrive_leader<true>(&tm_empty[buf]);
          }
          if constexpr (!TALL) {
            // [slab][block][columns / 4][128 rows] of four columns each
            const long long slab = a.parts > 1 ? t.item : first;
            float4* const to = reinterpret_cast<float4*>(a.part + (slab * 2 + rank) * kPartFloats) +
                               c / 4 * 128 + 32 * w + lane;
            if (c0 > t.kb0) {
#pragma unroll
              for (int q = 0; q < 16; ++q) {
                const float4 f = to[q * 128];
                v[4 * q] += f.x;
                v[4 * q + 1] += f.y;
                v[4 * q + 2] += f.z;
                v[4 * q + 3] += f.w;
              }
            }
            if (a.parts > 1 || c1 < t.kb1) {
#pragma unroll
              for (int q = 0; q < 16; ++q)
                to[q * 128] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
              continue;
            }
          }
          if (i < a.m && t.j0 + c < a.n) {
            if (a.bias) add_bias<T>(bias, g & 1, v);
            put_result<T>(a, i, t.j0 + c, v, turn);
          }
        }
      }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;\n" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
  __syncthreads();
  cluster_sync();  // neither block's memory is in use any more
  if (rank == 1 && threadIdx.x == 32) stage_wait(&drain, 0, a.err);  // as in wgrad_kernel
  if (warp == 2) {
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;\n" ::"r"(tmem));
  }
}

// The parts of a tile added in order: a thread has 16 columns of a row.
template <typename T>
__global__ void __launch_bounds__(128) join_rows_kernel(const __grid_constant__ PlainArgs a) {
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
  const T* const b = reinterpret_cast<const T*>(a.bias);
  T* const out = reinterpret_cast<T*>(a.out) + (long long)i * a.n + j;
#pragma unroll
  for (int q = 0; q < 16; ++q)
    if (j + q < a.n) out[q] = St<T>::v(b ? v[q] + Ld<T>::f(ldro(b + j + q)) : v[q]);
}

// Rows at a pitch of whole 16 bytes, for TMA: a warp a row, 8 of a lane's columns at a
// time, zeros in the pitch's last columns.
template <typename T>
__global__ void __launch_bounds__(256) pitch_kernel(const T* x, long long x_row, T* y, int pitch,
                                                    long long rows, int width) {
  const int lane = threadIdx.x & 31;
  for (long long r = blockIdx.x * 8ll + threadIdx.x / 32; r < rows; r += gridDim.x * 8ll) {
    const T* const from = x + r * x_row;
    T* const to = y + r * pitch;
    for (int c0 = lane; c0 < pitch; c0 += 256) {
      T v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = T();
        if (c0 + 32 * i < width) v[i] = ldro(from + c0 + 32 * i);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c0 + 32 * i < pitch) to[c0 + 32 * i] = v[i];
    }
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

constexpr long long kMaxRows = 1ll << 27;
constexpr int kMaxSide = (1 << 22) - 64;  // 32768 tiles of 128

static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

// [rows][pitch bytes] of 16-bit values in boxes of 64 x 64 in the 128-byte swizzle.
// Outside arrives as zeros.  BYTES: boxes of 128 bytes; RESULT: 32 rows high.
enum BoxKind { BOX, BYTES, RESULT };
static bool box_map(CUtensorMap* map, const void* p, long long rows, long long cols,
                    long long pitch, BoxKind kind) {
  return encode_map(map,
                    kind == BYTES ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, p,
                    {(cuuint64_t)cols, (cuuint64_t)rows, 1},
                    {(cuuint64_t)pitch, (cuuint64_t)(pitch * rows)},
                    {kind == BYTES ? 128u : 64u, kind == RESULT ? 32u : 64u, 1});
}

static int tiles_of(long long n) { return (int)((n + kTile - 1) / kTile); }

// Parts of the sum's axis: the number whose waves take the least time, at 0.42 us a
// stage of a pair, 6 us a chunk's end, and the parts' trip through memory.  Every part of
// every tile has a slab of its own, eight for a pair of blocks at most (155 MB).
static int parts_of(long long tiles, int kb, int pairs) {
  int best = 1;
  double least = 0;
  for (int p = 1; p <= 32 && p <= kb && (p == 1 || tiles * p <= 8ll * pairs); ++p) {
    const double waves = (double)((tiles * p + pairs - 1) / pairs);
    const int stages = (kb + p - 1) / p;
    double us = waves * (0.42 * stages + 6.0 * ((stages + kChunk - 1) / kChunk));
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
  cfg.blockDim = dim3(kWgThreads);
  cfg.dynamicSmemBytes = kWgSmem;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = 2;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (cudaFuncSetAttribute(wgrad_kernel<bf16_t, false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           kWgSmem) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, wgrad_kernel<bf16_t, false>, &cfg) != cudaSuccess || n < 1) {
    cudaGetLastError();
    n = std::max(1, sm_count(device) / 2);
  }
  if (device < MAXD) known[device].store(n);
  return n;
}

// A matrix of 16-bit values as an operand: TMA reads rows at a pitch of whole 16 bytes
// that do not overlap; others are copied to such rows first.
struct Operand {
  const void* p;
  long long rows, stride;
  int cols;
  size_t copy;                  // its place in the workspace
  bool copied;
};
static int pitch_of(int cols) { return (cols + 7) / 8 * 8; }
static Operand operand_of(const void* p, long long rows, int cols, long long stride, size_t* used) {
  Operand o = {p, rows, rows == 1 ? pitch_of(cols) : stride, cols, *used, false};
  o.copied = p && (reinterpret_cast<size_t>(p) % 16 ||
                   (rows > 1 && (stride % 8 || stride < cols)));
  if (o.copied) *used += up256((size_t)rows * pitch_of(cols) * 2);
  return o;
}
template <typename T>
static int ready_operand(Operand* o, char* ws, long long stride, int device, cudaStream_t st) {
  if (!o->copied) return FA_OK;
  const int pitch = pitch_of(o->cols);
  T* const copy = reinterpret_cast<T*>(ws + o->copy);
  const long long blocks = std::min((o->rows + 7) / 8, (long long)sm_count(device) * 16);
  pitch_kernel<T><<<(unsigned)blocks, 256, 0, st>>>(static_cast<const T*>(o->p), stride, copy,
                                                    pitch, o->rows, o->cols);
  FAB_LAUNCH_CHECK();
  o->p = copy;
  o->stride = pitch;
  o->copied = false;
  return FA_OK;
}

// What a call takes from its workspace: sums of columns, operands' copies, and the parts
// of one product after the other.
struct LinearPlan {
  Operand x, dy, w;
  int y_parts, dx_parts, dw_parts, pairs;
  size_t part, bytes;
};
static int stages_of(long long n) { return (int)((n + kDepth - 1) / kDepth); }
static LinearPlan linear_plan(const fa_linear8& l, int device) {
  LinearPlan p = {};
  size_t used = l.dbias ? up256(norm_ws_bytes(l.rows, l.outputs, device)) : 0, part = 0;
  if (l.dtype != FA_F32) {
    if (l.y) p.x = operand_of(l.x, l.rows, l.inputs, l.x_stride, &used);
    if (l.dx || l.dweight) p.dy = operand_of(l.dy, l.rows, l.outputs, l.dy_stride, &used);
    if (l.y || l.dx) p.w = operand_of(l.weight, l.outputs, l.inputs, l.weight_stride, &used);
    p.pairs = resident_pairs(device);
    const int in = tiles_of(l.inputs), out = tiles_of(l.outputs);
    const long long rows = tiles_of(l.rows);
    const auto parts = [&](bool wanted, long long tiles, int kb, bool even) {
      if (!wanted) return 1;
      const int n = tiles > p.pairs && !even ? 1 : parts_of(tiles, kb, p.pairs);
      const long long slabs = n > 1 ? tiles * n : kb > kChunk ? std::min(tiles, (long long)p.pairs) : 0;
      part = std::max(part, (size_t)slabs * 2 * kPartFloats * sizeof(float));
      return n;
    };
    // a long sum over more tiles than pairs is cut for the sake of its last wave (65280 rows,
    // 4096 x 4096: 2.0 ms in two parts, 2.4 in one)
    p.y_parts = parts(l.y, rows * out, stages_of(l.inputs), false);
    p.dx_parts = parts(l.dx, rows * in, stages_of(l.outputs), false);
    p.dw_parts = parts(l.dweight, (long long)in * out, stages_of(l.rows), l.rows > kLongest);
  }
  if (l.dtype == FA_F32) {
    // parts that fill the multiprocessors twice, of 256 and more of k; of sums longer than
    // 32768, also parts whose last wave is fuller, in 77 MB at most (65280 rows, 2560 x 2048:
    // dW 18.0 ms in one part, 14.1 in three)
    const auto parts = [&](bool wanted, long long m, long long n, long long k) {
      const long long tiles = ((m + kLaneTile - 1) / kLaneTile) * ((n + kLaneTile - 1) / kLaneTile);
      const long long room = 2ll * sm_count(device);
      if (!wanted) return 1;
      int c = (int)std::max(1ll, std::min((k + 255) / 256, room / tiles));
      const auto waves = [&](int q) { return (double)((tiles * q + room - 1) / room) / q; };
      if (k > kLongest && tiles > room)
        for (int q = 2; tiles * q <= 4 * room; ++q)
          if (waves(q) < waves(c)) c = q;
      if (c > 1) part = std::max(part, (size_t)(sizeof(float) * c * m * n));
      return c;
    };
    p.y_parts = parts(l.y, l.rows, l.outputs, l.inputs);
    p.dx_parts = parts(l.dx, l.rows, l.inputs, l.outputs);
    p.dw_parts = parts(l.dweight, l.outputs, l.inputs, l.rows);
  }
  p.part = used;
  p.bytes = used + part;
  return p;
}

static int linear_check(const fa_linear8* l) {
  if (!l) return FA_E_ARG;
  if (!train_dtype(l->dtype)) return FA_E_DTYPE;
  if (l->rows <= 0 || l->inputs <= 0 || l->outputs <= 0 || l->rows > kMaxRows ||
      l->inputs > kMaxSide || l->outputs > kMaxSide)
    return FA_E_SHAPE;
  const int item = item_size(l->dtype);
  for (const void* q : {l->x, l->dy, l->weight, l->bias, (const void*)l->y, (const void*)l->dx,
                        (const void*)l->dweight, (const void*)l->dbias})
    if (reinterpret_cast<size_t>(q) % item) return FA_E_ARG;
  if (!l->codes != !l->ranges || reinterpret_cast<size_t>(l->codes) % 16 ||
      reinterpret_cast<size_t>(l->ranges) % 8)
    return FA_E_ARG;
  if ((l->y && (!l->x || !l->weight)) || (l->dx && (!l->dy || !l->weight)) ||
      (l->dweight && (!l->dy || !l->codes)) || (l->dbias && !l->dy))
    return FA_E_ARG;
  return FA_OK;
}

int stage_wait_selftest(unsigned long long limit_ns, int device, cudaStream_t st) {
  if (limit_ns > 1000000000ull) return FA_E_ARG;
  FAB_DEVICE_SCOPE(device);
  unsigned* const w = wait_error_word();
  if (!w) return FA_E_INTERNAL;
  stage_wait_selftest_kernel<<<1, 32, 0, st>>>(w, limit_ns);
  FAB_LAUNCH_CHECK();
  return FA_OK;
}

int linear8_ws_bytes(const fa_linear8* l, int device, size_t* out) {
  if (const int rc = linear_check(l)) return rc;
  *out = linear_plan(*l, device).bytes;
  return FA_OK;
}

static int workspace_check(const LinearPlan& p, const void* ws, size_t bytes) {
  return p.bytes && (!ws || reinterpret_cast<size_t>(ws) % 256 || bytes < p.bytes) ? FA_E_ARG : FA_OK;
}

// D (rows x cols) = A (rows x depth) B: B with depth along its rows, or as its rows.
// Whether the taller tiles take less time: waves of tiles, at 0.40 us a stage and 2 us a
// tile's end against 0.69 and 6.  Low tiles have two accumulators, so between waves the
// next tile's products run beside an end (18944 rows, bfloat16, sums of 512 to 8192 terms:
// 0.40 us a stage in 2, 4 and 8 waves, and 14, 16 and 17 us besides, the launch among
// them); a single wave, which parts_of is about, shows all of it.  Measured: 18944 rows,
// 4096 -> 1024, 2 waves of tall tiles 102 us, 4 of low ones 117; 4096 -> 512, 1 and 2
// waves, 59 and 66; 512 -> 2048, 4 waves of tall ones 54, 8 of low ones 49.
static bool tall_pays(long long rows, int cols, int kb, int pairs) {
  if (kb > kChunk) return false;
  const long long wide = tiles_of(cols);
  const auto waves = [&](long long row_tiles) { return (row_tiles * wide + pairs - 1) / pairs; };
  return waves((rows + 511) / 512) * (0.69 * kb + 6.0) < waves((rows + 255) / 256) * (0.40 * kb + 2.0);
}

template <typename T>
static int product_run(const Operand& x, const Operand& w, int depth, bool w_mn, const void* bias,
                       void* out, long long rows, int cols, int parts, char* part,
                       const LinearPlan& plan, cudaStream_t st) {
  PlainArgs a = {};
  a.tma_out = cols % 8 == 0 && reinterpret_cast<size_t>(out) % 16 == 0;
  if (!box_map(&a.a, x.p, rows, depth, x.stride * 2, BOX) ||
      !box_map(&a.b, w.p, w.rows, w.cols, w.stride * 2, BOX) ||
      (a.tma_out && !box_map(&a.d, out, rows, cols, cols * 2ll, RESULT)))
    return FA_E_INTERNAL;
  a.m = (int)rows;
  a.n = cols;
  a.kb = stages_of(depth);
  a.b_mn = w_mn;
  a.tiles_m = tiles_of(rows);
  a.tiles_n = tiles_of(cols);
  a.parts = parts;
  a.out = out;
  a.bias = bias;
  a.bias_vec = reinterpret_cast<size_t>(bias) % 16 == 0;
  a.part = reinterpret_cast<float*>(part);
  a.err = wait_error_word();
  if (!a.err) return FA_E_INTERNAL;  // a wait that gave up could not be reported
  if (parts == 1 && tall_pays(rows, cols, a.kb, plan.pairs)) {
    a.tiles_m = (int)((rows + 511) / 512);
    FAB_TRY(cudaFuncSetAttribute(product_kernel<T, true>,
                                 cudaFuncAttributeMaxDynamicSharedMemorySize, kPlainSmem));
    product_kernel<T, true><<<2 * std::min(a.tiles_m * a.tiles_n, plan.pairs), kPlainThreads,
                              kPlainSmem, st>>>(a);
    FAB_LAUNCH_CHECK();
    return FA_OK;
  }
  FAB_TRY(cudaFuncSetAttribute(product_kernel<T, false>,
                               cudaFuncAttributeMaxDynamicSharedMemorySize, kPlainSmem));
  const int items = a.tiles_m * a.tiles_n * parts;
  product_kernel<T, false><<<2 * std::min(items, plan.pairs), kPlainThreads, kPlainSmem, st>>>(a);
  FAB_LAUNCH_CHECK();
  if (parts > 1) {
    join_rows_kernel<T><<<(unsigned)(a.tiles_m * a.tiles_n * 32), 128, 0, st>>>(a);
    FAB_LAUNCH_CHECK();
  }
  return FA_OK;
}

template <typename T>
static int wgrad_run(const fa_linear8& l, const Operand& dy, char* part, const LinearPlan& plan,
                     cudaStream_t st) {
  ProductArgs a = {};
  const long long groups = groups8(l.inputs);
  if (!box_map(&a.dy, dy.p, l.rows, l.outputs, dy.stride * 2, BOX) ||
      !box_map(&a.codes, l.codes, l.rows, groups * kGroup8, groups * kGroup8, BYTES))
    return FA_E_INTERNAL;
  a.m = l.inputs;
  a.n = l.outputs;
  a.kb = stages_of(l.rows);
  a.tiles_m = tiles_of(l.inputs);
  a.tiles_n = tiles_of(l.outputs);
  a.parts = plan.dw_parts;
  a.ranges = static_cast<const unsigned*>(l.ranges);
  a.rows = l.rows;
  a.groups = (int)groups;
  a.out = l.dweight;
  a.part = reinterpret_cast<float*>(part);
  a.err = wait_error_word();
  if (!a.err) return FA_E_INTERNAL;  // a wait that gave up could not be reported
  const auto kernel = (a.kb + a.parts - 1) / a.parts > kChunk ? wgrad_kernel<T, true>
                                                              : wgrad_kernel<T, false>;
  FAB_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kWgSmem));
  const int items = a.tiles_m * a.tiles_n * a.parts;
  kernel<<<2 * std::min(items, plan.pairs), kWgThreads, kWgSmem, st>>>(a);
  FAB_LAUNCH_CHECK();
  if (a.parts > 1) {
    join_parts_kernel<T><<<(unsigned)(a.tiles_m * a.tiles_n * 32), 128, 0, st>>>(a);
    FAB_LAUNCH_CHECK();
  }
  return FA_OK;
}

template <typename T>
static int linear_forward(const fa_linear8& l, LinearPlan& p, char* ws, int device, cudaStream_t st) {
  if (const int rc = ready_operand<T>(&p.x, ws, l.x_stride, device, st)) return rc;
  if (const int rc = ready_operand<T>(&p.w, ws, l.weight_stride, device, st)) return rc;
  return product_run<T>(p.x, p.w, l.inputs, false, l.bias, l.y, l.rows, l.outputs, p.y_parts,
                        ws + p.part, p, st);
}

static int bias_run(const fa_linear8& l, void* ws, size_t bytes, int device, cudaStream_t st) {
  return bias_grad_impl(l.dy, l.dy_stride, l.dbias, l.dtype, l.rows, l.outputs, ws, bytes, device, st);
}
// Whether the bias's gradient runs beside dW: where dW's tiles leave multiprocessors idle,
// and dy is large enough to be worth a second stream's host time.  All gradients, bfloat16,
// beside and after one another: 16320 rows, 1024 -> 4096, 219 and 252 us; 65280 rows,
// 256 -> 256, 70 and 84 us; 510 rows, 1024 -> 4096, 45 and 53 us.
static bool bias_beside(const fa_linear8& l, const LinearPlan& p) {
  const long long items = (long long)tiles_of(l.inputs) * tiles_of(l.outputs) * p.dw_parts;
  return items <= p.pairs - 6 && l.rows * l.outputs >= 1 << 20;
}

template <typename T>
static int linear_backward(const fa_linear8& l, LinearPlan& p, char* ws, size_t bytes, bool beside,
                           int device, cudaStream_t st) {
  if (const int rc = ready_operand<T>(&p.dy, ws, l.dy_stride, device, st)) return rc;
  if (const int rc = ready_operand<T>(&p.w, ws, l.weight_stride, device, st)) return rc;
  if (l.dx)
    if (const int rc = product_run<T>(p.dy, p.w, l.outputs, true, nullptr, l.dx, l.rows, l.inputs,
                                      p.dx_parts, ws + p.part, p, st))
      return rc;
  if (!l.dweight) return FA_OK;
  if (!beside) return wgrad_run<T>(l, p.dy, ws + p.part, p, st);
  Side* const side = side_fork(device, st);
  int rc = wgrad_run<T>(l, p.dy, ws + p.part, p, st);
  if (!rc) rc = bias_run(l, ws, bytes, device, side ? side->stream : st);
  if (side) {
    const int joined = side_join(side, device, st);
    if (!rc) rc = joined;
  }
  return rc;
}

template <LaneOperand A, LaneOperand B>
static int lanes_run(LaneArgs a, int parts, float* out, float* part, int device, cudaStream_t st) {
  const long long stages = (a.k + kLaneDepth - 1) / kLaneDepth;
  a.per_part = (stages + parts - 1) / parts * kLaneDepth;
  a.parts = (int)((a.k + a.per_part - 1) / a.per_part);
  a.d = a.parts > 1 ? part : out;
  const dim3 grid((unsigned)((a.m + kLaneTile - 1) / kLaneTile),
                  (unsigned)((a.n + kLaneTile - 1) / kLaneTile), (unsigned)a.parts);
  if (a.per_part > kLongest) lanes_kernel<A, B, true><<<grid, 256, 0, st>>>(a);
  else lanes_kernel<A, B, false><<<grid, 256, 0, st>>>(a);
  FAB_LAUNCH_CHECK();
  if (a.parts > 1) {
    const long long size = (long long)a.m * a.n;
    join_lanes_kernel<<<(unsigned)std::min((size + 255) / 256, 8ll * sm_count(device)), 256, 0, st>>>(
        part, out, a.parts, size, a.bias, a.n);
    FAB_LAUNCH_CHECK();
  }
  return FA_OK;
}
static int whole4(const void* p, long long row, long long rows) {
  return reinterpret_cast<size_t>(p) % 16 == 0 && (rows == 1 || row % 4 == 0);
}

static int lanes_forward(const fa_linear8& l, const LinearPlan& p, char* ws, int device,
                         cudaStream_t st) {
  LaneArgs a = {};
  a.a = static_cast<const float*>(l.x);
  a.a_row = l.x_stride;
  a.a_vec = whole4(l.x, l.x_stride, l.rows);
  a.b = static_cast<const float*>(l.weight);
  a.b_row = l.weight_stride;
  a.b_vec = whole4(l.weight, l.weight_stride, l.outputs);
  a.k = l.inputs;
  a.m = (int)l.rows;
  a.n = l.outputs;
  a.bias = static_cast<const float*>(l.bias);
  return lanes_run<ALONG_K, ALONG_K>(a, p.y_parts, static_cast<float*>(l.y),
                                     reinterpret_cast<float*>(ws + p.part), device, st);
}

static int lanes_backward(const fa_linear8& l, const LinearPlan& p, char* ws, int device,
                          cudaStream_t st) {
  LaneArgs a = {};
  a.a = static_cast<const float*>(l.dy);
  a.a_row = l.dy_stride;
  a.a_vec = whole4(l.dy, l.dy_stride, l.rows);
  if (l.dx) {
    a.b = static_cast<const float*>(l.weight);
    a.b_row = l.weight_stride;
    a.b_vec = whole4(l.weight, l.weight_stride, l.outputs);
    a.k = l.outputs;
    a.m = (int)l.rows;
    a.n = l.inputs;
    if (const int rc = lanes_run<ALONG_K, ROWS_K>(a, p.dx_parts, static_cast<float*>(l.dx),
                                                  reinterpret_cast<float*>(ws + p.part), device, st))
      return rc;
  }
  if (!l.dweight) return FA_OK;
  a.codes = static_cast<const unsigned char*>(l.codes);
  a.ranges = static_cast<const float2*>(l.ranges);
  a.groups = (int)groups8(l.inputs);
  a.k = l.rows;
  a.m = l.outputs;
  a.n = l.inputs;
  return lanes_run<ROWS_K, CODES_K>(a, p.dw_parts, static_cast<float*>(l.dweight),
                                    reinterpret_cast<float*>(ws + p.part), device, st);
}

int linear8_impl(const fa_linear8* l, void* ws, size_t bytes, int device, cudaStream_t st) {
  if (const int rc = linear_check(l)) return rc;
  if (l->dx || l->dweight || l->dbias || (!l->y && !l->codes) || !l->x) return FA_E_ARG;
  LinearPlan p = linear_plan(*l, device);
  if (const int rc = workspace_check(p, ws, bytes)) return rc;
  FAB_DEVICE_SCOPE(device);
  if (l->codes)
    if (const int rc = pack8_impl(l->x, l->x_stride, l->codes, l->ranges, l->dtype, l->rows,
                                  l->inputs, device, st))
      return rc;
  if (!l->y) return FA_OK;
  if (l->dtype == FA_F32) return lanes_forward(*l, p, static_cast<char*>(ws), device, st);
  if (l->dtype == FA_F16) return linear_forward<f16_t>(*l, p, static_cast<char*>(ws), device, st);
  return linear_forward<bf16_t>(*l, p, static_cast<char*>(ws), device, st);
}

int linear8_backward_impl(const fa_linear8* l, void* ws, size_t bytes, int device, cudaStream_t st) {
  if (const int rc = linear_check(l)) return rc;
  if (l->y || (!l->dx && !l->dweight && !l->dbias)) return FA_E_ARG;
  LinearPlan p = linear_plan(*l, device);
  if (const int rc = workspace_check(p, ws, bytes)) return rc;
  FAB_DEVICE_SCOPE(device);
  char* const work = static_cast<char*>(ws);
  const bool beside = l->dbias && l->dweight && l->dtype != FA_F32 && bias_beside(*l, p);
  if (l->dbias && !beside)
    if (const int rc = bias_run(*l, ws, bytes, device, st)) return rc;
  if (l->dtype == FA_F16) return linear_backward<f16_t>(*l, p, work, bytes, beside, device, st);
  if (l->dtype == FA_BF16) return linear_backward<bf16_t>(*l, p, work, bytes, beside, device, st);
  return lanes_backward(*l, p, work, device, st);
}

}  // namespace fab
