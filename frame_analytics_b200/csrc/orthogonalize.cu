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
//
// Three launches serve up to 128 matrices of up to 8 shapes: momentum and norms,
// packing, and one persistent kernel for all products of all steps.  Matrices
// that fit one block have a kernel of their own.
//
// Measured on one B200, a call: 4096 x 8192 bfloat16 2.7 ms (0.88 PFLOP/s of
// the products it cannot do without, at the 1.56 GHz that the power limit leaves),
// 12 x 768 x 768 bfloat16 0.27 ms (0.40), 2304 x 768 float32 0.26 ms (0.086,
// three times that in products run).  Large matrices are bound by the products
// (0.45 us for 256 x 256 x 64 on a pair of blocks) and the ends of the phases,
// middle ones by operand bytes out of the second-level cache and the
// ends of the phases, small ones by the latency of 15 dependent products (at
// least 4 us each).
//
// Number formats.  The products run on the tensor cores with float16 operands
// and float32 accumulators; float16 has three more bits than bfloat16 at the
// same rate, and powers of two per step (from a bound on the singular values)
// keep every value inside its range.  A rounding of relative size e in the
// term a X grows with the small singular values (by a per step), while one in
// B X does not: B vanishes on small singular directions.  So X travels as a
// pair of float16 (hi, lo: 22 bits); only hi enters the products and the term
// a X uses both.  The diagonals of A and B, which hold most of their mass near
// convergence, travel in float32 beside the float16 off-diagonal parts O:
//   A = D + O:  A^2 = D^2 + D O + O D + O O,   B X = diag(B) X + offdiag(B) X.
// Together: 5e-4 to 1.2e-3 relative for bfloat16 matrices (bfloat16 products:
// 1e-2 to 1e-1).  float32 and float16 matrices run every product three times
// (hi hi + hi lo + lo hi), which is float32-like (about 1e-6).
#include <algorithm>
#include <atomic>
#include <cmath>
#include <new>

#include "tensor.cuh"
#include "train.cuh"

namespace fab {

constexpr int kMats = 128;         // matrices of one launch sequence
constexpr int kGroups = 8;         // shapes of one launch sequence
constexpr int kMaxSteps = 32;
constexpr int kNormBlocks = 512;   // partial sums of squares of one matrix, at most

constexpr int BM = 128;            // tile rows: the lanes of tensor memory
constexpr int BK = 64;             // 128 bytes of float16: one swizzle row
constexpr int kEpilogue = 256;     // 8 epilogue warps: 4 quarters of the rows x 2 column halves
constexpr int kSplitUnits = 148;   // parts of split tiles at most: one a multiprocessor
constexpr int kSplitTiles = kSplitUnits / 2;
constexpr int kMaxParts = 16;
constexpr int kPart = BM * 64;     // floats of a part: split tiles have 64 columns
constexpr int kThreads = 128 + kEpilogue;  // producer, issuer, allocator, spare before them
// The tensor cores add into an accumulator with truncation, a relative loss of
// about 2^-25 for each 16 columns of K, always towards zero.  float32-like
// products therefore move their sums to registers (rounded adds) every
// kChunk K blocks, and keep the small products hi lo + lo hi in an accumulator
// of their own: 2304 x 768 float32 is 2e-5 off without, see the tests.
constexpr int kChunk = 4;

// Tensor maps of one shape: X twice (it alternates), O and offdiag(B); hi, lo.
enum { MAP_X0, MAP_X1, MAP_A, MAP_B, kMaps };

struct NsGroup {
  CUtensorMap map[kMaps][2];
  int rows, cols, s, l;            // s = shorter side, l = longer
  int tall, batch, first;          // matrices [first, first + batch)
  int px, pa;                      // row pitches of X and of A, B in elements
  int bn_sym, bn_app;              // tile columns of the symmetric products and of B X
  int tiles_sym, tiles_app;        // tiles of one matrix (of pairs, where blocks pair up)
  int ks[2];                       // parts of K that A's and A^2's tiles are split into
  int slot;                        // the first of this shape's tiles among those split
  __half *x[2][2], *a[2], *b[2];   // [alternation][hi, lo]
  float *da, *db;                  // diagonals, [batch][pa]
};

struct NsMat {
  const void* src;                 // x, or the gradient
  void* dst;                       // out, or the weight
  float* mom;                      // momentum, or null
  long long src_row, dst_row;
  float step;                      // W <- decay W - step O
  short cols, s, l;                // of one that fits a block; s, l: shorter, longer side
  bool tall;
  unsigned char group;
  bool vec;                        // rows are whole aligned 16-byte vectors
  bool vec_dst;                    // the result's rows are whole aligned vectors of four
};

struct NsStep {
  float a, b, c;
  int ex, ea, eb, ex2;             // stored value = true value x 2^e: X, A, B, next X
};

struct NsArgs {
  NsGroup g[kGroups];
  NsMat m[kMats];
  NsStep k[kMaxSteps];
  int groups, mats, steps;
  int tiles[3];                    // of the three products, over all matrices
  unsigned* done;                  // [3][kMats] finished tiles of the three products
  unsigned* joins;                 // [2][kSplitTiles] finished parts of the split tiles
  float* parts;                    // [kSplitUnits] sums of a part of a tile
  unsigned* failed;                // set when a wait of this call gave up
  double* part;                    // [kMats][kNormBlocks]
  unsigned* err;
  unsigned long long limit_ns;     // of a wait
  int pair;                        // two blocks a tile
  int ks;                          // parts of a tile at most
  float mu, decay;
  int nesterov;
};

// ---------------------------------------------------------------------------
// momentum, norm, packing
// ---------------------------------------------------------------------------

// Both passes read the gradient and the momentum once each: a warp takes 512
// columns of a row at a time, 8 to a lane and load.
constexpr int kSpan = 512;

// Update values u[8] of columns [c, c + 8) of row r (zeros past the last
// column).  STORE writes the new momentum; otherwise it was written before.
template <typename T, bool STORE>
__device__ __forceinline__ void ns_update(const NsArgs& a, const NsMat& m, int r, int c, int cols,
                                          float (&u)[8]) {
  const T* src = reinterpret_cast<const T*>(m.src) + r * m.src_row + c;
  const int n = min(8, cols - c);
  if (m.vec) {  // n is 8
    __align__(16) T e[8];
#pragma unroll
    for (int q = 0; q < (int)sizeof(T) / 2; ++q)
      reinterpret_cast<uint4*>(e)[q] = __ldg(reinterpret_cast<const uint4*>(src) + q);
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = Ld<T>::f(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = i < n ? Ld<T>::f(src[i]) : 0.f;
  }
  if (!m.mom) return;
  float* mom = m.mom + (long long)r * cols + c;
  __align__(16) float v[8];
  if (m.vec) {
    reinterpret_cast<float4*>(v)[0] = reinterpret_cast<const float4*>(mom)[0];
    reinterpret_cast<float4*>(v)[1] = reinterpret_cast<const float4*>(mom)[1];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? mom[i] : 0.f;
  }
  if constexpr (STORE) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = fmaf(a.mu, v[i], u[i]);
    if (m.vec) {
      reinterpret_cast<float4*>(mom)[0] = reinterpret_cast<const float4*>(v)[0];
      reinterpret_cast<float4*>(mom)[1] = reinterpret_cast<const float4*>(v)[1];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) mom[i] = v[i];
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) u[i] = a.nesterov ? fmaf(a.mu, v[i], u[i]) : v[i];
}

// Updates the momentum and sums the squares of the update, in double: float32
// squares of a float32 matrix could leave its range.
template <typename T>
__global__ void __launch_bounds__(256) ns_norm_kernel(const __grid_constant__ NsArgs a) {
  __shared__ double sm[32];
  const NsMat& m = a.m[blockIdx.y];
  const NsGroup& g = a.g[m.group];
  const int spans = (g.cols + kSpan - 1) / kSpan, lane = threadIdx.x & 31;
  const long long items = (long long)g.rows * spans;
  double ss = 0;
  for (long long it = blockIdx.x * 8ll + (threadIdx.x >> 5); it < items; it += 8ll * gridDim.x) {
    const int r = (int)(it / spans), c0 = (int)(it - (long long)r * spans) * kSpan + 8 * lane;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = c0 + 256 * h;
      if (c >= g.cols) continue;
      float u[8];
      ns_update<T, true>(a, m, r, c, g.cols, u);
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += (double)u[i] * u[i];
    }
  }
  ss = block_sum(ss, sm);
  if (threadIdx.x == 0) a.part[blockIdx.y * kNormBlocks + blockIdx.x] = ss;
  // the product kernel's counters, for this call
  if (blockIdx.x == 0 && threadIdx.x < 3) a.done[threadIdx.x * kMats + blockIdx.y] = 0u;
  if (blockIdx.x == 0 && blockIdx.y == 0) {
    if (threadIdx.x == 3) *a.failed = 0u;
    if (threadIdx.x < 2 * kSplitTiles) a.joins[threadIdx.x] = 0u;
  }
}

__device__ __forceinline__ void split_half(float v, __half* hi, __half* lo) {
  *hi = __float2half_rn(v);
  *lo = __float2half_rn(v - __half2float(*hi));
}

// X = update / norm as (hi, lo) at the pitch px; the pitch's tail is zeroed.
template <typename T>
__global__ void __launch_bounds__(256) ns_pack_kernel(const __grid_constant__ NsArgs a,
                                                      int norm_blocks) {
  __shared__ double sm[32];
  const NsMat& m = a.m[blockIdx.y];
  const NsGroup& g = a.g[m.group];
  double ss = 0;
  for (int i = threadIdx.x; i < norm_blocks; i += 256)
    ss += __ldg(a.part + blockIdx.y * kNormBlocks + i);
  ss = block_sum(ss, sm);
  const bool finite = ss <= 1.7e308;
  const double inv = ss > 0 ? ldexp(1.0, a.k[0].ex) / sqrt(ss) : 0.0;
  // inv = f 2^e, the power in two exact steps: no product leaves float's range
  int e;
  const float f = (float)frexp(inv, &e);
  const float e1 = ldexpf(1.f, e / 2), e2 = ldexpf(1.f, e - e / 2);
  const int spans = (g.px + kSpan - 1) / kSpan, lane = threadIdx.x & 31;
  const long long items = (long long)g.rows * spans;
  const long long base = (long long)(blockIdx.y - g.first) * g.rows * g.px;
  for (long long it = blockIdx.x * 8ll + (threadIdx.x >> 5); it < items; it += 8ll * gridDim.x) {
    const int r = (int)(it / spans), c0 = (int)(it - (long long)r * spans) * kSpan + 8 * lane;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = c0 + 256 * h;
      if (c >= g.px) continue;
      float u[8] = {};
      if (c < g.cols) ns_update<T, false>(a, m, r, c, g.cols, u);
      __align__(16) __half hi[8], lo[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float x = u[i] * e1 * e2 * f;
        if (!finite && c + i < g.cols) x = __int_as_float(0x7fffffff);
        split_half(x, &hi[i], &lo[i]);
      }
      const long long o = base + (long long)r * g.px + c;
      *reinterpret_cast<uint4*>(g.x[0][0] + o) = *reinterpret_cast<const uint4*>(hi);
      *reinterpret_cast<uint4*>(g.x[0][1] + o) = *reinterpret_cast<const uint4*>(lo);
    }
  }
}

// ---------------------------------------------------------------------------
// the products: tcgen05, TMA
// ---------------------------------------------------------------------------

__device__ __forceinline__ unsigned ld_acquire(const unsigned* p) {
  unsigned v;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];\n" : "=r"(v) : "l"(p) : "memory");
  return v;
}

// Bounded wait on an mbarrier phase, or on a counter of finished tiles, that
// tells whether it was reached.  On giving up (after the launch's limit, or when
// another wait of the launch already has) it records FA_E_TIMEOUT and the caller
// leaves its loop.  The launch's own word tells the other waits: the host-mapped
// word is across the bus and is only written.  No wait spans more than the few
// tiles that it is for, the longest about 0.1 s (65536 blocks of K): a launch may
// last longer than the limit.
template <bool PAIR>
__device__ __noinline__ bool wait_slow(unsigned bar, unsigned parity, const unsigned* flag,
                                       unsigned want, const NsArgs& a) {
  const unsigned long long t0 = globaltimer_ns();
  for (unsigned i = 1;; ++i) {
    if (flag ? ld_acquire(flag) >= want : mbar_try_pair<PAIR>(bar, parity)) return true;
    if ((i & 255u) == 0u) {
      const bool failed = *reinterpret_cast<volatile unsigned*>(a.failed) != 0u;
      if (failed || globaltimer_ns() - t0 > a.limit_ns) {
        if (!failed) {
          *reinterpret_cast<volatile unsigned*>(a.failed) = 1u;
          *reinterpret_cast<volatile unsigned*>(a.err) = (unsigned)FA_E_TIMEOUT;
          __threadfence_system();
        }
        return false;
      }
    }
  }
}
// PAIR: threads of the pair's other block arrive there, too.
template <bool PAIR = false>
__device__ __forceinline__ bool wait_bar(unsigned long long* bar, unsigned parity,
                                         const NsArgs& a) {
  const unsigned b = smem_u32(bar);
#pragma unroll 1
  for (int i = 0; i < 8; ++i)
    if (mbar_try_pair<PAIR>(b, parity)) return true;
  return wait_slow<PAIR>(b, parity, nullptr, 0, a);
}
__device__ __forceinline__ bool wait_flag(const unsigned* flag, unsigned want, const NsArgs& a) {
  if (ld_acquire(flag) >= want) return true;
  return wait_slow<false>(0, 0, flag, want, a);
}

// Where a tile is.  Tiles are numbered phase by phase (A, A^2, B X of step 0,
// of step 1, ...), inside a phase matrix by matrix; block (or pair) c takes
// numbers c, c + units, ...  A tile waits only for tiles of earlier phases, and
// every block is resident, so the lowest unfinished tile can always proceed.
struct Tile {
  int phase, step;                 // phase 0: A, 1: A^2, 2: B X
  int group, mat;                  // mat counts over the whole call
  int i0, j0, bn, kb0, kb1;        // i0: this block's 128 rows; K blocks [kb0, kb1)
  int ks, part, slot, region;      // parts of K, which one, the tile and its first part's place
};

// Tiles of the lower triangle of an s x s product, bm rows by bn columns: row
// block ti takes the tiles that start at or left of its own last column.
__host__ __device__ __forceinline__ int sym_tiles(int s, int bm, int bn) {
  const int T = (s + bm - 1) / bm, u = T / 2;
  if (bm == bn) return T * (T + 1) / 2;
  if (bm < bn) return T % 2 ? (u + 1) * (u + 1) : u * (u + 1);  // bn = 2 bm
  return T * (T + 1);                                            // bm = 2 bn
}

template <bool PAIR>
struct Walk {
  static constexpr int kRows = PAIR ? 2 * BM : BM;
  int step = 0, phase = 0;
  const int units, rank;
  long long t;
  __device__ Walk() : units(PAIR ? gridDim.x / 2 : gridDim.x), rank(PAIR ? blockIdx.x & 1 : 0),
                      t(PAIR ? blockIdx.x / 2 : blockIdx.x) {}
  __device__ bool next(const NsArgs& a, Tile* o) {
    for (;;) {
      const int n = a.tiles[phase];
      if (t < n) break;
      t -= n;
      if (++phase == 3) {
        phase = 0;
        if (++step == a.steps) return false;
      }
    }
    int r = (int)t, gi = 0;
    for (;; ++gi) {
      const NsGroup& g = a.g[gi];
      const int n = g.batch * (phase == 2 ? g.tiles_app : g.tiles_sym * g.ks[phase]);
      if (r < n) break;
      r -= n;
    }
    const NsGroup& g = a.g[gi];
    o->phase = phase;
    o->step = step;
    o->group = gi;
    o->ks = 1;
    o->part = 0;
    o->kb0 = 0;
    int ti, tj;
    if (phase == 2) {
      const int b = r / g.tiles_app;
      r -= b * g.tiles_app;
      o->mat = g.first + b;
      o->bn = g.bn_app;
      const int tn = (g.cols + o->bn - 1) / o->bn;
      ti = r / tn;
      tj = r - ti * tn;
      o->kb1 = (g.s + BK - 1) / BK;
    } else {
      const int ks = g.ks[phase];
      const int tile = r / ks;
      o->ks = ks;
      o->part = r - tile * ks;
      o->slot = g.slot + tile;
      // a place of its own for both products: matrices are in different phases
      o->region = o->slot * a.ks;
      const int b = tile / g.tiles_sym;
      r = tile - b * g.tiles_sym;
      o->mat = g.first + b;
      o->bn = g.bn_sym;
      if (o->bn == kRows) {
        int u = (int)((sqrtf(8.f * r + 1.f) - 1.f) * 0.5f);
        while (u * (u + 1) / 2 > r) --u;
        while ((u + 1) * (u + 2) / 2 <= r) ++u;
        ti = u;
        tj = r - u * (u + 1) / 2;
      } else {
        int u = (int)((sqrtf(4.f * r + 1.f) - 1.f) * 0.5f);
        while (u * (u + 1) > r) --u;
        while ((u + 1) * (u + 2) <= r) ++u;
        r -= u * (u + 1);
        ti = o->bn > kRows ? 2 * u + r / (u + 1) : u;
        tj = o->bn > kRows ? r % (u + 1) : r;
      }
      const int kb = ((phase == 0 ? g.l : g.s) + BK - 1) / BK;
      o->kb0 = (int)((long long)kb * o->part / ks);
      o->kb1 = (int)((long long)kb * (o->part + 1) / ks);
    }
    o->i0 = ti * kRows + rank * BM;
    o->j0 = tj * o->bn;
    t += units;
    return true;
  }
};

// Shared memory: operand stages, then a 32 x 32 float buffer for each epilogue
// warp.  A stage holds 64 K columns of the row operand (128 rows) and of the
// column operand (256 rows; split: 128, twice).
// A pair of blocks shares a tile of 256 rows: each block keeps its own 128 rows
// of the row operand and half of the column operand.
template <bool SPLIT, bool PAIR>
struct Stage {
  static constexpr int kParts = SPLIT ? 2 : 1;
  static constexpr int kWidest = SPLIT ? 128 : 256;                    // tile columns
  static constexpr int kWide = PAIR ? kWidest / 2 : kWidest;           // column operand here
  static constexpr int kBytes = kParts * (BM / 64 + kWide / 64) * kBox;  // 48, 32, 64 KB
  static constexpr int kCount = PAIR ? 6 : SPLIT ? 3 : 4;              // 192 KB
  static constexpr int kTurn = (kEpilogue / 32) * 4096;
  static constexpr int kSmem = kCount * kBytes + kTurn + 1024;
};

__device__ __forceinline__ float exp2i(int e) { return __int_as_float((127 + e) << 23); }

// Four float16 (8 bytes) to float, and to the pair hi + lo.
__device__ __forceinline__ float4 half4_float(uint2 u) {
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
  return make_float4(a.x, a.y, b.x, b.y);
}
template <bool LO>
__device__ __forceinline__ void put_half4(float4 v, __half* hi, __half* lo) {
  const __half2 h0 = __floats2half2_rn(v.x, v.y), h1 = __floats2half2_rn(v.z, v.w);
  uint2 u;
  u.x = *reinterpret_cast<const unsigned*>(&h0);
  u.y = *reinterpret_cast<const unsigned*>(&h1);
  *reinterpret_cast<uint2*>(hi) = u;
  if (LO) {
    const float2 f0 = __half22float2(h0), f1 = __half22float2(h1);
    const __half2 l0 = __floats2half2_rn(v.x - f0.x, v.y - f0.y);
    const __half2 l1 = __floats2half2_rn(v.z - f1.x, v.w - f1.y);
    u.x = *reinterpret_cast<const unsigned*>(&l0);
    u.y = *reinterpret_cast<const unsigned*>(&l1);
    *reinterpret_cast<uint2*>(lo) = u;
  }
}

// What the epilogue of a tile needs, gathered while its products run.  Every
// output is  v = p * sum + q * (e + f (d_i + d_j)),  q the stored value at the
// same place (O for the square, X for the last product, nothing for A), d the
// diagonals that apply, and the powers of two of the formats folded into p, e, f.
struct Out {
  int rows, cols, pitch;
  float p, e, f;
  const __half *q0, *q1;           // null: no such part
  const float *di, *dj;            // diagonals by row and by column, or null
  __half *o0, *o1;                 // null o0: the result itself
  float *diag;                     // where the diagonal goes (symmetric products)
  float ds, dp, dq;                // on it: dp * (sum * ds + d^2) + dq * d
};

template <bool SPLIT>
__device__ __forceinline__ void ns_out(const NsArgs& a, const Tile& t, Out* o) {
  const NsGroup& g = a.g[t.group];
  const NsStep& k = a.k[t.step];
  const long long b = t.mat - g.first;
  if (t.phase < 2) {
    const long long plane = b * g.s * g.pa;
    o->rows = o->cols = g.s;
    o->pitch = g.pa;
    o->di = o->dj = nullptr;
    o->q0 = o->q1 = nullptr;
    o->e = o->f = 0.f;
    if (t.phase == 0) {
      o->p = exp2i(k.ea - 2 * k.ex);
      o->o0 = g.a[0] + plane;
      o->o1 = SPLIT ? g.a[1] + plane : nullptr;
      o->diag = g.da + b * g.pa;
      o->ds = exp2i(-2 * k.ex);
      o->dp = 1.f;
      o->dq = 0.f;
    } else {
      o->p = k.c * exp2i(k.eb - 2 * k.ea);
      o->e = k.b * exp2i(k.eb - k.ea);
      o->f = k.c * exp2i(k.eb - k.ea);
      o->q0 = g.a[0] + plane;
      o->q1 = SPLIT ? g.a[1] + plane : nullptr;
      o->di = o->dj = g.da + b * g.pa;
      o->o0 = g.b[0] + plane;
      o->o1 = SPLIT ? g.b[1] + plane : nullptr;
      o->diag = g.db + b * g.pa;
      o->ds = exp2i(-2 * k.ea);
      o->dp = k.c;
      o->dq = k.b;
    }
  } else {
    const int from = t.step & 1;
    const long long plane = b * g.rows * g.px;
    const bool last = t.step + 1 == a.steps;
    const float up = last ? 1.f : exp2i(k.ex2);
    o->rows = g.rows;
    o->cols = g.cols;
    o->pitch = g.px;
    o->p = exp2i(-k.eb - k.ex) * up;
    o->f = exp2i(-k.ex) * up;
    o->e = k.a * o->f;
    o->q0 = g.x[from][0] + plane;
    o->q1 = g.x[from][1] + plane;
    o->di = g.tall ? nullptr : g.db + b * g.pa;
    o->dj = g.tall ? g.db + b * g.pa : nullptr;
    o->o0 = last ? nullptr : g.x[1 - from][0] + plane;
    o->o1 = g.x[1 - from][1] + plane;
    o->diag = nullptr;
  }
}

// A warp's 32 x 32 buffer, in units of four columns: unit q of row r lies at
// q ^ (r mod 8) ^ (r / 8).  Eight rows at one unit (turning in), a row's eight
// units (reading rows) and rows 0, 4, 8, ... at one column (reading columns)
// are in different banks.
__device__ __forceinline__ int turn_unit(int r, int q) { return r * 8 + (q ^ (r & 7) ^ (r >> 3)); }

// The last step's output: rows i + 4 it, four columns from j, as the result or
// into the weight.
template <typename T, int NB>
__device__ __forceinline__ void ns_result(const NsArgs& a, const Tile& t, const Out& o, int i,
                                          int j, int left, const float4 (&v)[NB]) {
  const NsMat& m = a.m[t.mat];
  T* w = reinterpret_cast<T*>(m.dst) + i * m.dst_row + j;
  const float step = m.step;
  const bool update = m.mom != nullptr;
  if (m.vec_dst) {  // whole vectors of four
    typedef typename RawOf<4 * sizeof(T)>::type V4;
    if (j >= o.cols) return;
    V4 old[NB];
    if (update) {
#pragma unroll
      for (int it = 0; it < NB; ++it)
        if (4 * it < left) old[it] = *reinterpret_cast<const V4*>(w + 4 * it * m.dst_row);
    }
#pragma unroll
    for (int it = 0; it < NB; ++it) {
      if (4 * it >= left) break;
      const float vs[4] = {v[it].x, v[it].y, v[it].z, v[it].w};
      V4 u;
      T* e4 = reinterpret_cast<T*>(&u);
      const T* o4 = reinterpret_cast<const T*>(&old[it]);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        e4[e] = St<T>::v(update ? fmaf(a.decay, Ld<T>::f(o4[e]), -step * vs[e]) : vs[e]);
      *reinterpret_cast<V4*>(w + 4 * it * m.dst_row) = u;
    }
  } else {
#pragma unroll
    for (int it = 0; it < NB; ++it) {
      if (4 * it >= left) break;
      T* x = w + 4 * it * m.dst_row;
      const float vs[4] = {v[it].x, v[it].y, v[it].z, v[it].w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (j + e < o.cols)
          x[e] = St<T>::v(update ? fmaf(a.decay, Ld<T>::f(x[e]), -step * vs[e]) : vs[e]);
    }
  }
}

// Epilogue of a 32 x 32 block of a tile, rows [i0, i0 + 32), columns
// [j0, j0 + 32).  `sums` of row i0 + lane are turned in shared memory so that
// eight lanes share a row's 64 bytes of float16, four columns to a lane.
template <bool SPLIT, typename T>
__device__ __forceinline__ void ns_emit(const NsArgs& a, const Tile& t, const Out& o, int i0,
                                        int j0, float4* turn, const float (&sums)[32]) {
  const bool sym = t.phase < 2;
  // warp-uniform: outside the matrix, or above the diagonal blocks
  if (i0 >= o.rows || j0 >= o.cols || (sym && j0 / BM > t.i0 / BM)) return;
  const int lane = threadIdx.x & 31, r0 = lane >> 3, q4 = lane & 7, j = j0 + 4 * q4;
  // Each loop below is a batch of independent accesses: a scheduler has two of
  // these warps, so latency is hidden inside a warp or not at all.  Split tiles
  // hold another 32 sums in registers meanwhile: half the rows at a time.
  constexpr int NB = SPLIT ? 4 : 8;
  const long long four = 4ll * o.pitch;
  const float row_d = o.di && i0 + lane < o.rows ? __ldcg(o.di + i0 + lane) : 0.f;
  float4 cd = make_float4(0.f, 0.f, 0.f, 0.f);
  if (o.dj) cd = __ldcg(reinterpret_cast<const float4*>(o.dj + j));  // inside the pitch of 64
#pragma unroll
  for (int q = 0; q < 8; ++q)
    turn[turn_unit(lane, q)] =
        make_float4(sums[4 * q], sums[4 * q + 1], sums[4 * q + 2], sums[4 * q + 3]);
  const bool mirror = sym && j0 / BM < t.i0 / BM;
  const float fd_row = o.f * row_d;
  cd.x = fmaf(o.f, cd.x, o.e);
  cd.y = fmaf(o.f, cd.y, o.e);
  cd.z = fmaf(o.f, cd.z, o.e);
  cd.w = fmaf(o.f, cd.w, o.e);
  __syncwarp();
  if (sym && i0 == j0) {  // the diagonal stays in float32, and zero in its place
    if (lane < o.rows - i0) {
      float* d = reinterpret_cast<float*>(turn) + 4 * turn_unit(lane, lane >> 2) + (lane & 3);
      o.diag[i0 + lane] = fmaf(o.dp, fmaf(*d, o.ds, row_d * row_d), o.dq * row_d);
      *d = 0.f;
    }
    __syncwarp();
  }
#pragma unroll 1
  for (int rb = r0; rb < 32; rb += 4 * NB) {
    const long long at0 = (long long)(i0 + rb) * o.pitch + j;
    const int left = o.rows - i0 - rb;  // rows rb + 4 it are inside for 4 it < left
    uint2 hi[NB], lo[NB];
#pragma unroll
    for (int it = 0; it < NB; ++it) hi[it] = lo[it] = make_uint2(0u, 0u);
    if (o.q0) {
      const __half* p = o.q0 + at0;
#pragma unroll
      for (int it = 0; it < NB; ++it, p += four)
        if (4 * it < left) hi[it] = __ldcg(reinterpret_cast<const uint2*>(p));
    }
    if (o.q1) {
      const __half* p = o.q1 + at0;
#pragma unroll
      for (int it = 0; it < NB; ++it, p += four)
        if (4 * it < left) lo[it] = __ldcg(reinterpret_cast<const uint2*>(p));
    }
    float4 v[NB];
#pragma unroll
    for (int it = 0; it < NB; ++it) v[it] = turn[turn_unit(rb + 4 * it, q4)];
    if (o.q0) {
#pragma unroll
      for (int it = 0; it < NB; ++it) {
        const float fd = __shfl_sync(0xffffffffu, fd_row, rb + 4 * it);
        float4 x = half4_float(hi[it]);
        if (SPLIT || !sym) {
          const float4 l = half4_float(lo[it]);
          x.x += l.x;
          x.y += l.y;
          x.z += l.z;
          x.w += l.w;
        }
        v[it].x = fmaf(x.x, cd.x + fd, v[it].x * o.p);
        v[it].y = fmaf(x.y, cd.y + fd, v[it].y * o.p);
        v[it].z = fmaf(x.z, cd.z + fd, v[it].z * o.p);
        v[it].w = fmaf(x.w, cd.w + fd, v[it].w * o.p);
      }
    } else {
#pragma unroll
      for (int it = 0; it < NB; ++it) {
        v[it].x *= o.p;
        v[it].y *= o.p;
        v[it].z *= o.p;
        v[it].w *= o.p;
      }
    }
    if (mirror) {
#pragma unroll
      for (int it = 0; it < NB; ++it) turn[turn_unit(rb + 4 * it, q4)] = v[it];
    }
    if (o.o0) {
      __half *p0 = o.o0 + at0, *p1 = o.o1 + at0;
#pragma unroll
      for (int it = 0; it < NB; ++it, p0 += four, p1 += four) {
        if (4 * it < left) {
          if (SPLIT || !sym) put_half4<true>(v[it], p0, p1);
          else put_half4<false>(v[it], p0, nullptr);
        }
      }
    } else {
      ns_result<T, NB>(a, t, o, i0 + rb, j, left, v);
    }
  }
  if (mirror) {  // the same values above the diagonal: four rows to a lane
    __syncwarp();
    const float* f = reinterpret_cast<const float*>(turn) + r0;
#pragma unroll 1
    for (int cb = 0; cb < 8; cb += NB) {
      // column 4 (cb + it) + r0: unit cb + it, place r0
      const long long to = (long long)(j0 + 4 * cb + r0) * o.pitch + i0 + 4 * q4;
      __half *p0 = o.o0 + to, *p1 = o.o1 + to;
      float4 v[NB];
#pragma unroll
      for (int it = 0; it < NB; ++it)
        v[it] = make_float4(
            f[4 * turn_unit(4 * q4, cb + it)], f[4 * turn_unit(4 * q4 + 1, cb + it)],
            f[4 * turn_unit(4 * q4 + 2, cb + it)], f[4 * turn_unit(4 * q4 + 3, cb + it)]);
#pragma unroll
      for (int it = 0; it < NB; ++it, p0 += four, p1 += four) {
        if (j0 + 4 * (cb + it) + r0 < o.cols) {
          if (SPLIT) put_half4<true>(v[it], p0, p1);
          else put_half4<false>(v[it], p0, nullptr);
        }
      }
    }
  }
  __syncwarp();  // the buffer is free for the next block
}

// A part of a split tile: its sums go to memory, and the block that finishes the
// last part adds all of them in their order (so the result does not depend on
// which block that is) and goes on with the tile.
__device__ __forceinline__ bool ns_join(const NsArgs& a, const Tile& t, int w, int h,
                                        float (&sums)[32], volatile int* joined) {
  const int lane = threadIdx.x & 31;
  // four columns of 32 rows are 512 contiguous bytes
  const long long at = (long long)(8 * h) * BM + 32 * w + lane;
  float4* const tile = reinterpret_cast<float4*>(a.parts) + (long long)t.region * (kPart / 4);
  float4* p = tile + t.part * (kPart / 4) + at;
#pragma unroll
  for (int q = 0; q < 8; ++q)
    __stcg(p + q * BM, make_float4(sums[4 * q], sums[4 * q + 1], sums[4 * q + 2], sums[4 * q + 3]));
  __threadfence();
  asm volatile("bar.sync 1, 256;\n" ::: "memory");
  if (threadIdx.x == 128) {
    const unsigned old = atomicAdd(a.joins + t.phase * kSplitTiles + t.slot, 1u);
    *joined = old % (unsigned)t.ks == (unsigned)t.ks - 1u;
    __threadfence();
  }
  asm volatile("bar.sync 1, 256;\n" ::: "memory");
  if (!*joined) return false;
#pragma unroll
  for (int c = 0; c < 32; ++c) sums[c] = 0.f;
  const float4* from = tile + at;
  for (int k = 0; k < t.ks; ++k, from += kPart / 4) {
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const float4 v = __ldcg(from + q * BM);
      sums[4 * q] += v.x;
      sums[4 * q + 1] += v.y;
      sums[4 * q + 2] += v.z;
      sums[4 * q + 3] += v.w;
    }
  }
  return true;
}

// Products of the current matrices.  Warp 0 copies operand tiles into shared
// memory (TMA), warp 1 issues the products (one thread), warps 4-11 read the
// accumulators (two, so that a tile's epilogue overlaps the next tile's
// products).
template <bool SPLIT, bool PAIR, typename T>
__global__ void __launch_bounds__(kThreads, 1) ns_product_kernel(const __grid_constant__ NsArgs a) {
  using St_ = Stage<SPLIT, PAIR>;
  constexpr int S = St_::kCount, PARTS = St_::kParts;
  extern __shared__ char smem_raw[];
  const unsigned smem0 = (smem_u32(smem_raw) + 1023u) & ~1023u;
  __shared__ unsigned long long full[6], empty[6], tm_full[2], tm_empty[2], sm_empty[2],
      drain;
  __shared__ unsigned tmem_base;
  __shared__ volatile int dead, joined;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tm_full[i], 1);
      mbar_init(&tm_empty[i], (kEpilogue / 32) * (PAIR ? 2 : 1));  // a warp each
      mbar_init(&sm_empty[i], (kEpilogue / 32) * (PAIR ? 2 : 1));
    }
    mbar_init(&drain, 1);
    dead = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    fence_async_smem();
  }
  if (warp == 2) {
    if constexpr (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(
                       smem_u32(&tmem_base))
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(
                       smem_u32(&tmem_base))
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n");
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
  __syncthreads();
  if constexpr (PAIR) cluster_sync();  // the other block's barriers are ready
  asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
  const unsigned tmem = tmem_base;
  const int rank = PAIR ? blockIdx.x & 1 : 0;

  if (warp == 0) {
    if (lane == 0) {
      Walk<PAIR> walk;
      Tile t;
      unsigned n = 0;  // stages issued
      bool ok = true;
      while (ok && walk.next(a, &t)) {
        const NsGroup& g = a.g[t.group];
        // what this tile reads: X of the last step, O, or offdiag(B)
        const int from = t.phase == 0 ? 2 : t.phase - 1;
        const int rounds = t.phase == 0 ? t.step : t.step + 1;
        const unsigned want =
            (unsigned)rounds * (t.phase == 0 ? g.tiles_app : g.tiles_sym) * (PAIR ? 2u : 1u);
        if (!wait_flag(a.done + from * kMats + t.mat, want, a)) break;
        asm volatile("fence.proxy.async.global;\n" ::: "memory");
        const int xi = MAP_X0 + (t.step & 1);
        const int mp = t.phase == 0 ? xi : t.phase == 1 ? MAP_A : g.tall ? xi : MAP_B;
        const int mq = t.phase == 0 ? xi : t.phase == 1 ? MAP_A : g.tall ? MAP_B : xi;
        const bool p_mn = t.phase == 0 && g.tall;
        const bool q_mn = t.phase == 0 ? g.tall : t.phase == 2 && !g.tall;
        const int z = t.mat - g.first, qw = t.bn / (PAIR ? 2 : 1), qb = qw / 64;
        const int jq = t.j0 + rank * qw;
        for (int kb = t.kb0; kb < t.kb1; ++kb, ++n) {
          const int s = n % S;
          if (n >= (unsigned)S && !wait_bar(&empty[s], (n / S - 1) & 1, a)) {
            ok = false;
            break;
          }
          // both blocks' copies count on the first block's barrier
          const unsigned bar = PAIR ? in_leader(smem_u32(&full[s])) : smem_u32(&full[s]);
          const unsigned base = smem0 + s * St_::kBytes;
          if (rank == 0)
            mbar_expect_tx(&full[s], (PAIR ? 2 : 1) * PARTS * (BM / 64 + qb) * kBox);
#pragma unroll
          for (int part = 0; part < PARTS; ++part) {
            const unsigned bp = base + part * (BM / 64) * kBox;
            const unsigned bq = base + (PARTS * (BM / 64) + part * (St_::kWide / 64)) * kBox;
            for (int i = 0; i < BM / 64; ++i)
              tma_box<PAIR>(bp + i * kBox, &g.map[mp][part], p_mn ? t.i0 + 64 * i : kb * BK,
                      p_mn ? kb * BK : t.i0 + 64 * i, z, bar);
            for (int i = 0; i < qb; ++i)
              tma_box<PAIR>(bq + i * kBox, &g.map[mq][part], q_mn ? jq + 64 * i : kb * BK,
                      q_mn ? kb * BK : jq + 64 * i, z, bar);
          }
        }
      }
      // copies still in flight land before the block ends
      for (unsigned i = n > (unsigned)S ? n - S : 0; rank == 0 && i < n; ++i)
        wait_bar(&full[i % S], (i / S) & 1, a);
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      Walk<PAIR> walk;
      Tile t;
      unsigned n = 0, tile = 0, sums = 0;
      bool ok = true;
      for (; ok && walk.next(a, &t); ++tile) {
        const NsGroup& g = a.g[t.group];
        const bool p_mn = t.phase == 0 && g.tall;
        const bool q_mn = t.phase == 0 ? g.tall : t.phase == 2 && !g.tall;
        // float32 accumulators, float16 operands, M = 128 (256 over a pair)
        const unsigned idesc = (1u << 4) | ((unsigned)p_mn << 15) | ((unsigned)q_mn << 16) |
                               ((unsigned)(t.bn / 8) << 17) | ((unsigned)((PAIR ? 2 : 1) * BM / 16) << 24);
        const int chunk = SPLIT ? kChunk : t.kb1 - t.kb0;
        const unsigned ps = (p_mn ? 2048u : 32u) >> 4, qs = (q_mn ? 2048u : 32u) >> 4;
        if (SPLIT && tile >= 2 && !wait_bar<PAIR>(&sm_empty[tile & 1], (tile / 2 - 1) & 1, a)) break;
        const unsigned dsmall = tmem + 256 + (tile & 1) * 128;
        for (int kb0 = t.kb0; ok && kb0 < t.kb1; kb0 += chunk, ++sums) {
          const int buf = sums & 1;
          if (sums >= 2 && !wait_bar<PAIR>(&tm_empty[buf], (sums / 2 - 1) & 1, a)) {
            ok = false;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
          const unsigned d = tmem + buf * (SPLIT ? 128 : 256);
          const int kb1 = min(t.kb1, kb0 + chunk);
          for (int kb = kb0; kb < kb1; ++kb, ++n) {
            const int s = n % S;
            if (!wait_bar<PAIR>(&full[s], (n / S) & 1, a)) {
              ok = false;
              break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
            const unsigned base = smem0 + s * St_::kBytes;
            const unsigned long long p0 = operand(base);
            const unsigned long long q0 = operand(base + PARTS * (BM / 64) * kBox);
            const unsigned long long p1 = p0 + ((BM / 64) * kBox >> 4);
            const unsigned long long q1 = q0 + ((St_::kWide / 64) * kBox >> 4);
#pragma unroll
            for (int k = 0; k < BK / 16; ++k) {
              const unsigned long long po = k * ps, qo = k * qs;
              if (SPLIT) {
                mma_f16<PAIR>(dsmall, p0 + po, q1 + qo, idesc, kb > t.kb0 || k > 0);
                mma_f16<PAIR>(dsmall, p1 + po, q0 + qo, idesc, true);
              }
              mma_f16<PAIR>(d, p0 + po, q0 + qo, idesc, kb > kb0 || k > 0);
            }
            mma_commit<PAIR>(&empty[s]);
          }
          mma_commit<PAIR>(&tm_full[buf]);
        }
      }
      // products still in flight end before tensor memory is given back
      mma_commit<PAIR>(&drain);
      wait_bar(&drain, 0, a);
    }
  } else if (warp >= 4) {
    Walk<PAIR> walk;
    Tile t;
    const int w = warp & 3, h = (warp - 4) >> 2;
    float4* const turn = reinterpret_cast<float4*>(smem_raw + (smem0 - smem_u32(smem_raw)) +
                                                 S * St_::kBytes + (warp - 4) * 4096);
    unsigned sums = 0;
    for (unsigned tile = 0; walk.next(a, &t); ++tile) {
      const int half = t.bn / 2;
      const unsigned lanes = (unsigned)(32 * w) << 16;
      // this warp's rows, columns t.j0 + h * half + [0, half)
      const int i = t.i0 + 32 * w, jh = t.j0 + h * half;
      Out out;
      ns_out<SPLIT>(a, t, &out);
      const int chunks = SPLIT ? (t.kb1 - t.kb0 + kChunk - 1) / kChunk : 1;
      __align__(16) float sum[SPLIT ? 2 : 1][32];
      bool ok = true;
      for (int ch = 0; ch < chunks; ++ch, ++sums) {
        const int buf = sums & 1;
        if (lane == 0) ok = ok && wait_bar(&tm_full[buf], (sums / 2) & 1, a);
        __syncwarp();
        if constexpr (SPLIT) {
          asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            if (q * 32 >= half) break;
            float v[32];
            tmem_load32(tmem + buf * 128 + h * half + q * 32 + lanes, v);
#pragma unroll
            for (int c = 0; c < 32; ++c) sum[q][c] = ch ? sum[q][c] + v[c] : v[c];
          }
          __syncwarp();
          asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
          if (lane == 0) arrive_leader<PAIR>(&tm_empty[buf]);
        }
      }
      if (!ok) dead = 1;
      asm volatile("bar.sync 1, 256;\n" ::: "memory");
      if (dead) break;
      // What this tile's epilogue loads was finished before the producer's wait
      // for it, and the chain of barriers from there to here orders it; the loads
      // bypass the first-level cache, which may hold an older step's lines.
      if constexpr (SPLIT) {
        // the small products of the whole tile are complete with its last chunk
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          if (q * 32 >= half) break;
          float v[32];
          tmem_load32(tmem + 256 + (tile & 1) * 128 + h * half + q * 32 + lanes, v);
#pragma unroll
          for (int c = 0; c < 32; ++c) sum[q][c] += v[c];
        }
        __syncwarp();
        asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
        if (lane == 0) arrive_leader<PAIR>(&sm_empty[tile & 1]);
        if (PAIR || t.ks == 1 || ns_join(a, t, w, h, sum[0], &joined)) {
#pragma unroll
          for (int q = 0; q < 2; ++q)
            if (q * 32 < half) ns_emit<SPLIT, T>(a, t, out, i, jh + q * 32, turn, sum[q]);
        } else {
          continue;
        }
      } else {
        const int buf = (sums - 1) & 1;
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        bool mine = true;
        for (int c0 = 0; c0 < half; c0 += 32) {
          tmem_load32(tmem + buf * 256 + h * half + c0 + lanes, sum[0]);
          if (c0 + 32 >= half) {
            __syncwarp();
            asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
            if (lane == 0) arrive_leader<PAIR>(&tm_empty[buf]);
          }
          mine = PAIR || t.ks == 1 || ns_join(a, t, w, h, sum[0], &joined);
          if (mine) ns_emit<SPLIT, T>(a, t, out, i, jh + c0, turn, sum[0]);
        }
        if (!mine) continue;
      }
      // other blocks read these values through TMA: order them before the count,
      // whose release covers the whole block's stores after the barrier
      asm volatile("fence.proxy.async.global;\n" ::: "memory");
      asm volatile("bar.sync 1, 256;\n" ::: "memory");
      if (threadIdx.x == 128) {
        asm volatile("red.release.gpu.global.add.u32 [%0], 1;\n" ::"l"(a.done + t.phase * kMats +
                                                                       t.mat)
                     : "memory");
      }
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
  __syncthreads();
  if constexpr (PAIR) {
    cluster_sync();  // neither block's memory is in use any more
    // The first block has issued its last commit, which arrives at the second
    // block's barriers too: that block stays until it has.
    if (rank == 1 && threadIdx.x == 32) wait_bar(&drain, 0, a);
  }
  if (warp == 2) {
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
    if constexpr (PAIR)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;\n" ::"r"(tmem));
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(tmem));
  }
}

// ---------------------------------------------------------------------------
// small matrices: one block each, one launch
// ---------------------------------------------------------------------------

// Up to 64 x 128 (or 128 x 64) a matrix and its products fit one block's shared
// memory in float32, and the 15 dependent products cost float32 FMAs and block
// barriers (2.5 us each at 64 x 64) in place of trips through memory:
// 64 x 64 bfloat16 42 us on the GPU against 77 with the three launches of the tiled
// kernel, 64 x 128 about 60 against 80.  At twice the longer side the products
// alone take as long as the tiled kernel.  A matrix's own shape decides, so that
// it is updated alike whatever else a list holds.
constexpr int kSmallS = 64, kSmallL = 128;
constexpr int kLdX = kSmallL + 4, kLdA = kSmallS + 4;  // 8 rows' vectors in 8 bank groups
constexpr int kSmallSmem = (int)sizeof(float) * (kSmallS * kLdX + 2 * kSmallS * kLdA);

// acc[u][v] = sum over k < n of P[ty + 16 u][k] P[tx + 16 v][k]
__device__ __forceinline__ void rows_product(const float* P, int ld, int n, int ty, int tx,
                                             float (&acc)[4][4]) {
#pragma unroll
  for (int u = 0; u < 4; ++u)
#pragma unroll
    for (int v = 0; v < 4; ++v) acc[u][v] = 0.f;
  for (int k = 0; k < n; k += 4) {
    float4 p[4], q[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      p[u] = *reinterpret_cast<const float4*>(P + (ty + 16 * u) * ld + k);
      q[u] = *reinterpret_cast<const float4*>(P + (tx + 16 * u) * ld + k);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        acc[u][v] = fmaf(p[u].x, q[v].x, acc[u][v]);
        acc[u][v] = fmaf(p[u].y, q[v].y, acc[u][v]);
        acc[u][v] = fmaf(p[u].z, q[v].z, acc[u][v]);
        acc[u][v] = fmaf(p[u].w, q[v].w, acc[u][v]);
      }
  }
}

template <typename T>
__global__ void __launch_bounds__(256) ns_small_kernel(const __grid_constant__ NsArgs a) {
  extern __shared__ char smem_raw[];
  float* const X = reinterpret_cast<float*>(smem_raw);  // [64][kLdX]: the shorter side in rows
  float* const A = X + kSmallS * kLdX;
  float* const B = A + kSmallS * kLdA;
  __shared__ double sm[32];
  const NsMat& m = a.m[blockIdx.x];
  const int cols = m.cols, tall = m.tall, s = m.s, l = m.l, n = s * l;
  for (int i = threadIdx.x; i < kSmallS * kLdX; i += 256) X[i] = 0.f;  // beyond s and l too
  __syncthreads();
  const T* src = reinterpret_cast<const T*>(m.src);
  double ss = 0;
  for (int i = threadIdx.x; i < n; i += 256) {
    const int r = i / cols, c = i - r * cols;
    float u = Ld<T>::f(src[r * m.src_row + c]);
    if (m.mom) {
      const float v = fmaf(a.mu, m.mom[i], u);
      m.mom[i] = v;
      u = a.nesterov ? fmaf(a.mu, v, u) : v;
    }
    ss += (double)u * u;
    X[tall ? c * kLdX + r : r * kLdX + c] = u;
  }
  ss = block_sum(ss, sm);
  const bool finite = ss <= 1.7e308;
  const double inv = ss > 0 ? 1.0 / sqrt(ss) : 0.0;
  int e;
  const float f = (float)frexp(inv, &e);
  const float e1 = ldexpf(1.f, e / 2), e2 = ldexpf(1.f, e - e / 2);
  __syncthreads();
  for (int i = threadIdx.x; i < s * l; i += 256) {
    const int r = i / l, at = r * kLdX + (i - r * l);
    X[at] = finite ? X[at] * e1 * e2 * f : __int_as_float(0x7fffffff);
  }
  __syncthreads();
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int s4 = (s + 3) & ~3, l4 = (l + 3) & ~3;
  for (int st = 0; st < a.steps; ++st) {
    const NsStep& k = a.k[st];
    float acc[4][4];
    rows_product(X, kLdX, l4, ty, tx, acc);
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int v = 0; v < 4; ++v) A[(ty + 16 * u) * kLdA + tx + 16 * v] = acc[u][v];
    __syncthreads();
    rows_product(A, kLdA, s4, ty, tx, acc);  // A is symmetric
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int at = (ty + 16 * u) * kLdA + tx + 16 * v;
        B[at] = fmaf(k.b, A[at], k.c * acc[u][v]);
      }
    __syncthreads();
    // rows ty + 16 u, columns 4 tx + 64 w + [0, 4)
    float4 y[2][4];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      if (64 * w >= l) break;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        y[w][u] = *reinterpret_cast<const float4*>(X + (ty + 16 * u) * kLdX + 4 * tx + 64 * w);
        y[w][u].x *= k.a;
        y[w][u].y *= k.a;
        y[w][u].z *= k.a;
        y[w][u].w *= k.a;
      }
      for (int q = 0; q < s4; q += 4) {
        float4 b4[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          b4[u] = *reinterpret_cast<const float4*>(B + (ty + 16 * u) * kLdA + q);
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const float4 x = *reinterpret_cast<const float4*>(X + (q + d) * kLdX + 4 * tx + 64 * w);
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float bv = d == 0 ? b4[u].x : d == 1 ? b4[u].y : d == 2 ? b4[u].z : b4[u].w;
            y[w][u].x = fmaf(bv, x.x, y[w][u].x);
            y[w][u].y = fmaf(bv, x.y, y[w][u].y);
            y[w][u].z = fmaf(bv, x.z, y[w][u].z);
            y[w][u].w = fmaf(bv, x.w, y[w][u].w);
          }
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      if (64 * w >= l) break;
#pragma unroll
      for (int u = 0; u < 4; ++u)
        *reinterpret_cast<float4*>(X + (ty + 16 * u) * kLdX + 4 * tx + 64 * w) = y[w][u];
    }
    __syncthreads();
  }
  T* dst = reinterpret_cast<T*>(m.dst);
  for (int i = threadIdx.x; i < n; i += 256) {
    const int r = i / cols, c = i - r * cols;
    const float v = X[tall ? c * kLdX + r : r * kLdX + c];
    T* w = dst + r * m.dst_row + c;
    *w = St<T>::v(m.mom ? fmaf(a.decay, Ld<T>::f(*w), -m.step * v) : v);
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

// [batch][rows][pitch] float16 with `cols` live columns; boxes of 64 x 64.
// Elements outside arrive as zeros.
static bool half_map(CUtensorMap* map, __half* p, int batch, int rows, int cols, int pitch) {
  return encode_map(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, p,
                    {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)batch},
                    {(cuuint64_t)pitch * 2, (cuuint64_t)pitch * 2 * rows}, {64, 64, 1});
}

static constexpr size_t kNsHead = sizeof(double) * kMats * kNormBlocks + 4 * (3 * kMats + 1 + 2 * kSplitTiles);

// Workspace of a list whose matrices fit a block each: none, but not null.
static constexpr size_t kNsNoWs = 256;

// Limit of the device-side waits of the launches to come.
static std::atomic<unsigned long long> g_wait_limit{kWaitLimitNs};

int ns_wait_limit(unsigned long long limit_ns) {
  if (limit_ns > kWaitLimitNs) return FA_E_ARG;
  g_wait_limit.store(limit_ns ? limit_ns : kWaitLimitNs);
  return FA_OK;
}

static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
static int pitch64(int n) { return (n + 63) / 64 * 64; }

// Workspace of one shape, and its pointers when `base` is given.
static size_t group_layout(NsGroup* g, bool split, char* base) {
  size_t off = 0;
  auto take = [&](size_t bytes) {
    char* p = base ? base + off : nullptr;
    off += up256(bytes);
    return p;
  };
  const size_t x = (size_t)2 * g->batch * g->rows * g->px, q = (size_t)2 * g->batch * g->s * g->pa;
  for (int i = 0; i < 2; ++i)
    for (int h = 0; h < 2; ++h) g->x[i][h] = reinterpret_cast<__half*>(take(x));
  for (int h = 0; h < (split ? 2 : 1); ++h) {
    g->a[h] = reinterpret_cast<__half*>(take(q));
    g->b[h] = reinterpret_cast<__half*>(take(q));
  }
  g->da = reinterpret_cast<float*>(take((size_t)4 * g->batch * g->pa));
  g->db = reinterpret_cast<float*>(take((size_t)4 * g->batch * g->pa));
  return off;
}

static void group_shape(NsGroup* g, int rows, int cols, int batch, int first) {
  g->rows = rows;
  g->cols = cols;
  g->s = std::min(rows, cols);
  g->l = std::max(rows, cols);
  g->tall = rows > cols;
  g->batch = batch;
  g->first = first;
  g->px = pitch64(cols);
  g->pa = pitch64(g->s);
}

// At least a matrix's part of its group_layout.
static size_t matrix_bytes(int rows, int cols, bool split) {
  const int s = std::min(rows, cols), pa = pitch64(s);
  return 4 * up256((size_t)2 * rows * pitch64(cols)) + (split ? 4 : 2) * up256((size_t)2 * s * pa) +
         2 * up256((size_t)4 * pa);
}

// The next matrices that share a launch sequence: at most kMats, of at most
// kGroups shapes, and of at most kMostBytes of workspace (but at least one).
// Members of one shape are numbered together.  Matrices that fit one block are
// passed over: they have launches of their own.
struct Batch {
  int n = 0, groups = 0;
  int member[kMats];               // call index of matrix i
  int group[kMats];                // its shape
  int rows[kGroups], cols[kGroups], count[kGroups], first[kGroups];
};

// A matrix needs 8 to 16 bytes an element of workspace, a hundred large ones
// more than the model they belong to.  A few gigabytes of matrices fill the
// machine: in sequences of 4, 2, 1 and 0.4 GB, 20 x 4096 x 4096 bfloat16 takes
// 31.1, 30.1, 29.7 and 29.9 ms; in 2.3, 1.1 and 0.6 GB, 60 x 1024 x 4096 takes
// 6.9, 7.4 and 7.9 ms.
constexpr size_t kMostBytes = (size_t)2 << 30;

static bool fits_block(const fa_matrix& m) {
  return std::min(m.rows, m.cols) <= kSmallS && std::max(m.rows, m.cols) <= kSmallL;
}

// False when none is left from *next on.
static bool take_batch(const fa_matrix* m, int* next, int count, bool split, Batch* o) {
  int raw_group[kMats], raw_member[kMats];
  int n = 0, i = *next;
  size_t bytes = 0;
  o->groups = 0;
  for (; n < kMats && i < count; ++i) {
    if (fits_block(m[i])) continue;
    bytes += matrix_bytes(m[i].rows, m[i].cols, split);
    if (n > 0 && bytes > kMostBytes) break;
    int g = 0;
    while (g < o->groups && (o->rows[g] != m[i].rows || o->cols[g] != m[i].cols)) ++g;
    if (g == o->groups) {
      if (g == kGroups) break;
      o->rows[g] = m[i].rows;
      o->cols[g] = m[i].cols;
      o->count[g] = 0;
      ++o->groups;
    }
    ++o->count[g];
    raw_member[n] = i;
    raw_group[n++] = g;
  }
  *next = i;
  int at[kGroups], sum = 0;
  for (int g = 0; g < o->groups; ++g) {
    o->first[g] = at[g] = sum;
    sum += o->count[g];
  }
  for (int k = 0; k < n; ++k) {
    const int to = at[raw_group[k]]++;
    o->member[to] = raw_member[k];
    o->group[to] = raw_group[k];
  }
  o->n = n;
  return n > 0;
}

static int tile_count(const NsGroup& g, bool sym, int bm, int bn) {
  return sym ? sym_tiles(g.s, bm, bn)
             : ((g.rows + bm - 1) / bm) * ((g.cols + bn - 1) / bn);
}

// Time of a tile on one multiprocessor in microseconds: us for each 64 columns
// of K, tail for the part of the epilogue that nothing hides.  Tile columns 64,
// 128, 256, and 256 with both blocks of a pair on one tile.  Measured on
// 4096 x 8192, 12 x 768 x 768 and 2048 x 2048 (bfloat16) and 2304 x 768
// (float32).  The products themselves take a third to a half of it: copying a
// tile's operands in and reading them out of shared memory take the rest, so
// what counts is bytes a tile.  float32 tiles hold their sums in registers and
// two accumulators, which leaves room for 128 columns; a pair gained nothing
// there (2048 x 2048: 794 against 781 us).  With pairs and without, bfloat16, in
// turn on one card: 4096 x 8192 2.70 and 2.99 ms, 4096 x 4096 1.61 and 1.76 ms,
// 5 x 2100 x 1500 0.66 and 0.77 ms, 20 x 1030 x 1100 1.04 and 0.98 ms.
struct TileTime { int bn; bool pair; double us, tail; };
static const TileTime kTimes[2][4] = {
    {{64, false, 0.41, 3.0}, {128, false, 0.50, 6.0}, {256, false, 0.69, 12.0}, {256, true, 0.47, 15.0}},
    {{64, false, 0.95, 3.5}, {128, false, 1.03, 6.5}, {0, false, 0, 0}, {0, true, 0, 0}}};

// Tile columns with the least time, and that time: waves of tiles times a
// tile's.  kb: 64-column blocks of K, over both products where sym.
static double pick_bn(const NsGroup& g, bool sym, bool split, bool pair, int units, int* bn) {
  double least = 1e300;
  const int kb = ((sym ? g.l + g.s : g.s) + BK - 1) / BK;
  for (const TileTime& c : kTimes[split]) {
    if (c.bn == 0 || c.pair != pair) continue;
    const long long tiles = (long long)g.batch * tile_count(g, sym, pair ? 2 * BM : BM, c.bn);
    const double t = (double)((tiles + units - 1) / units) * kb * c.us + (sym ? 2 : 1) * c.tail;
    if (t < least) {
      least = t;
      *bn = c.bn;
    }
  }
  return least;
}

size_t ns_ws_bytes(const fa_matrix* m, int count, int dtype) {
  size_t most = 0;
  Batch b;
  const size_t parts = sizeof(float) * kPart * kSplitUnits;
  for (int next = 0; take_batch(m, &next, count, dtype != FA_BF16, &b);) {
    size_t sum = 0;
    for (int g = 0; g < b.groups; ++g) {
      NsGroup gr{};
      group_shape(&gr, b.rows[g], b.cols[g], b.count[g], 0);
      sum += group_layout(&gr, dtype != FA_BF16, nullptr);
    }
    most = std::max(most, sum);
  }
  return most ? up256(kNsHead) + parts + most : kNsNoWs;
}

// The longer side keeps a tile, and so a wait for one, below 0.1 s.
bool ns_shape_ok(int rows, int cols) {
  return std::min(rows, cols) >= 1 && std::min(rows, cols) <= 32768 &&
         std::max(rows, cols) <= (1 << 22);
}

// Everything about a call that can be refused before the device is touched.
int ns_check(const fa_matrix* m, int count, int dtype, bool update) {
  if (!m || count <= 0) return FA_E_ARG;
  if (dtype != FA_F16 && dtype != FA_BF16 && dtype != FA_F32) return FA_E_DTYPE;
  for (int i = 0; i < count; ++i) {
    if (!m[i].src || !m[i].dst || (update && !m[i].momentum)) return FA_E_ARG;
    if (!ns_shape_ok(m[i].rows, m[i].cols)) return FA_E_SHAPE;
    if (m[i].src_row_stride < m[i].cols || m[i].dst_row_stride < m[i].cols) return FA_E_SHAPE;
  }
  return FA_OK;
}

// Exponents that keep the stored float16 values below 2^15: the largest
// singular value after each step follows from the polynomial on [0, the last
// bound], and every entry of X, A, B is at most the matrix's largest singular
// value.  False where the iteration may grow beyond what they can hold.
static bool plan_steps(NsStep* k, const double* coef, int steps) {
  double top = 1.0;
  auto exponent = [](double bound) { return 14 - (int)std::ceil(std::log2(std::max(bound, 1.0))); };
  for (int i = 0; i < steps; ++i) {
    const double a = coef[3 * i], b = coef[3 * i + 1], c = coef[3 * i + 2];
    if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return false;
    k[i].a = (float)a;
    k[i].b = (float)b;
    k[i].c = (float)c;
    const double edge = top * 1.02;
    double next = 0, inner = 0;
    for (int j = 0; j <= 2048; ++j) {
      const double s = edge * j / 2048, q = s * s * (b + c * s * s);
      inner = std::max(inner, std::fabs(q));
      next = std::max(next, std::fabs(s * (a + q)));
    }
    k[i].ex = exponent(edge);
    k[i].ea = exponent(edge * edge);
    k[i].eb = exponent(inner);
    k[i].ex2 = exponent(next * 1.02);
    if (!(next <= 128.0) || !(inner <= 8192.0)) return false;
    top = next;
  }
  return true;
}

// Tile shapes of a launch: single blocks or pairs for all of it, the faster by
// estimate.  Where the symmetric products have so few tiles that half of the
// multiprocessors would idle, their tiles take 64 columns and K is split as
// well, at most one part a multiprocessor and at least six blocks a part
// (joining the parts costs about 4 us: 64 x 5000 bfloat16 236 -> 138 us, but
// 512 x 512 with parts of three blocks 153 -> 169 us).
static void plan_tiles(NsArgs& a, bool split, int sms, int pairs) {
  constexpr int kLeast = 6;
  int few = 0;
  for (int i = 0; i < a.groups; ++i)
    few += a.g[i].batch * std::min(1 << 12, sym_tiles(a.g[i].s, BM, 64));
  const int units = std::min(sms, kSplitUnits);
  a.ks = few * 2 <= units ? std::min(units / few, kMaxParts) : 1;
  bool parts = false;
  for (int i = 0; i < a.groups; ++i)
    for (int p = 0; p < 2; ++p) {
      const int kb = ((p == 0 ? a.g[i].l : a.g[i].s) + BK - 1) / BK;
      a.g[i].ks[p] = std::max(1, std::min(a.ks, kb / kLeast));
      parts |= a.g[i].ks[p] > 1;
    }
  int bn[2][kGroups][2];
  double time[2] = {0, 0};
  for (int pair = 0; pair < (split ? 1 : 2); ++pair)
    for (int g = 0; g < a.groups; ++g)
      for (int sym = 0; sym < 2; ++sym)
        time[pair] += pick_bn(a.g[g], sym, split, pair, pair ? std::max(pairs, 1) : sms,
                              &bn[pair][g][sym]);
  a.pair = !split && !parts && pairs > 0 && time[1] < time[0];
  const int bm = a.pair ? 2 * BM : BM;
  a.tiles[0] = a.tiles[1] = a.tiles[2] = 0;
  int slot = 0;
  for (int i = 0; i < a.groups; ++i) {
    NsGroup& g = a.g[i];
    const bool in_parts = g.ks[0] > 1 || g.ks[1] > 1;
    g.bn_app = bn[a.pair][i][0];
    g.bn_sym = in_parts ? 64 : bn[a.pair][i][1];
    g.tiles_sym = tile_count(g, true, bm, g.bn_sym);
    g.tiles_app = tile_count(g, false, bm, g.bn_app);
    g.slot = slot;
    if (in_parts) slot += g.batch * g.tiles_sym;
    for (int p = 0; p < 2; ++p) a.tiles[p] += g.batch * g.tiles_sym * g.ks[p];
    a.tiles[2] += g.batch * g.tiles_app;
  }
}

// Pairs of blocks that are resident together, at most one block on a
// multiprocessor; asked once for each device.
template <typename T>
static int pairs_resident(int device) {
  constexpr int MAXD = 64;
  static std::atomic<int> known[MAXD];
  if (device < 0 && cudaGetDevice(&device) != cudaSuccess) return 0;
  if (device < MAXD && known[device].load() > 0) return known[device].load() - 1;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = 2;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)(sm_count(device) / 2 * 2));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Stage<false, true>::kSmem;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaFuncSetAttribute(ns_product_kernel<false, true, T>,
                           cudaFuncAttributeMaxDynamicSharedMemorySize,
                           Stage<false, true>::kSmem) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, ns_product_kernel<false, true, T>, &cfg) != cudaSuccess) {
    cudaGetLastError();
    n = 0;
  }
  if (device < MAXD) known[device].store(n + 1);
  return n;
}

template <bool SPLIT, bool PAIR, typename T>
static int ns_products(const NsArgs& a, int units, cudaStream_t st) {
  constexpr int smem = Stage<SPLIT, PAIR>::kSmem;
  FAB_TRY(cudaFuncSetAttribute(ns_product_kernel<SPLIT, PAIR, T>,
                               cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  // every block waits for other blocks' tiles: a cooperative launch makes them resident
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeCooperative;
  at[0].val.cooperative = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = 2;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)std::min(units, std::max(a.tiles[0], std::max(a.tiles[1], a.tiles[2]))) *
                     (PAIR ? 2u : 1u));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = PAIR ? 2 : 1;
  FAB_TRY(cudaLaunchKernelEx(&cfg, ns_product_kernel<SPLIT, PAIR, T>, a));
  return FA_OK;
}

template <typename T>
static int ns_run_small(const NsArgs& a, cudaStream_t st) {
  FAB_TRY(cudaFuncSetAttribute(ns_small_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               kSmallSmem));
  ns_small_kernel<T><<<a.mats, 256, kSmallSmem, st>>>(a);
  FAB_LAUNCH_CHECK();
  return FA_OK;
}

static void ns_fill(NsMat* o, const fa_matrix& f, int group, bool update, int dtype) {
  o->src = f.src;
  o->dst = f.dst;
  o->mom = update ? f.momentum : nullptr;
  o->src_row = f.src_row_stride;
  o->dst_row = f.dst_row_stride;
  o->step = (float)f.step;
  if (fits_block(f)) {
    o->cols = (short)f.cols;
    o->s = (short)std::min(f.rows, f.cols);
    o->l = (short)std::max(f.rows, f.cols);
    o->tall = f.rows > f.cols;
  }
  o->group = (unsigned char)group;
  const int item = dtype == FA_F32 ? 4 : 2;
  o->vec = f.cols % 8 == 0 && reinterpret_cast<uintptr_t>(f.src) % 16 == 0 &&
           (f.rows == 1 || f.src_row_stride * item % 16 == 0) &&
           (!o->mom || reinterpret_cast<uintptr_t>(o->mom) % 16 == 0);
  o->vec_dst = f.cols % 4 == 0 && reinterpret_cast<uintptr_t>(f.dst) % (4 * item) == 0 &&
               (f.rows == 1 || f.dst_row_stride % 4 == 0);
}

template <bool SPLIT, typename T>
static int ns_run(NsArgs& a, int device, cudaStream_t st) {
  const int sms = sm_count(device);
  long long most = 0;
  for (int g = 0; g < a.groups; ++g)
    most = std::max<long long>(most, (long long)a.g[g].rows * a.g[g].px);
  const int nb = (int)std::max<long long>(
      1, std::min<long long>(std::min<long long>(kNormBlocks, (most + 4095) / 4096),
                             std::max(1, sms * 8 / a.mats)));  // 8 warps of 512 columns
  ns_norm_kernel<T><<<dim3(nb, a.mats), 256, 0, st>>>(a);
  FAB_LAUNCH_CHECK();
  const int pb = (int)std::max<long long>(
      1, std::min<long long>((most + 4095) / 4096, std::max(1, sms * 8 / a.mats)));
  ns_pack_kernel<T><<<dim3(pb, a.mats), 256, 0, st>>>(a, nb);
  FAB_LAUNCH_CHECK();
  if constexpr (SPLIT) {
    plan_tiles(a, SPLIT, sms, 0);
  } else {
    const int pairs = pairs_resident<T>(device);
    plan_tiles(a, SPLIT, sms, pairs);
    if (a.pair) return ns_products<SPLIT, true, T>(a, pairs, st);
  }
  return ns_products<SPLIT, false, T>(a, sms, st);
}

// The matrices that fit one block, each.
static int ns_blocks(NsArgs& a, const fa_matrix* mats, int count, int dtype, bool update,
                     cudaStream_t st) {
  a.mats = 0;
  for (int i = 0; i < count; ++i) {
    if (fits_block(mats[i])) ns_fill(&a.m[a.mats++], mats[i], 0, update, dtype);
    if (a.mats == 0 || (a.mats < kMats && i + 1 < count)) continue;
    const int rc = dtype == FA_F16    ? ns_run_small<f16_t>(a, st)
                   : dtype == FA_BF16 ? ns_run_small<bf16_t>(a, st)
                                      : ns_run_small<float>(a, st);
    if (rc) return rc;
    a.mats = 0;
  }
  return FA_OK;
}

// The others.
static int ns_tiles(NsArgs& a, const fa_matrix* mats, int count, int dtype, bool update, char* ws,
                    int device, cudaStream_t st) {
  const bool split = dtype != FA_BF16;
  Batch bt;
  for (int next = 0; take_batch(mats, &next, count, split, &bt);) {
    size_t off = up256(kNsHead) + sizeof(float) * kPart * kSplitUnits;
    a.groups = bt.groups;
    a.mats = bt.n;
    for (int gi = 0; gi < bt.groups; ++gi) {
      NsGroup& g = a.g[gi];
      group_shape(&g, bt.rows[gi], bt.cols[gi], bt.count[gi], bt.first[gi]);
      off += group_layout(&g, split, ws + off);
      for (int h = 0; h < (split ? 2 : 1); ++h) {
        if (!half_map(&g.map[MAP_X0][h], g.x[0][h], g.batch, g.rows, g.cols, g.px) ||
            !half_map(&g.map[MAP_X1][h], g.x[1][h], g.batch, g.rows, g.cols, g.px) ||
            !half_map(&g.map[MAP_A][h], g.a[h], g.batch, g.s, g.s, g.pa) ||
            !half_map(&g.map[MAP_B][h], g.b[h], g.batch, g.s, g.s, g.pa))
          return FA_E_INTERNAL;
      }
    }
    for (int i = 0; i < bt.n; ++i) ns_fill(&a.m[i], mats[bt.member[i]], bt.group[i], update, dtype);
    const int rc = dtype == FA_F16    ? ns_run<true, f16_t>(a, device, st)
                   : dtype == FA_BF16 ? ns_run<false, bf16_t>(a, device, st)
                                      : ns_run<true, float>(a, device, st);
    if (rc) return rc;
  }
  return FA_OK;
}

int ns_impl(const fa_matrix* mats, int count, int dtype, const double* coef, int steps,
            bool update, double mu, int nesterov, double decay, void* ws, size_t ws_bytes,
            int device, cudaStream_t st) {
  if (!coef || !ws) return FA_E_ARG;
  if (steps < 1 || steps > kMaxSteps) return FA_E_SHAPE;
  NsArgs a;
  a.steps = steps;
  if (!plan_steps(a.k, coef, steps)) return FA_E_ARG;
  a.err = wait_error_word();
  if (!a.err) return FA_E_INTERNAL;
  a.limit_ns = g_wait_limit.load();
  a.mu = (float)mu;
  a.decay = (float)decay;
  a.nesterov = nesterov;
  const uintptr_t base = reinterpret_cast<uintptr_t>(ws);
  const size_t need = ns_ws_bytes(mats, count, dtype);
  if ((base & 255) || ws_bytes < need) return FA_E_ARG;
  bool small = false;
  for (int i = 0; i < count && !small; ++i) small = fits_block(mats[i]);
  a.part = reinterpret_cast<double*>(ws);
  a.done = reinterpret_cast<unsigned*>(a.part + kMats * kNormBlocks);
  a.failed = a.done + 3 * kMats;
  a.joins = a.failed + 1;
  a.parts = reinterpret_cast<float*>(static_cast<char*>(ws) + up256(kNsHead));
  // tiled matrices need a workspace: both kinds are in the list
  // Where a list holds both kinds, its one-block matrices run on a stream of their own
  // beside the tiled ones: 3 x 64 x 64 with 6 x 64 x 576 and 4 x 180 x 180, bfloat16,
  // take 105 us so, and 157 us one kind after the other.
  Side* side = need > kNsNoWs && small ? side_fork(device, st) : nullptr;
  int rc = ns_blocks(a, mats, count, dtype, update, side ? side->stream : st);
  if (!rc) rc = ns_tiles(a, mats, count, dtype, update, static_cast<char*>(ws), device, st);
  if (side) {
    const int joined = side_join(side, device, st);
    if (!rc) rc = joined;
  }
  return rc;
}

}  // namespace fab
