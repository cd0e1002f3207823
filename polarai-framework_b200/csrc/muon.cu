// One step of orthogonalised momentum over many matrices: the momentum's matrix U is brought close to the nearest one with orthonormal rows
// (or columns) by rounds of  X <- a X + b G X + c G^2 X,  G = X X^T (of the shorter side),  X = U / |U| at the beginning, and taken off the weights.
//
// Every round is three matrix products, G, P = a + b G + c G G and P X, on the tensor cores.  They hold their operands as PAIRS of
// fp16 numbers, hi + lo with 22 bits between them, and multiply hi hi + lo hi + hi lo with sums in fp32: three products at the fp16 rate,
// twice as fast as three of TF32 and as exact, which is possible because the range of all values is known.  No singular value of X passes
// kBound on the way, so that no entry of X, G or P leaves fp16 when they are held times the powers of two kX, kG and kP; what lo cannot
// hold below 2^-24 is small against the largest entries.  The pairs are written by the product before, so that a product needs no pass over its
// operands: TMA brings both planes of a tile in one box, and nothing but tcgen05.mma touches shared memory.
// G and P are symmetric: tiles below the diagonal are not computed, the epilogue of the others writes both halves.
//
// All matrices of a step take part in each launch: those of one shape lie behind one another and share a tensor map, and a launch's tiles
// are those of all shapes.
#include <cuda.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <exception>
#include <mutex>
#include <utility>
#include <vector>

#include "muon_plan.hpp"
#include "rows.cuh"
#include "tc_ptx.cuh"

namespace polar_b200 {
namespace {
using namespace tc;
using namespace muon;

constexpr float kBound = 1.4f, kBoundP = 3.98f;            // largest singular value of X, of P: 1.4^2 * 2^15 and 3.98 * 2^14 are below 65504

// ---- the passes before the products

struct Target {                                            // a matrix's weights, for the last product
  float* weights;
  float decay, scale;
};
struct Matrix {
  float* weights;
  const float* gradient;
  float* momentum;
  __half* x;                                               // hi plane; lo `plane` behind it
  uint64_t plane, count;
  uint32_t cols, pitch, chunk;                             // chunk: elements per CTA
  uint32_t first;                                          // its first chunk
  float decay, scale;
};
template <int N>
struct Table {
  uint32_t count;
  uint32_t chunks_before, matrices_before;                 // of tables launched before
  float momentum;
  int nesterov;
  double* partial;                                         // of each chunk: the sum of its squares
  Target* targets;
  int* failed;                                             // not zero: a wait of this step has given up (the last products leave the weights alone then)
  Matrix m[N];
};
constexpr int kFewMatrices = 16, kManyMatrices = 400;
static_assert(sizeof(Table<kManyMatrices>) <= 32764, "kernel parameters");
constexpr int kThreads = 256;
constexpr uint32_t kChunk = 4096, kMostChunks = 512;       // elements of a CTA, or more where a matrix has more than 512 times as many

template <int N>
__device__ __forceinline__ uint32_t matrix_of(const Table<N>& t, uint32_t chunk) {
  uint32_t lo = 0, end = t.count;
  while (end - lo > 1) {
    const uint32_t middle = (lo + end) / 2;
    if (t.m[middle].first <= chunk) lo = middle;
    else end = middle;
  }
  return lo;
}
__device__ __forceinline__ double block_sum(double v, double* slots) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) v += slots[i];
  return v;
}

// A stream (and the one below it): 64 matrices of 1024 x 1024 with 32 of 1024 x 4096 take 0.35 and 0.37 ms, 6.6 to 7 TB/s.
// m <- momentum * m + g, and the sum of the squares of u = g + momentum * m (nesterov) or m: in 64 bits, where no square of an fp32 number
// overflows or vanishes.
template <int N>
__global__ void __launch_bounds__(kThreads) momentum_kernel(const __grid_constant__ Table<N> t) {
  __shared__ double slots[kThreads / 32];
  pdl_enter();
  const uint32_t at = matrix_of(t, blockIdx.x);
  const Matrix& m = t.m[at];
  const uint32_t chunk = blockIdx.x - m.first;
  if (chunk == 0 && threadIdx.x == 0) t.targets[t.matrices_before + at] = Target{m.weights, m.decay, m.scale};
  if (t.chunks_before == 0 && blockIdx.x == 0 && threadIdx.x == 0) *t.failed = 0;
  const uint64_t from = (uint64_t)chunk * m.chunk, to = min(from + m.chunk, m.count);
  const bool vectors = ((reinterpret_cast<uintptr_t>(m.gradient) | reinterpret_cast<uintptr_t>(m.momentum)) & 15) == 0;
  double sum = 0;
  auto one = [&](float g, float& v) {
    v = fmaf(t.momentum, v, g);
    const float u = t.nesterov ? fmaf(t.momentum, v, g) : v;
    sum += (double)u * (double)u;
  };
  // (four loads on their way before the first store, past which none moves by itself, and none behind a branch: what lies behind the end reads the end)
  uint64_t i = from + threadIdx.x;
  if (vectors) {
    const uint64_t end = from + (to - from) / 4 * 4;
    for (uint64_t first = from + 4 * threadIdx.x; first < end; first += 16 * kThreads) {
      float4 g[4], v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint64_t at = min(first + 4 * kThreads * k, end - 4);
        g[k] = *reinterpret_cast<const float4*>(m.gradient + at), v[k] = *reinterpret_cast<const float4*>(m.momentum + at);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (first + 4 * kThreads * k >= end) break;
        one(g[k].x, v[k].x), one(g[k].y, v[k].y), one(g[k].z, v[k].z), one(g[k].w, v[k].w);
        *reinterpret_cast<float4*>(m.momentum + first + 4 * kThreads * k) = v[k];
      }
    }
    i = end + threadIdx.x;
  }
  for (; i < to; i += 4 * kThreads) {
    float g[4], v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) g[k] = m.gradient[min(i + kThreads * k, to - 1)], v[k] = m.momentum[min(i + kThreads * k, to - 1)];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (i + kThreads * k >= to) break;
      one(g[k], v[k]);
      m.momentum[i + kThreads * k] = v[k];
    }
  }
  sum = block_sum(sum, slots);
  if (threadIdx.x == 0) t.partial[t.chunks_before + blockIdx.x] = sum;
}

// A value times a power of two as a pair of fp16 numbers.
__device__ __forceinline__ void split(float v, __half* hi, __half* lo) {
  *hi = __float2half_rn(v);
  *lo = __float2half_rn(v - __half2float(*hi));
}

// X = u / |u| as pairs, zeros for a matrix of zeros.
template <int N>
__global__ void __launch_bounds__(kThreads) begin_kernel(const __grid_constant__ Table<N> t) {
  __shared__ double slots[kThreads / 32];
  pdl_enter();
  const uint32_t at = matrix_of(t, blockIdx.x);
  const Matrix& m = t.m[at];
  const uint32_t chunk = blockIdx.x - m.first, chunks = (uint32_t)((m.count + m.chunk - 1) / m.chunk);
  double sum = 0;
  for (uint32_t i = threadIdx.x; i < chunks; i += kThreads) sum += t.partial[t.chunks_before + m.first + i];
  sum = block_sum(sum, slots);
  const double by = sum == 0 ? 0 : (double)kX / sqrt(sum);
  const uint64_t from = (uint64_t)chunk * m.chunk, to = min(from + m.chunk, m.count);
  const bool vectors = ((reinterpret_cast<uintptr_t>(m.gradient) | reinterpret_cast<uintptr_t>(m.momentum)) & 15) == 0 && (m.cols & 3) == 0;
  auto value = [&](float g, float v) { return (float)((double)(t.nesterov ? fmaf(t.momentum, v, g) : v) * by); };
  // places in 32 bits from the chunk's first row on; loads before stores as above
  const uint64_t row0 = from / m.cols;
  const uint32_t in_row = (uint32_t)(from - row0 * m.cols), n = (uint32_t)(to - from);
  const float *const gradient = m.gradient + from, *const momentum = m.momentum + from;
  auto place = [&](uint32_t i) {
    const uint32_t row = (in_row + i) / m.cols;
    return m.x + (row0 + row) * m.pitch + (in_row + i - row * m.cols);
  };
  if (vectors) {                                           // (the chunk is vectors: whole rows are)
    for (uint32_t first = 4 * threadIdx.x; first < n; first += 8 * kThreads) {
      float4 g[2], v[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint32_t at = min(first + 4 * kThreads * k, n - 4);
        g[k] = *reinterpret_cast<const float4*>(gradient + at), v[k] = *reinterpret_cast<const float4*>(momentum + at);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (first + 4 * kThreads * k >= n) break;
        union { __half h[4]; uint2 bits; } hi, lo;
#pragma unroll
        for (int e = 0; e < 4; ++e) split(value((&g[k].x)[e], (&v[k].x)[e]), &hi.h[e], &lo.h[e]);
        __half* const x = place(first + 4 * kThreads * k);
        *reinterpret_cast<uint2*>(x) = hi.bits;
        *reinterpret_cast<uint2*>(x + m.plane) = lo.bits;
      }
    }
    return;
  }
  for (uint32_t first = threadIdx.x; first < n; first += 4 * kThreads) {
    float g[4], v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) g[k] = gradient[min(first + kThreads * k, n - 1)], v[k] = momentum[min(first + kThreads * k, n - 1)];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (first + kThreads * k >= n) break;
      __half* const x = place(first + kThreads * k);
      split(value(g[k], v[k]), x, x + m.plane);
    }
  }
}

// ---- the products

constexpr int BM = 128, BK = 32;
constexpr int kRun = 4;                                    // slabs that are summed in tensor memory
constexpr int kEpilogueWarps = 8, kProductThreads = 32 * (4 + kEpilogueWarps);
// Registers of a thread where tiles are 256 wide: 168 at launch (three warpgroups of 128 threads, 64512 in all), then what the sums need for the epilogue's two and
// what is left for the other: 2 * 128 * 232 + 128 * 40 = 64512.
constexpr int kFewRegisters = 40, kManyRegisters = 232, kSplitRegisters = 128 * kFewRegisters + 256 * kManyRegisters;
static_assert(kProductThreads == 384, "one warpgroup with few registers, two with many");
constexpr uint32_t kSlotBytes = 32 * 32 * 2 * 2;           // a block of 32 x 32 as pairs
template <int BN, bool SPLIT>
struct Cfg {
  static constexpr uint32_t kAPlane = BM * BK * 2, kBPlane = BN * BK * 2, kStageBytes = 2 * (kAPlane + kBPlane);   // both planes of both operands
  // (Tiles of 256 columns: a fourth stage, with one block in place of two, was 11.35 ms for 11.1 at 1024 columns and 8.44 for 8.7 at 4096 x 16384.)
  static constexpr int kStages = BN == 256 ? 3 : 5;
  static constexpr int kSlots = SPLIT ? 0 : 2;             // blocks on their way to memory, for each warp of the epilogue
  static constexpr uint32_t kWarpBytes = kSlots * kSlotBytes;
  static constexpr uint32_t kTileBytes = kStages * kStageBytes;
  // behind the slabs: those blocks; or what the other CTAs of a cluster, up to seven, send
  static constexpr uint32_t kTurnBytes = SPLIT ? BM * BN * 4 / 8 * 7 : kEpilogueWarps * kWarpBytes;
  static constexpr uint32_t kBytes = kTileBytes + kTurnBytes + 1024 + 256;
  static_assert(kBytes <= 227 * 1024, "shared memory");
};

enum Kind : int { kSymmetric, kRound, kUpdate };

struct Shape {                                             // the matrices of one shape, in one product
  CUtensorMap a, b, c;                                     // operands and result
  int kind;
  float by, add_by, diagonal;                              // result = by * sum + add_by * add + diagonal (on the diagonal)
  uint32_t m, n, k;
  uint32_t tiles_m, tiles_n, tiles;                        // tiles: of one matrix
  uint32_t first_tile;                                     // of the launch
  int a_mn, b_mn;                                          // operands whose rows are not contiguous along k
  __half* out;                                             // matrix z: planes 2 z (hi) and 2 z + 1 (lo)
  const __half* add;                                       // of the same layout; or nullptr
  uint64_t plane;
  uint32_t pitch;
  uint32_t first_target;
};
constexpr int kShapes = 16;
struct Product {
  uint32_t shapes, tiles, splits;
  float lr;
  const float* schedule;
  const Target* targets;
  int *status, *failed;
  unsigned long long wait_ns;
  Shape s[kShapes];
};
struct Place {
  uint32_t shape, z;
  int m0, n0;
};
// The launch's tile t, of 128 x BN.  A symmetric product has the tiles that reach above the diagonal, row by row; else 16 tile rows walk the columns
// together and share their operands in L2.
template <int BN>
__device__ __forceinline__ Place place_of(const Product& p, uint32_t t) {
  Place at;
  at.shape = 0;
  while (at.shape + 1 < p.shapes && p.s[at.shape + 1].first_tile <= t) ++at.shape;
  const Shape& s = p.s[at.shape];
  t -= s.first_tile;
  at.z = t / s.tiles;
  t -= at.z * s.tiles;
  if (s.kind == kSymmetric) {
    uint32_t i = 0, skip = 0;
    while (t >= s.tiles_n - skip) {
      t -= s.tiles_n - skip;
      skip = ++i * BM / BN;
    }
    at.m0 = (int)(i * BM);
    at.n0 = (int)((skip + t) * BN);
  } else {
    const uint32_t per = 16 * s.tiles_n, g = t / per, rows = min(s.tiles_m - g * 16, 16u), r = t - g * per;
    at.m0 = (int)((g * 16 + r % rows) * BM);
    at.n0 = (int)(r / rows * BN);
  }
  return at;
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst), "l"(map), "r"(bar),
      "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}
__device__ __forceinline__ void store_3d(const CUtensorMap* map, uint32_t src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map), "r"(src), "r"(x), "r"(y), "r"(z) : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
template <int GROUPS>
__device__ __forceinline__ void stores_read() {            // all but the last GROUPS stores have read their shared memory
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(GROUPS) : "memory");
}
__device__ __forceinline__ void stores_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

__device__ __forceinline__ void mma_f16(uint32_t d_tmem, Operand a, uint32_t a_units, Operand b, uint32_t b_units, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "mov.b64 da, {%1, %2};\n\t"
      "mov.b64 db, {%3, %4};\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n\t}" ::"r"(d_tmem),
      "r"(a.lo + a_units), "r"(a.hi), "r"(b.lo + b_units), "r"(b.hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
// fp32 sums of fp16 operands (format 0 of both), 128 x n.
__device__ __forceinline__ uint32_t f16_idesc(int n, int a_mn, int b_mn) {
  return (1u << 4) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
}
// Shared memory of this CTA to that of another one of its cluster, whose mbarrier (at the same place as `bar` here) counts the bytes.
__device__ __forceinline__ void send(uint32_t dst, uint32_t src, uint32_t bytes, uint32_t bar, uint32_t rank) {
  uint32_t there, count;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(dst), "r"(rank));
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(count) : "r"(bar), "r"(rank));
  asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(there), "r"(src), "r"(bytes), "r"(count) : "memory");
}
__device__ __forceinline__ Target target_of(const Product& p, const Shape& q, const Place& at) {
  return q.kind == kUpdate ? p.targets[q.first_target + at.z] : Target{};
}

// Both planes of 16 columns of what is added to a product.  Loaded ahead of use, since no load moves before a store by itself, and (as all loads here) not behind
// a branch of a lane's own, where each would be waited for: a row past the last one reads the last.
struct Beside {
  uint4 v[4];
};
__device__ __forceinline__ Beside beside16(const Shape& q, const Place& at, uint32_t row, uint32_t c0) {
  Beside b = {};
  if (!q.add || (row & ~31u) >= q.m || c0 >= q.n || (c0 | 31u) < (row & ~31u)) return b;   // (the same for all lanes)
  const uint4* const add = reinterpret_cast<const uint4*>(q.add + 2 * at.z * q.plane + (uint64_t)min(row, q.m - 1) * q.pitch + c0);
  b.v[0] = add[0], b.v[1] = add[1], b.v[2] = add[q.plane / 8], b.v[3] = add[q.plane / 8 + 1];
  return b;
}
// The result's 16 columns from c0 on of a row, from their sums: by * sum + add_by * add + diagonal.
__device__ __forceinline__ void complete(const Shape& q, uint32_t row, uint32_t c0, const Beside& beside, uint32_t* v) {
  if (q.add) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 x = __half22float2(reinterpret_cast<const __half2*>(beside.v)[j]), y = __half22float2(reinterpret_cast<const __half2*>(beside.v + 2)[j]);
      float a = fmaf(q.by, __uint_as_float(v[2 * j]), q.add_by * (x.x + y.x));
      float b = fmaf(q.by, __uint_as_float(v[2 * j + 1]), q.add_by * (x.y + y.y));
      if (c0 + 2 * j == row) a += q.diagonal;
      if (c0 + 2 * j + 1 == row) b += q.diagonal;
      v[2 * j] = __float_as_uint(a), v[2 * j + 1] = __float_as_uint(b);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = __float_as_uint(q.by * __uint_as_float(v[j]));
  }
}
// 16 neighbours as pairs, two of them to each word of `hi` and `lo`.
__device__ __forceinline__ void split16(const uint32_t* v, uint32_t* hi, uint32_t* lo) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float a = __uint_as_float(v[2 * j]), b = __uint_as_float(v[2 * j + 1]);
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
    hi[j] = *reinterpret_cast<const uint32_t*>(&h), lo[j] = *reinterpret_cast<const uint32_t*>(&l);
  }
}

// A block of 32 x 32 pairs in shared memory as TMA takes it: 64-byte rows in the 64-byte swizzle, hi, and lo behind it.  Where 8 columns of a row lie:
__device__ __forceinline__ uint32_t in_slot(uint32_t row, uint32_t eighth) { return row * 64 + (eighth ^ (row >> 1 & 3)) * 16; }
// The block turned over, 8 x 8 at a time.
__device__ __forceinline__ void turn_over(uint32_t from, uint32_t to, int lane) {
#pragma unroll
  for (uint32_t plane = 0; plane < kSlotBytes; plane += kSlotBytes / 2)
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {                     // eight rows; each eight lanes look at eight columns of them
      uint32_t r[4];
      asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                   : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                   : "r"(from + plane + in_slot(8 * i + (lane & 7), lane >> 3))
                   : "memory");
      asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(to + plane + in_slot(lane, i)), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3])
                   : "memory");
    }
}

// Writes 32 rows from r0 on (one to each lane) and COLS columns from c0 on, whose sums are in `v`; `beside` belongs to the first 16 of them.  Blocks of 32 x 32 go
// through two slots in shared memory of this warp's own by turns and leave them by TMA, for a symmetric product the mirror image too: with a lane's own stores,
// 32 rows of 32 bytes to an instruction, two matrices each of 301 x 514, 999 x 301 and 1511 x 777 took 393 us for 348.  Weights are turned over there, so that the warp reads and writes 32
// neighbours.  `stores`: how many have left so far.
template <int COLS>
__device__ __forceinline__ void finish(const Shape& q, const Place& at, const Target& target, const int* failed, float lr, uint32_t r0, uint32_t c0, int lane, uint32_t (&v)[COLS], Beside beside,
                                       uint8_t* slots, uint32_t& stores) {
  const uint32_t row = r0 + lane;
#pragma unroll
  for (int part = 0; part < COLS / 32; ++part) {           // blocks of 32 columns
    const uint32_t block = c0 + 32 * part;
    uint32_t* const x = v + 32 * part;
    if (block >= q.n || r0 >= q.m) return;
    if (q.kind == kUpdate) {
      const float keep = 1.f - lr * target.decay, rate = q.by * lr * target.scale;
      uint32_t* const turn = reinterpret_cast<uint32_t*>(slots);
      const bool live = block + lane < q.n;                // (a lane is a column here)
      float* const w = target.weights + (uint64_t)r0 * q.n + min(block + lane, q.n - 1);
      float old[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) old[i] = w[(uint64_t)min((uint32_t)i, q.m - 1 - r0) * q.n];
      const bool sound = *failed == 0;
      if (lane == 0) stores_read<0>();
      __syncwarp();
#pragma unroll
      for (int j = 0; j < 32; ++j) turn[lane * 32 + (j ^ lane)] = x[j];
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (live && sound && r0 + i < q.m) w[(uint64_t)i * q.n] = old[i] * keep - rate * __uint_as_float(turn[i * 32 + (lane ^ i)]);
      __syncwarp();
      continue;
    }
    const bool below = q.kind == kSymmetric && block < r0; // written by the block above the diagonal
    uint8_t* const slot = slots + (stores & 1) * kSlotBytes;
    if (lane == 0) stores_read<1>();
    __syncwarp();
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const Beside now = beside;
      if (32 * part + 16 * half + 16 < COLS) beside = beside16(q, at, row, block + 16 * half + 16);
      if (below) continue;
      uint32_t hi[8], lo[8];                               // two columns to a word
      complete(q, row, block + 16 * half, now, x + 16 * half);
      split16(x + 16 * half, hi, lo);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint8_t* const at16 = slot + in_slot(lane, 2 * half + j);
        *reinterpret_cast<uint4*>(at16) = make_uint4(hi[4 * j], hi[4 * j + 1], hi[4 * j + 2], hi[4 * j + 3]);
        *reinterpret_cast<uint4*>(at16 + kSlotBytes / 2) = make_uint4(lo[4 * j], lo[4 * j + 1], lo[4 * j + 2], lo[4 * j + 3]);
      }
    }
    if (below) continue;
    fence_async_smem();
    __syncwarp();
    if (lane == 0) store_3d(&q.c, smem_u32(slot), (int)block, (int)r0, (int)(2 * at.z));
    ++stores;
    if (q.kind == kSymmetric && block > r0) {
      uint8_t* const other = slots + (stores & 1) * kSlotBytes;
      if (lane == 0) stores_read<1>();
      __syncwarp();
      turn_over(smem_u32(slot), smem_u32(other), lane);
      fence_async_smem();
      __syncwarp();
      if (lane == 0) store_3d(&q.c, smem_u32(other), (int)r0, (int)block, (int)(2 * at.z));
      ++stores;
    }
  }
}
// 16 columns of a row, of which the CTAs of a cluster that shares a tile have few: straight to memory.
__device__ __forceinline__ void finish16(const Shape& q, const Place& at, const Target& target, const int* failed, float lr, uint32_t r0, uint32_t c0, int lane, uint32_t (&v)[16],
                                         const Beside& beside) {
  const uint32_t row = r0 + lane, block = c0 & ~31u;
  if (c0 >= q.n || r0 >= q.m) return;
  if (q.kind == kSymmetric && block < r0) return;
  if (q.kind == kUpdate) {
    const float keep = 1.f - lr * target.decay, rate = q.by * lr * target.scale;
    float* const w = target.weights + (uint64_t)min(row, q.m - 1) * q.n + c0;
    const bool sound = *failed == 0;
    float x[16];                                           // (all loads before the first store, which might change what they read)
    if ((q.n & 3) == 0 && (reinterpret_cast<uintptr_t>(target.weights) & 15) == 0 && c0 + 16 <= q.n) {
#pragma unroll
      for (int j = 0; j < 4; ++j) *reinterpret_cast<float4*>(x + 4 * j) = reinterpret_cast<const float4*>(w)[j];
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = x[j] * keep - rate * __uint_as_float(v[j]);
      if (row >= q.m || !sound) return;
#pragma unroll
      for (int j = 0; j < 4; ++j) reinterpret_cast<float4*>(w)[j] = *reinterpret_cast<const float4*>(x + 4 * j);
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = w[min((uint32_t)j, q.n - 1 - c0)];
      if (row >= q.m || !sound) return;
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (c0 + j < q.n) w[j] = x[j] * keep - rate * __uint_as_float(v[j]);
    }
    return;
  }
  __half* const matrix = q.out + 2 * at.z * q.plane;
  uint32_t hi[8], lo[8];
  complete(q, row, c0, beside, v);
  split16(v, hi, lo);
  if (row < q.m) {                                         // (columns behind the last one lie in the row's padding)
    float* const out = reinterpret_cast<float*>(matrix + (uint64_t)row * q.pitch + c0);
    st_global_v8(out, hi);
    st_global_v8(out + q.plane / 2, lo);
  }
  if (q.kind == kSymmetric && block > r0) {                // its mirror image: a column of the block is a row there, 32 lanes side by side
    unsigned short* const mirror = reinterpret_cast<unsigned short*>(matrix) + (uint64_t)c0 * q.pitch + row;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      if (c0 + j < q.n) {
        mirror[(uint64_t)j * q.pitch] = (unsigned short)(hi[j / 2] >> (j & 1) * 16);
        mirror[(uint64_t)j * q.pitch + q.plane] = (unsigned short)(lo[j / 2] >> (j & 1) * 16);
      }
    }
  }
}

// One CTA per SM walks tiles of 128 x BN; or, SPLIT, where there are too few tiles to go round, a cluster of up to eight CTAs has one, each CTA a share of its
// slabs, and they send one another their sums, each for a part of the tile (784 x 4096 and 4096 x 10: 590 us without clusters, 266 with sums pulled by loads,
// 256 with sums sent by bulk copies).  Large products are bound by the power limit: 4096 x 16384, five rounds, 8.7 to 8.9 ms, 1120 to 1150 TFLOP/s of fp16 products, the tensor
// pipe at 72 to 81 % of its cycles; those of a few hundred columns by what stands around them, 7.5 us of 9.5.  (Pairs of CTAs on tiles of 256 x 256, which fetch a third less, were slower:
// 4096 x 16384 10.2 ms for 8.5.  A slab of 128 x 256 x 32 takes 0.58 us, which is what the library's largest products of this type take.)
//   warp 0     TMA: both planes of a slab of 32 k of each operand, one instruction each.  An operand that is contiguous along k is K-major
//              (rows of 64 bytes in the 64-byte swizzle), else MN-major (chunks of 64 columns, 128-byte swizzle, a row per k).
//   warp 1     tcgen05.mma: per 16 k  hi hi, lo hi, hi lo, into two accumulators in tensor memory by turns, each for kRun slabs.
//   warps 4-11 add the finished accumulators to the tile's sums in registers, two warps to each 32 rows and half of the columns each, and
//              write the tile, while the next one's products run.
// The tensor core cuts every sum off at fp32's last bit, towards zero: over the 3 k / 16 additions of a long k that makes the sums too small by
// more than all else does to them (784 x 4096: the update 6.4e-5 from the exact one).  The registers' sums are rounded to nearest, and with runs
// of 128 k there are 24 additions to a cut sum (784 x 4096: 7.7e-6); reading the accumulators costs the tensor core nothing.
// Every wait is bounded; when one gives up, all roles leave, the status word holds its code (7xx), and the step's last products, whose operands
// then mean nothing, leave the weights alone.
template <int BN, bool SPLIT>
__global__ void __launch_bounds__(kProductThreads, 1) product_kernel(const __grid_constant__ Product p) {
  using C = Cfg<BN, SPLIT>;
  constexpr int S = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t bar_base = smem_base + C::kTileBytes + C::kTurnBytes;
  auto full = [&](int s) { return bar_base + 8u * s; };
  auto empty = [&](int s) { return bar_base + 8u * (S + s); };
  auto acc_full = [&](int a) { return bar_base + 8u * (2 * S + a); };
  auto acc_empty = [&](int a) { return bar_base + 8u * (2 * S + 2 + a); };
  const uint32_t received = bar_base + 8u * (2 * S + 4);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem_gen + C::kTileBytes + C::kTurnBytes + 8 * (2 * S + 5));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = uniform_warp();
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) mbar_init(full(s), 1), mbar_init(empty(s), 1);
    for (int a = 0; a < 2; ++a) mbar_init(acc_full(a), 1), mbar_init(acc_empty(a), kEpilogueWarps);
    if (SPLIT) {
      mbar_init(received, 1);
      mbar_expect_tx(received, BM * BN * 4 / p.splits * (p.splits - 1));
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0 && elect_one()) {                          // (the maps are parameters: they may be fetched before the kernel before has finished)
    const Shape& q = p.s[place_of<BN>(p, SPLIT ? blockIdx.x / p.splits : blockIdx.x).shape];
    prefetch_map(&q.a);
    prefetch_map(&q.b);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), 2 * BN);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  if (SPLIT) cluster_arrive();                             // (nothing is sent before the receiver's barrier is there)
  pdl_enter();
  if (SPLIT) cluster_wait();
  const uint32_t rank = SPLIT ? cluster_rank() : 0, splits = SPLIT ? p.splits : 1;
  const uint32_t first = SPLIT ? blockIdx.x / splits : blockIdx.x, step = SPLIT ? p.tiles : gridDim.x;
  auto slabs_of = [&](const Shape& q, int* end) {          // the CTA's
    const int slabs = (int)((q.k + BK - 1) / BK);
    if (!SPLIT) {
      *end = slabs;
      return 0;
    }
    const int each = (slabs + (int)splits - 1) / (int)splits;
    *end = min(slabs, (int)(rank + 1) * each);
    return min(slabs, (int)rank * each);
  };
  const float lr = p.schedule ? p.schedule[1] : p.lr;

  if (warp >= 4) {
    if constexpr (BN == 256) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kManyRegisters));
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    uint8_t* const place = smem_gen + C::kTileBytes + (warp - 4) * C::kWarpBytes;
    uint32_t run = 0, stores = 0;
    bool ok = true;
    for (uint32_t t = first; ok && t < p.tiles; t += step) {
      const Place at = place_of<BN>(p, t);
      const Shape& q = p.s[at.shape];
      const uint32_t r0 = (uint32_t)at.m0 + quarter * 32, c0 = (uint32_t)at.n0 + half * (BN / 2);
      uint32_t sum[BN / 2];                              // this thread's row of its half of the tile, as bits of floats
      int end;
      const int begin = slabs_of(q, &end), runs = (end - begin + kRun - 1) / kRun;
      Beside beside = {};
      if (!SPLIT && q.kind == kUpdate) {                   // the weights come to L2 meanwhile
        const Target target = target_of(p, q, at);
        const uint32_t row = min(r0 + lane, q.m - 1);
        for (uint32_t c = c0; c < min(c0 + BN / 2, q.n); c += 32)
          asm volatile("prefetch.global.L2 [%0];" ::"l"(target.weights + (uint64_t)row * q.n + c));
      }
      if (SPLIT && runs == 0) {
#pragma unroll
        for (int e = 0; e < BN / 2; ++e) sum[e] = 0;
      }
      for (int i = 0; i < runs; ++i, ++run) {
        const uint32_t as = run & 1u;
        if (!SPLIT && i + 1 == runs) beside = beside16(q, at, r0 + lane, c0);
        ok = mbar_wait(acc_full(as), (run >> 1) & 1u, abort_flag, p.status, 704, p.wait_ns);
        if (!ok) break;
        tc_fence_after();
        const uint32_t acc = tmem_base + as * BN + half * (BN / 2) + ((uint32_t)(quarter * 32) << 16);
        if (i == 0) {
#pragma unroll
          for (int j = 0; j < BN / 2; j += 32) tmem_ld_32x32(acc + j, sum + j);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int j = 0; j < BN / 2; j += 16) {
            uint32_t v[16];
            tmem_ld_32x16(acc + j, v);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) sum[j + e] = __float_as_uint(__uint_as_float(sum[j + e]) + __uint_as_float(v[e]));
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(acc_empty(as));
      }
      if (!SPLIT && !ok) break;                            // (SPLIT: all eight warps meet below, whatever has given up; there is one tile)
      if constexpr (SPLIT) {
        // Each CTA completes its share of the columns: the sums of the others' go to them, theirs come here.
        // (The slabs have been read: the last product has been waited for.)
        const uint32_t cols = BN / splits, share = cols * BM * 4;
        uint4* const mine = reinterpret_cast<uint4*>(smem_gen);   // four neighbours of a row to a place, rows side by side
#pragma unroll
        for (int j = 0; j < BN / 8; ++j)
          mine[(half * (BN / 8) + j) * BM + quarter * 32 + lane] = make_uint4(sum[4 * j], sum[4 * j + 1], sum[4 * j + 2], sum[4 * j + 3]);
        fence_async_smem();
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpilogueWarps) : "memory");
        if (ok && warp == 4 && lane < (int)splits && lane != (int)rank)
          send(smem_base + C::kTileBytes + (rank - (rank > (uint32_t)lane)) * share, smem_base + lane * share, share, received, lane);
        const Target target = target_of(p, q, at);
        const float4* const sent = reinterpret_cast<const float4*>(smem_gen + C::kTileBytes);
        // pieces of 32 rows and 16 columns
        for (uint32_t piece = warp - 4; ok && piece < cols / 4; piece += kEpilogueWarps) {
          const uint32_t rows = piece & 3, c = piece / 4 * 16, from = c / 4 * BM + rows * 32 + lane;
          const Beside now = beside16(q, at, (uint32_t)at.m0 + rows * 32 + lane, (uint32_t)at.n0 + rank * cols + c);
          ok = mbar_wait(received, 0, abort_flag, p.status, 705, p.wait_ns);
          if (!ok) break;
          float v[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] = 0.f;
          for (uint32_t r = 0; r < splits; ++r) {
            const float4* const x = r == rank ? reinterpret_cast<const float4*>(mine) + rank * (share / 16) : sent + (r - (r > rank)) * (share / 16);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float4 y = x[from + j * BM];
              v[4 * j] += y.x, v[4 * j + 1] += y.y, v[4 * j + 2] += y.z, v[4 * j + 3] += y.w;
            }
          }
          uint32_t bits[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) bits[j] = __float_as_uint(v[j]);
          finish16(q, at, target, p.failed, lr, (uint32_t)at.m0 + rows * 32, (uint32_t)at.n0 + rank * cols + c, lane, bits, now);
        }
      } else {
        finish<BN / 2>(q, at, target_of(p, q, at), p.failed, lr, r0, c0, lane, sum, beside, place, stores);
        __syncwarp();
      }
    }
    if (!SPLIT && lane == 0) stores_done();
  } else {
    if constexpr (BN == 256) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegisters));
    if (warp == 0) {
      const bool leader = elect_one();
      int s = 0;
      uint32_t ph = 1;
      bool ok = true;
      for (uint32_t t = first; ok && t < p.tiles; t += step) {
        const Place at = place_of<BN>(p, t);
        const Shape& q = p.s[at.shape];
        const int plane = (int)(2 * at.z);
        int end;
        for (int kb = slabs_of(q, &end); kb < end; ++kb) {
          if (!mbar_wait(empty(s), ph, abort_flag, p.status, 701, p.wait_ns)) { ok = false; break; }
          if (leader) {
            const uint32_t stage = smem_base + s * C::kStageBytes;
            mbar_expect_tx(full(s), C::kStageBytes);
            if (q.a_mn) tma_load_4d(stage, &q.a, full(s), 0, kb * BK, at.m0 / 64, plane);
            else tma_load_3d(stage, &q.a, full(s), kb * BK, at.m0, plane);
            if (q.b_mn) tma_load_4d(stage + 2 * C::kAPlane, &q.b, full(s), 0, kb * BK, at.n0 / 64, plane);
            else tma_load_3d(stage + 2 * C::kAPlane, &q.b, full(s), kb * BK, at.n0, plane);
          }
          if (++s == S) s = 0, ph ^= 1;
        }
      }
    } else if (warp == 1) {
      const bool leader = elect_one();
      int s = 0;
      uint32_t ph = 0, run = 0;
      bool ok = true;
      for (uint32_t t = first; ok && t < p.tiles; t += step) {
        const Place at = place_of<BN>(p, t);
        const Shape& q = p.s[at.shape];
        // where the left half of a symmetric product's tile lies below the diagonal, the right half alone: 128 rows or two chunks further
        const uint32_t left_out = BN == 256 && q.kind == kSymmetric && at.m0 == at.n0 + 128 ? 128 : 0;
        const uint32_t idesc = f16_idesc(BN - left_out, q.a_mn, q.b_mn);
        // K-major: 64-byte swizzle (layout 4), groups of 8 rows 512 bytes apart, 16 k 32 bytes on.  MN-major: 128-byte swizzle (layout 2), chunks
        // of 64 columns BK rows apart, groups of 8 k 1024 bytes, 16 k 2048 bytes on.
        const Operand a_op = q.a_mn ? make_desc(0, BK * 128, 1024, 2) : make_desc(0, 16, 512, 4);
        const Operand b_op = q.b_mn ? make_desc(0, BK * 128, 1024, 2) : make_desc(0, 16, 512, 4);
        const uint32_t a_step = (q.a_mn ? 2048u : 32u) >> 4, b_step = (q.b_mn ? 2048u : 32u) >> 4;
        int slabs;
        for (int kb = slabs_of(q, &slabs); kb < slabs; ++run) {
          const uint32_t as = run & 1u, acc = tmem_base + as * BN + left_out;
          ok = mbar_wait(acc_empty(as), ((run >> 1) & 1u) ^ 1u, abort_flag, p.status, 702, p.wait_ns);
          if (!ok) break;
          tc_fence_after();
          const int end = min(kb + kRun, slabs);           // of the run
          for (uint32_t more = 0; kb < end; ++kb, more = 1) {
            ok = mbar_wait(full(s), ph, abort_flag, p.status, 703, p.wait_ns);
            if (!ok) break;
            tc_fence_after();
            const uint32_t a_hi = ((smem_base & 0x3FFFFu) + s * C::kStageBytes) >> 4, a_lo = a_hi + (C::kAPlane >> 4);
            const uint32_t b_hi = a_lo + (C::kAPlane >> 4) + left_out * (BK * 2) / 16, b_lo = b_hi + (C::kBPlane >> 4);
            if (leader) {
#pragma unroll
              for (int kk = 0; kk < BK / 16; ++kk) {
                mma_f16(acc, a_op, a_hi + kk * a_step, b_op, b_hi + kk * b_step, idesc, kk ? 1u : more);
                mma_f16(acc, a_op, a_lo + kk * a_step, b_op, b_hi + kk * b_step, idesc, 1u);
                mma_f16(acc, a_op, a_hi + kk * a_step, b_op, b_lo + kk * b_step, idesc, 1u);
              }
              tc_commit(empty(s));
            }
            if (++s == S) s = 0, ph ^= 1;
          }
          if (!ok) break;
          if (leader) tc_commit(acc_full(as));
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    if (threadIdx.x == 0) *p.failed = 1;
    // let copies and products in flight finish before the memory that they use goes away
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000ll) { }
    __syncthreads();
  }
  if constexpr (SPLIT) {
    // no CTA leaves before all have what it has sent; nothing that was written has to be seen by then (with a release, which waits for the stores, 1 us more)
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    cluster_wait();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 2 * BN);
  }
}

// ---- small matrices: a whole step by one CTA for each

// Its X lies in shared memory as pairs all the while, the shorter side's rows behind one another: 64 or 128 rows, in chunks of 64 columns and the 128-byte
// swizzle, which is a K-major operand for X X^T and an MN-major one for P X.  Tall matrices are turned over on the way in and out.  The products are 0.2
// to 0.8 us each; what stands between them - the sums out of tensor memory, the pairs into shared memory, a barrier - is as much: 36 matrices up to
// 64 x 128 take 27 us, where the products' launches took 118.
struct Small {
  float* weights;
  const float* gradient;
  float* momentum;
  uint32_t rows, cols;
  float decay, scale;
};
template <int N>
struct SmallTable {
  float lr, momentum, a, b, c;
  int nesterov;
  uint32_t steps;
  const float* schedule;
  int* status;
  unsigned long long wait_ns;
  Small m[N];
};
constexpr int kFewSmall = 64, kManySmall = 800;
static_assert(sizeof(SmallTable<kManySmall>) <= 32764, "kernel parameters");
constexpr int kSmallThreads = 512, kSmallEach = 64;        // elements of a thread at most
constexpr uint32_t kSmallX = 128 * 1024, kSmallP = 64 * 1024;
// (an operand of 128 rows may reach 64 rows past the end of what lies there: those rows of the result are not read)
constexpr uint32_t kSmallBytes = kSmallX + kSmallP + 16 * 1024 + 1024 + 256;
__host__ __device__ constexpr bool is_small(uint64_t rows, uint64_t cols) {
  const uint64_t side = rows < cols ? rows : cols, other = rows < cols ? cols : rows;
  return (side <= 128 && other <= 256) || (side <= 64 && other <= 512);
}

template <int N>
__global__ void __launch_bounds__(kSmallThreads, 1) small_kernel(const __grid_constant__ SmallTable<N> t) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ double slots[kSmallThreads / 32];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const smem = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t bar = smem_base + kSmallBytes - 1024 - 256;
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(smem + kSmallBytes - 1024 - 256 + 8);
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = uniform_warp(), lane = threadIdx.x & 31;
  const Small& m = t.m[blockIdx.x];
  const bool tall = m.rows > m.cols;
  const uint32_t side = tall ? m.cols : m.rows, length = tall ? m.rows : m.cols;
  const uint32_t height = side <= 64 ? 64 : 128;           // rows that are held
  const uint32_t chunk = height * 128;                     // bytes of a chunk of 64 columns
  const uint32_t x_plane = (length + 63) / 64 * chunk, p_plane = (side + 63) / 64 * chunk;
  if (threadIdx.x == 0) {
    mbar_init(bar, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  // zeros behind the last row and column: they are part of sums
  for (uint32_t i = threadIdx.x; i < (kSmallX + kSmallP) / 16; i += kSmallThreads) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
  pdl_enter();

  // the momentum, u and its size
  const uint32_t count = m.rows * m.cols;
  float u[kSmallEach];
  double sum = 0;
#pragma unroll
  for (int from = 0; from < kSmallEach; from += 8) {        // eight elements' loads on their way
    if (from * kSmallThreads >= count) break;
    float g[8], v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t e = (from + i) * kSmallThreads + threadIdx.x;
      g[i] = m.gradient[min(e, count - 1)], v[i] = m.momentum[min(e, count - 1)];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t e = (from + i) * kSmallThreads + threadIdx.x;
      v[i] = fmaf(t.momentum, v[i], g[i]);
      if (e < count) m.momentum[e] = v[i];
      u[from + i] = e >= count ? 0.f : t.nesterov ? fmaf(t.momentum, v[i], g[i]) : v[i];
      sum += (double)u[from + i] * (double)u[from + i];
    }
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  if (lane == 0) slots[warp] = sum;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  sum = 0;
#pragma unroll
  for (int i = 0; i < kSmallThreads / 32; ++i) sum += slots[i];
  const double by = sum == 0 ? 0 : (double)kX / sqrt(sum);
  // where 16 bytes of a row lie
  auto place = [&](uint32_t row, uint32_t col) { return col / 64 * chunk + row * 128 + (((col & 63) / 8 ^ (row & 7)) << 4); };
  {
    uint32_t row = threadIdx.x / m.cols, col = threadIdx.x - row * m.cols;
    const uint32_t down = kSmallThreads / m.cols, right = kSmallThreads - down * m.cols;
#pragma unroll
    for (int i = 0; i < kSmallEach; ++i) {
      if (i * kSmallThreads >= count) break;
      if (row < m.rows) {
        const uint32_t r = tall ? col : row, c = tall ? row : col;
        __half* const x = reinterpret_cast<__half*>(smem + place(r, c)) + (c & 7);
        split((float)((double)u[i] * by), x, x + x_plane / 2);
      }
      row += down, col += right;
      if (col >= m.cols) col -= m.cols, ++row;
    }
  }

  const int quarter = warp & 3, group = warp >> 2;
  const uint32_t row = quarter * 32 + lane;
  const uint32_t lane_at = tmem + ((uint32_t)(quarter * 32) << 16);
  const bool mine = quarter * 32 < side;                   // (the whole warp)
  const uint32_t x_at = (smem_base & 0x3FFFFu) >> 4, p_at = x_at + (kSmallX >> 4);
  const uint32_t side16 = (side + 15) / 16 * 16, length16 = (length + 15) / 16 * 16;
  const Operand k_major = make_desc(0, 16, 1024, 2), mn_major = make_desc(0, chunk, 1024, 2);
  uint32_t phase = 0;
  // Products of the whole CTA's operands in shared memory: issued by one lane of a warp that runs its loops as a whole, waited for by all.
  const bool leader = elect_one();
  auto multiplied = [&](auto issue) {
    fence_async_smem();
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) return false;
    if (warp == 0) {
      tc_fence_after();
      issue();
      if (leader) tc_commit(bar);
      __syncwarp();
    }
    mbar_wait(bar, phase, abort_flag, t.status, 711, t.wait_ns);
    phase ^= 1;
    tc_fence_after();
    return true;
  };
  auto three = [&](uint32_t acc, Operand a, uint32_t a_hi, uint32_t a_lo, Operand b, uint32_t b_hi, uint32_t b_lo, uint32_t idesc, uint32_t more) {
    if (!leader) return;
    mma_f16(acc, a, a_hi, b, b_hi, idesc, more);
    mma_f16(acc, a, a_lo, b, b_hi, idesc, 1u);
    mma_f16(acc, a, a_hi, b, b_lo, idesc, 1u);
  };
  auto k_offset = [&](uint32_t k16) { return (k16 / 4 * chunk + k16 % 4 * 32) >> 4; };
  // 16 columns of this thread's row as pairs
  auto keep = [&](uint32_t at, uint32_t plane, uint32_t col, const float* v) {
    union { __half h[16]; uint4 bits[2]; } hi, lo;
#pragma unroll
    for (int j = 0; j < 16; ++j) split(v[j], &hi.h[j], &lo.h[j]);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint8_t* const x = smem + at + place(row, col + 8 * j);
      *reinterpret_cast<uint4*>(x) = hi.bits[j];
      *reinterpret_cast<uint4*>(x + plane) = lo.bits[j];
    }
  };

  for (uint32_t step = 0; step < t.steps; ++step) {
    // G = X X^T; every 128 k in an accumulator of its own, as in the product kernel
    if (!multiplied([&] {
          for (uint32_t k = 0; k < length16 / 16; ++k) {
            const uint32_t at = x_at + k_offset(k);
            three(tmem + k / 8 * 128, k_major, at, at + (x_plane >> 4), k_major, at, at + (x_plane >> 4), f16_idesc((int)side16, 0, 0), k % 8 ? 1u : 0u);
          }
        }))
      break;
    float g[32];
    if (mine && (uint32_t)group * 32 < side16) {
#pragma unroll
      for (int j = 0; j < 32; ++j) g[j] = 0.f;
      for (uint32_t run = 0; run < (length16 + 127) / 128; ++run) {
        uint32_t v[32];
        tmem_ld_32x32(lane_at + run * 128 + group * 32, v);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; ++j) g[j] += __uint_as_float(v[j]);
      }
#pragma unroll
      for (int j = 0; j < 32; ++j) g[j] = group * 32 + j < side ? g[j] * (kG / (kX * kX)) : 0.f;
      if (row < side) keep(kSmallX, p_plane, group * 32, g), keep(kSmallX, p_plane, group * 32 + 16, g + 16);
    }
    // P = a + b G + c G G, in the place of G
    if (!multiplied([&] {
          for (uint32_t k = 0; k < side16 / 16; ++k) {
            const uint32_t at = p_at + k_offset(k);
            three(tmem, k_major, at, at + (p_plane >> 4), k_major, at, at + (p_plane >> 4), f16_idesc((int)side16, 0, 0), k ? 1u : 0u);
          }
        }))
      break;
    if (mine && (uint32_t)group * 32 < side16) {
      uint32_t v[32];
      tmem_ld_32x32(lane_at + group * 32, v);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        const uint32_t col = group * 32 + j;
        g[j] = fmaf(t.c * (kP / (kG * kG)), __uint_as_float(v[j]), t.b * (kP / kG) * g[j]) + (col == row ? t.a * kP : 0.f);
        if (col >= side) g[j] = 0.f;
      }
      if (row < side) keep(kSmallX, p_plane, group * 32, g), keep(kSmallX, p_plane, group * 32 + 16, g + 16);
    }
    // P X
    if (!multiplied([&] {
          for (uint32_t from = 0; from < length16; from += 256) {
            const uint32_t n = min(length16 - from, 256u), b_at = x_at + (from / 64 * chunk >> 4);
            for (uint32_t k = 0; k < side16 / 16; ++k) {
              const uint32_t a_at = p_at + k_offset(k), b = b_at + (k * 2048 >> 4);
              three(tmem + from, k_major, a_at, a_at + (p_plane >> 4), mn_major, b, b + (x_plane >> 4), f16_idesc((int)n, 0, 1), k ? 1u : 0u);
            }
          }
        }))
      break;
    const bool last = step + 1 == t.steps;
    if (last) {                                            // (a wait that has given up shows behind the next barrier)
      __syncthreads();
      if (*abort_flag) break;
    }
    if (!mine) continue;
    const float lr = t.schedule ? t.schedule[1] : t.lr, kept = 1.f - lr * m.decay, rate = lr * m.scale / (kP * kX);
    for (uint32_t col = group * 16; col < length16; col += 64) {
      uint32_t v[16];
      __syncwarp();
      tmem_ld_32x16(lane_at + col, v);
      tmem_ld_wait();
      float x[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = __uint_as_float(v[j]) * (last ? rate : 1.f / kP);
      if (!last) {
        // (behind the last column X is zeros, and so are these)
        if (row < side) keep(0, x_plane, col, x);
      } else {
        const uint32_t r = min(row, side - 1);             // (no load behind a branch of a lane's own)
        float* const w = m.weights + (tall ? col * m.cols + r : r * m.cols + col);
        const uint32_t next = tall ? m.cols : 1;
        if (!tall && (m.cols & 3) == 0 && (reinterpret_cast<uintptr_t>(m.weights) & 15) == 0 && col + 16 <= length) {
#pragma unroll
          for (int j = 0; j < 16; j += 4) {
            const float4 o = *reinterpret_cast<const float4*>(w + j);
            x[j] = o.x * kept - x[j], x[j + 1] = o.y * kept - x[j + 1], x[j + 2] = o.z * kept - x[j + 2], x[j + 3] = o.w * kept - x[j + 3];
          }
          if (row < side)
#pragma unroll
            for (int j = 0; j < 16; j += 4) *reinterpret_cast<float4*>(w + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
        } else {
          float o[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) o[j] = w[min((uint32_t)j, length - 1 - col) * next];
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (row < side && col + j < length) w[j * next] = o[j] * kept - x[j];
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000ll) { }
    __syncthreads();
  }
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---- narrow matrices: what lies between two products with X, by one CTA for each

// The symmetric matrices of a matrix with a short side of up to 128 fit a CTA's shared memory: P, T, G', P' and Q of two rounds (or P of one), 1 to 1.5 us each, in
// one launch for five of some 7: a step of 32 x 8192 takes 88 us for 108, 128 x 512 93 for 127.  Squares as X in the kernel above, 128 rows.
struct Chain {
  const __half* g;                                         // matrix z: planes 2 z (hi) and 2 z + 1 (lo)
  __half* out;
  uint64_t plane;
  uint32_t side, pitch, first;                             // first: its first CTA
};
constexpr int kChains = 64;
struct ChainTable {
  float a, b, c;
  int two;
  uint32_t shapes;
  int *status, *failed;
  unsigned long long wait_ns;
  Chain s[kChains];
};
constexpr uint32_t kSquare = 64 * 1024;                    // 128 x 128 pairs
static_assert(kSquare == kNarrow * kNarrow * 4, "a square for each of them");
constexpr uint32_t kChainBytes = 3 * kSquare + 1024 + 256;

__global__ void __launch_bounds__(kSmallThreads, 1) chain_kernel(const __grid_constant__ ChainTable t) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const smem = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t bar = smem_base + 3 * kSquare;
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(smem + 3 * kSquare + 8);
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = uniform_warp(), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(bar, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    tmem_alloc(smem_u32(tmem_slot), 128);
    tmem_relinquish();
  }
  uint32_t shape = 0;
  while (shape + 1 < t.shapes && t.s[shape + 1].first <= blockIdx.x) ++shape;
  const Chain& q = t.s[shape];
  const uint64_t first = 2 * (uint64_t)(blockIdx.x - q.first) * q.plane;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  pdl_enter();

  const uint32_t side = q.side, side16 = (side + 15) / 16 * 16, row = (warp & 3) * 32 + lane, col = (warp >> 2) * 32;
  const bool mine = (warp & 3) * 32 < side && col < side16;   // a block of 32 x 32 (the whole warp)
  constexpr uint32_t kChunk64 = 128 * 128, kPlane = kSquare / 2;
  const Operand k_major = make_desc(0, 16, 1024, 2);
  const bool leader = elect_one();
  uint32_t phase = 0;
  // The product of the matrices in squares l and r.
  auto product = [&](uint32_t l, uint32_t r) {
    fence_async_smem();
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) return false;
    if (warp == 0) {
      tc_fence_after();
      const uint32_t base = (smem_base & 0x3FFFFu) >> 4, lo = kPlane >> 4, idesc = f16_idesc((int)side16, 0, 0);
      if (leader) {
        for (uint32_t k = 0; k < side16 / 16; ++k) {
          const uint32_t at = (k / 4 * kChunk64 + k % 4 * 32) >> 4, a = base + (l * kSquare >> 4) + at, b = base + (r * kSquare >> 4) + at;
          mma_f16(tmem, k_major, a, k_major, b, idesc, k ? 1u : 0u);
          mma_f16(tmem, k_major, a + lo, k_major, b, idesc, 1u);
          mma_f16(tmem, k_major, a, k_major, b + lo, idesc, 1u);
        }
        tc_commit(bar);
      }
      __syncwarp();
    }
    mbar_wait(bar, phase, abort_flag, t.status, 721, t.wait_ns);
    phase ^= 1;
    tc_fence_after();
    return true;
  };
  auto sums = [&](float* v) {
    uint32_t bits[32];
    tmem_ld_32x32(tmem + ((uint32_t)((warp & 3) * 32) << 16) + col, bits);
    tmem_ld_wait();
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(bits[j]);
  };
  // 32 columns of this thread's row into a square; behind the last column zeros, which are part of sums
  auto keep = [&](uint32_t square, float* v) {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = col + j < side ? v[j] : 0.f;
    if (row >= side) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      union { __half h[8]; uint4 bits; } hi, lo;
#pragma unroll
      for (int j = 0; j < 8; ++j) split(v[8 * i + j], &hi.h[j], &lo.h[j]);
      uint8_t* const x = smem + square * kSquare + col / 64 * kChunk64 + row * 128 + (((col & 63) / 8 + i) ^ (row & 7)) * 16;
      *reinterpret_cast<uint4*>(x) = hi.bits;
      *reinterpret_cast<uint4*>(x + kPlane) = lo.bits;
    }
  };
  auto polynomial = [&](const float* g, float* v) {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = fmaf(t.c * (kP / (kG * kG)), v[j], t.b * (kP / kG) * g[j]) + (col + j == row ? t.a * kP : 0.f);
  };
  auto times = [&](float by, float* v) {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] *= by;
  };

  float g[32], v[32];
  if (mine) {
    const __half* const in = q.g + first + (uint64_t)min(row, side - 1) * q.pitch + col;
    uint4 hi[4], lo[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) hi[i] = reinterpret_cast<const uint4*>(in)[i], lo[i] = reinterpret_cast<const uint4*>(in + q.plane)[i];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float2 x = __half22float2(reinterpret_cast<const __half2*>(hi)[j]), y = __half22float2(reinterpret_cast<const __half2*>(lo)[j]);
      g[2 * j] = x.x + y.x, g[2 * j + 1] = x.y + y.y;
    }
    keep(0, g);
  }
  bool ok = product(0, 0);
  if (mine && ok) {
    sums(v);
    polynomial(g, v);
    if (t.two) keep(1, v);
  }
  if (t.two) {
    ok = ok && product(1, 0);                              // T
    if (mine && ok) {
      sums(v);
      times(1.f / kP, v);
      keep(2, v);
    }
    ok = ok && product(1, 2);                              // G'
    if (mine && ok) {
      sums(g);
      times(1.f / kP, g);
      keep(0, g);
    }
    ok = ok && product(0, 0);                              // P'
    if (mine && ok) {
      sums(v);
      polynomial(g, v);
      keep(2, v);
    }
    ok = ok && product(2, 1);                              // Q
    if (mine && ok) {
      sums(v);
      times(kQ / (kP * kP), v);
    }
  }
  if (mine && ok && row < side) {                          // (columns behind the last one lie in the row's padding)
    __half* const out = q.out + first + (uint64_t)row * q.pitch + col;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      union { __half h[8]; uint4 bits; } hi, lo;
#pragma unroll
      for (int j = 0; j < 8; ++j) split(v[8 * i + j], &hi.h[j], &lo.h[j]);
      reinterpret_cast<uint4*>(out)[i] = hi.bits;
      reinterpret_cast<uint4*>(out + q.plane)[i] = lo.bits;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    if (threadIdx.x == 0) *t.failed = 1;
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000ll) { }
    __syncthreads();
  }
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 128);
  }
}

// ---- host side

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
  static EncodeTiled fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiled>(p);
  });
  return fn;
}

// `planes` matrices of fp16 [rows][cols], rows `pitch` (a multiple of 64) apart, as an operand, in boxes of `tile` rows or columns and BK k, or as
// a result, in blocks of 32 x 32.  MN-major boxes are chunks of 64 columns: the last one may
// reach into a row's padding, whose values end in rows or columns of a product that nobody reads.
int make_map(CUtensorMap* map, const __half* base, uint64_t rows, uint64_t cols, uint64_t pitch, uint64_t planes, bool mn, uint32_t tile) {
  EncodeTiled encode = encode_tiled();
  if (!encode) return fail(POLAR_B200_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
  const cuuint32_t unit[4] = {1, 1, 1, 1};
  CUresult r;
  if (mn) {
    const cuuint64_t dims[4] = {64, rows, pitch / 64, planes}, strides[3] = {pitch * 2, 128, rows * pitch * 2};
    const cuuint32_t box[4] = {64, BK, tile / 64, 2};
    r = encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<__half*>(base), dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  } else {
    const cuuint64_t dims[3] = {cols, rows, planes}, strides[2] = {pitch * 2, rows * pitch * 2};
    const cuuint32_t box[3] = {BK, tile, 2};               // (a result's blocks are 32 columns wide as well)
    r = encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half*>(base), dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  }
  return r == CUDA_SUCCESS ? POLAR_B200_OK : fail(POLAR_B200_ERR_CUDA, "cuTensorMapEncodeTiled failed");
}

struct One {                                               // a matrix of the call
  float* weights;
  const float* gradient;
  float* momentum;
  uint64_t rows, cols;
  float decay, scale;
};
struct Kin {                                               // the matrices of one shape
  uint64_t rows, cols, count, first;                       // first: among the sorted matrices
  uint64_t pitch, side, side_pitch;                        // side: the shorter one
  __half *x[2], *s[3];                                     // X, and the symmetric matrices
};
uint64_t up64(uint64_t n) { return (n + 63) / 64 * 64; }
uint64_t up256(uint64_t n) { return (n + 255) & ~255ull; }
uint64_t chunk_of(uint64_t count) {
  const uint64_t each = (count + kMostChunks - 1) / kMostChunks;
  return each <= kChunk ? kChunk : (each + kChunk - 1) / kChunk * kChunk;
}
uint64_t bytes_of(uint64_t rows, uint64_t cols) {          // of one matrix: X twice and the symmetric ones, two planes each, and what is small, rounded up
  const uint64_t side = std::min(rows, cols);
  return 2 * 2 * (2 * rows * up64(cols) + (in_pairs(rows, cols) ? 3 : 2) * side * up64(side)) + kMostChunks * sizeof(double) + sizeof(Target) + 8 * 256;
}
// What one group of matrices may take; a step of more is done in several.
constexpr uint64_t kGroupBytes = 3ull << 30;

struct Group {                                             // what lies in the workspace
  std::vector<Kin> kin;
  int* failed;                                             // whether a wait has given up; it comes first
  double* partial;
  Target* targets;
};
// Lays out a group that is sorted by shape, in what lies behind `base`; its bytes.
uint64_t lay_out(char* base, const std::vector<One>& all, size_t from, size_t to, Group* group) {
  std::vector<Kin>* const kin = &group->kin;
  uint64_t at = 0, chunks = 0;
  auto take = [&](uint64_t n) {
    char* p = base + at;
    at += up256(n);
    return p;
  };
  for (size_t i = from; i < to; ++i) {
    const One& o = all[i];
    chunks += (o.rows * o.cols + chunk_of(o.rows * o.cols) - 1) / chunk_of(o.rows * o.cols);
    if (kin->empty() || kin->back().rows != o.rows || kin->back().cols != o.cols) {
      const uint64_t side = std::min(o.rows, o.cols);
      kin->push_back(Kin{o.rows, o.cols, 0, i - from, up64(o.cols), side, up64(side), {nullptr, nullptr}, {nullptr, nullptr, nullptr}});
    }
    ++kin->back().count;
  }
  group->failed = reinterpret_cast<int*>(take(sizeof(int)));
  group->partial = reinterpret_cast<double*>(take(chunks * sizeof(double)));
  group->targets = reinterpret_cast<Target*>(take((to - from) * sizeof(Target)));
  for (Kin& k : *kin) {
    for (int b = 0; b < 2; ++b) k.x[b] = reinterpret_cast<__half*>(take(k.count * 4 * k.rows * k.pitch));
    for (int b = 0; b < (in_pairs(k.rows, k.cols) ? 3 : 2); ++b) k.s[b] = reinterpret_cast<__half*>(take(k.count * 4 * k.side * k.side_pitch));
  }
  return at;
}

uint64_t workspace_of(const std::vector<One>& all, const std::vector<size_t>& ends) {
  uint64_t most = 0;
  size_t from = 0;
  for (size_t to : ends) {
    Group group;
    most = std::max(most, lay_out(nullptr, all, from, to, &group));
    from = to;
  }
  return most;
}

template <int N>
int launch_tables(const std::vector<One>& all, size_t from, size_t to, const Group& group, const polar_b200_muon_options& o, cudaStream_t st, bool begin) {
  const std::vector<Kin>& kin = group.kin;
  static thread_local Table<N> t;
  size_t k = 0, i = from;
  uint32_t chunks_before = 0;
  while (i < to) {
    t.count = 0;
    t.chunks_before = chunks_before, t.matrices_before = (uint32_t)(i - from);
    t.momentum = o.momentum, t.nesterov = o.nesterov, t.partial = group.partial, t.targets = group.targets, t.failed = group.failed;
    uint32_t chunks = 0;
    for (; i < to && t.count < N; ++i) {
      while (k + 1 < kin.size() && i - from >= kin[k + 1].first) ++k;
      const One& q = all[i];
      const uint64_t count = q.rows * q.cols, plane = q.rows * kin[k].pitch;
      t.m[t.count++] = Matrix{q.weights, q.gradient, q.momentum, kin[k].x[0] + 2 * (i - from - kin[k].first) * plane, plane, count, (uint32_t)q.cols,
                              (uint32_t)kin[k].pitch, (uint32_t)chunk_of(count), chunks, q.decay, q.scale};
      chunks += (uint32_t)((count + chunk_of(count) - 1) / chunk_of(count));
    }
    const int rc = begin ? launch_large("fmuon: X", begin_kernel<N>, dim3(chunks), kThreads, st, t)
                         : launch_large("fmuon: momentum", momentum_kernel<N>, dim3(chunks), kThreads, st, t);
    if (rc) return rc;
    chunks_before += chunks;
  }
  return POLAR_B200_OK;
}

// How a launch's products are computed: in tiles of 128 x bn, of which a cluster of `splits` CTAs has one (1: a CTA at a time).
struct Way {
  uint32_t bn, splits;
};
uint64_t tiles_of(uint64_t m, uint64_t n, bool symmetric, uint64_t bn) {
  const uint64_t tiles_m = (m + BM - 1) / BM, tiles_n = (n + bn - 1) / bn;
  if (!symmetric) return tiles_m * tiles_n;
  uint64_t tiles = 0;
  for (uint64_t i = 0; i < tiles_m; ++i) tiles += tiles_n - i * BM / bn;
  return tiles;
}
struct Extent {
  uint64_t m, n, k, count;
  bool symmetric;
};
// The way whose busiest SM is done first.  A slab takes 0.45 us with tiles of 256 columns and 0.28 with tiles of 128 (few at a time; all SMs at once are held up by
// the power they take), what stands around a tile 5.2 and 4 us, and with a cluster that shares one, and adds its sums, 6.5.  Clusters of four or eight leave some SMs out.
Way way_of(const std::vector<Extent>& e) {
  Way best = {256, 1};
  double least = 0;
  for (const Way w : {Way{256, 1}, Way{128, 1}, Way{128, 2}, Way{128, 4}, Way{128, 8}}) {
    const uint64_t sms = w.splits == 1 ? (uint64_t)sm_count() : w.splits == 2 ? 146 : w.splits == 4 ? 136 : 128;
    const double slab = w.bn == 256 ? 0.45 : 0.28, around = w.bn == 256 ? 5.2 : w.splits == 1 ? 4.0 : 6.5;
    double us = 0;
    uint64_t before = 0, next = 0;                         // tiles passed, and the next one of the first SM
    for (const Extent& x : e) {
      const uint64_t units = tiles_of(x.m, x.n, x.symmetric, w.bn) * x.count * w.splits, slabs = (x.k + BK - 1) / BK;
      const double each = (double)((slabs + w.splits - 1) / w.splits) * slab + around;
      for (before += units; next < before; next += sms) us += each;
    }
    if (least == 0 || us < least) least = us, best = w;
  }
  return best;
}

// The next operation of every shape, longest sums first.
template <int BN, bool SPLIT>
int launch_product(const Group& group, const std::vector<std::pair<size_t, Operation>>& ops, const std::vector<int>& from_x, const polar_b200_muon_options& o,
                   int* status, cudaStream_t st, uint32_t splits) {
  const std::vector<Kin>& kin = group.kin;
  if constexpr (BN == 256) {
    // the split waits for registers that the launch has to hold: built with fewer of them it would wait for good
    static const bool enough = [] {
      cudaFuncAttributes a;
      return cudaFuncGetAttributes(&a, product_kernel<BN, SPLIT>) == cudaSuccess && a.numRegs * kProductThreads >= kSplitRegisters;
    }();
    if (!enough) return fail(POLAR_B200_ERR_CUDA, "fmuon: the product kernel was built with too few registers");
  }
  static thread_local Product p;
  p.splits = splits;
  p.lr = o.lr, p.schedule = o.schedule, p.targets = group.targets, p.status = status, p.failed = group.failed, p.wait_ns = wait_limit_ns(2000000000ull);
  for (size_t k = 0; k < ops.size();) {
    p.shapes = p.tiles = 0;
    for (; k < ops.size() && p.shapes < kShapes; ++k) {
      const Kin& q = kin[ops[k].first];
      const Operation& op = ops[k].second;
      const int from = from_x[ops[k].first];
      const bool wide = q.rows <= q.cols, square = op.what != Operation::kMove;
      Shape& s = p.s[p.shapes];
      int rc = POLAR_B200_OK;
      auto x = [&](CUtensorMap* map, int which, bool mn, uint32_t tile) { return make_map(map, q.x[which], q.rows, q.cols, q.pitch, 2 * q.count, mn, tile); };
      auto symmetric = [&](CUtensorMap* map, int t, uint32_t tile) { return make_map(map, q.s[t], q.side, q.side, q.side_pitch, 2 * q.count, false, tile); };
      s.kind = square ? kSymmetric : op.last ? kUpdate : kRound;
      s.by = op.by, s.add_by = op.add_by, s.diagonal = op.diagonal;
      s.add = op.add >= 0 ? q.s[op.add] : nullptr;
      s.a_mn = s.b_mn = 0;
      if (op.what == Operation::kGram) {                   // X X^T, or X^T X
        s.m = s.n = (uint32_t)q.side, s.k = (uint32_t)std::max(q.rows, q.cols);
        s.a_mn = s.b_mn = !wide;
        rc = x(&s.a, from, !wide, BM);
        if (!rc) rc = x(&s.b, from, !wide, BN);
      } else if (op.what == Operation::kProduct) {
        s.m = s.n = s.k = (uint32_t)q.side;
        rc = symmetric(&s.a, op.left, BM);
        if (!rc) rc = symmetric(&s.b, op.right, BN);
      } else {                                             // P X, or X P
        s.m = (uint32_t)q.rows, s.n = (uint32_t)q.cols, s.k = (uint32_t)q.side;
        s.b_mn = wide;
        rc = wide ? symmetric(&s.a, op.left, BM) : x(&s.a, from, false, BM);
        if (!rc) rc = wide ? x(&s.b, from, true, BN) : symmetric(&s.b, op.left, BN);
      }
      if (!rc && !SPLIT && !op.last) rc = square ? symmetric(&s.c, op.out, 32) : x(&s.c, from ^ 1, false, 32);
      if (rc) return rc;
      s.out = square ? q.s[op.out] : q.x[from ^ 1];
      s.pitch = (uint32_t)(square ? q.side_pitch : q.pitch);
      s.plane = square ? q.side * q.side_pitch : q.rows * q.pitch;
      s.first_target = (uint32_t)q.first;
      s.tiles_m = (s.m + BM - 1) / BM, s.tiles_n = (s.n + BN - 1) / BN;
      s.tiles = (uint32_t)tiles_of(s.m, s.n, square, BN);
      s.first_tile = p.tiles;
      p.tiles += s.tiles * (uint32_t)q.count;
      ++p.shapes;
    }
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3(SPLIT ? p.tiles * splits : std::min(p.tiles, (uint32_t)sm_count()));
    c.blockDim = dim3(kProductThreads);
    c.dynamicSmemBytes = Cfg<BN, SPLIT>::kBytes;
    c.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = splits;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    c.attrs = at;
    c.numAttrs = SPLIT ? 2 : 1;
    cudaError_t e = cudaFuncSetAttribute(product_kernel<BN, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Cfg<BN, SPLIT>::kBytes);
    void* args[1] = {&p};
    if (e == cudaSuccess) e = cudaLaunchKernelExC(&c, reinterpret_cast<const void*>(product_kernel<BN, SPLIT>), args);
    if (e != cudaSuccess) {
      cudaGetLastError();
      return fail(POLAR_B200_ERR_CUDA, "fmuon: product", e);
    }
    count_launch();
  }
  return POLAR_B200_OK;
}

// The products of symmetric matrices between two with X, of all shapes (which are all narrow).
int launch_chain(const Group& group, const Operation& op, const polar_b200_muon_options& o, int* status, cudaStream_t st) {
  const std::vector<Kin>& kin = group.kin;
  static thread_local ChainTable t;
  t.a = o.a, t.b = o.b, t.c = o.c, t.two = op.what == Operation::kChain2;
  t.status = status, t.failed = group.failed, t.wait_ns = wait_limit_ns(2000000000ull);
  cudaError_t e = cudaFuncSetAttribute(chain_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kChainBytes);
  if (e != cudaSuccess) return fail(POLAR_B200_ERR_CUDA, "fmuon: narrow matrices", e);
  for (size_t k = 0; k < kin.size();) {
    uint32_t ctas = 0;
    for (t.shapes = 0; k < kin.size() && t.shapes < kChains; ++k) {
      const Kin& q = kin[k];
      t.s[t.shapes++] = Chain{q.s[op.left], q.s[op.out], q.side * q.side_pitch, (uint32_t)q.side, (uint32_t)q.side_pitch, ctas};
      ctas += (uint32_t)q.count;
    }
    const int rc = launch("fmuon: narrow matrices", chain_kernel, dim3(ctas), kSmallThreads, kChainBytes, st, t);
    if (rc) return rc;
  }
  return POLAR_B200_OK;
}

// The matrices of the call, longest sums first, and the groups they are done in; behind the last group's end the small ones.
void matrices_of(const polar_b200_muon_tensor* tensors, uint64_t count, std::vector<One>* all, std::vector<size_t>* ends, bool large_only) {
  all->reserve(count);
  for (uint64_t i = 0; i < count; ++i) {
    const polar_b200_muon_tensor& t = tensors[i];
    if (large_only && is_small(t.rows, t.cols)) continue;
    for (uint64_t z = 0; z < t.matrices && t.rows && t.cols; ++z) {
      const uint64_t at = z * t.rows * t.cols;
      all->push_back(One{t.weights + at, t.gradient + at, t.momentum + at, t.rows, t.cols, t.weight_decay, t.scale});
    }
  }
  std::stable_sort(all->begin(), all->end(), [](const One& a, const One& b) {
    const bool sa = is_small(a.rows, a.cols), sb = is_small(b.rows, b.cols);
    const uint64_t la = std::max(a.rows, a.cols), lb = std::max(b.rows, b.cols);
    return sa != sb ? sb : la != lb ? la > lb : a.rows != b.rows ? a.rows > b.rows : a.cols > b.cols;
  });
  uint64_t bytes = 0;
  size_t large = all->size();
  while (large && is_small((*all)[large - 1].rows, (*all)[large - 1].cols)) --large;
  for (size_t i = 0; i < large; ++i) {
    const uint64_t more = bytes_of((*all)[i].rows, (*all)[i].cols);
    if (bytes && bytes + more > kGroupBytes) ends->push_back(i), bytes = 0;
    bytes += more;
  }
  if (large) ends->push_back(large);
}

template <int N>
int launch_small(const std::vector<One>& all, size_t from, size_t to, const polar_b200_muon_options& o, int* status, cudaStream_t st) {
  static thread_local SmallTable<N> t;
  t.lr = o.lr, t.momentum = o.momentum, t.a = o.a, t.b = o.b, t.c = o.c, t.nesterov = o.nesterov, t.steps = o.steps, t.schedule = o.schedule;
  t.status = status, t.wait_ns = wait_limit_ns(2000000000ull);
  cudaError_t e = cudaFuncSetAttribute(small_kernel<N>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmallBytes);
  if (e != cudaSuccess) return fail(POLAR_B200_ERR_CUDA, "fmuon: small matrices", e);
  while (from < to) {
    const size_t n = std::min<size_t>(to - from, N);
    for (size_t i = 0; i < n; ++i) {
      const One& q = all[from + i];
      t.m[i] = Small{q.weights, q.gradient, q.momentum, (uint32_t)q.rows, (uint32_t)q.cols, q.decay, q.scale};
    }
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3((unsigned)n);
    c.blockDim = dim3(kSmallThreads);
    c.dynamicSmemBytes = kSmallBytes;
    c.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    c.attrs = at;
    c.numAttrs = 1;
    void* args[1] = {&t};
    e = cudaLaunchKernelExC(&c, reinterpret_cast<const void*>(small_kernel<N>), args);
    if (e != cudaSuccess) {
      cudaGetLastError();
      return fail(POLAR_B200_ERR_CUDA, "fmuon: small matrices", e);
    }
    count_launch();
    from += n;
  }
  return POLAR_B200_OK;
}

int run_group(const std::vector<One>& all, size_t from, size_t to, const polar_b200_muon_options& o, char* base, cudaStream_t st) {
  Group group;
  lay_out(base, all, from, to, &group);
  const std::vector<Kin>& kin = group.kin;
  int rc;
  int* status = device_status_word(&rc);
  if (rc) return rc;
  for (int begin = 0; begin < 2; ++begin) {
    rc = to - from <= kFewMatrices ? launch_tables<kFewMatrices>(all, from, to, group, o, st, begin)
                                   : launch_tables<kManyMatrices>(all, from, to, group, o, st, begin);
    if (rc) return rc;
  }
  std::vector<int> from_x(kin.size(), 0);
  std::vector<Sides> shapes;
  for (const Kin& k : kin) shapes.push_back(Sides{k.rows, k.cols});
  for (Launch& next : launches_of(shapes, o.steps, o.a, o.b, o.c)) {
    if (next.chain) {
      rc = launch_chain(group, next.ops[0].second, o, status, st);
      if (rc) return rc;
      continue;
    }
    auto& now = next.ops;
    auto sum = [&](const std::pair<size_t, Operation>& a) {
      return a.second.what == Operation::kGram ? std::max(kin[a.first].rows, kin[a.first].cols) : kin[a.first].side;
    };
    std::stable_sort(now.begin(), now.end(), [&](const auto& a, const auto& b) { return sum(a) > sum(b); });
    std::vector<Extent> extents;
    for (const auto& a : now) {
      const Kin& q = kin[a.first];
      const bool square = a.second.what != Operation::kMove;
      extents.push_back(Extent{square ? q.side : q.rows, square ? q.side : q.cols, sum(a), q.count, square});
    }
    const Way way = way_of(extents);
    rc = way.splits > 1  ? launch_product<128, true>(group, now, from_x, o, status, st, way.splits)
         : way.bn == 128 ? launch_product<128, false>(group, now, from_x, o, status, st, 1)
                         : launch_product<256, false>(group, now, from_x, o, status, st, 1);
    if (rc) return rc;
    for (const auto& a : now) from_x[a.first] ^= a.second.what == Operation::kMove;
  }
  return POLAR_B200_OK;
}

// Whether no singular value passes kBound, nor one of P kBoundP, in any round: X begins with singular values up to 1.
bool stays_bounded(float a, float b, float c, uint32_t steps) {
  if (!(std::isfinite(a) && std::isfinite(b) && std::isfinite(c))) return false;
  double most = 1.001;
  for (uint32_t i = 0; i < steps && i < 32; ++i) {
    double next = 0;
    for (int j = 0; j <= 1024; ++j) {
      const double s = most * j / 1024, p = a + s * s * (b + c * s * s);
      if (!(std::fabs(p) <= kBoundP)) return false;
      next = std::max(next, std::fabs(p) * s);
    }
    most = std::max(next * 1.0001, 1e-3);
    if (!(most <= kBound)) return false;
  }
  return true;
}

bool disjoint(const polar_b200_muon_tensor* tensors, uint64_t count, const float* schedule) {
  using Span = std::pair<uintptr_t, uintptr_t>;
  std::vector<Span> written, read;
  auto span = [](const void* p, uint64_t bytes) { return Span(reinterpret_cast<uintptr_t>(p), reinterpret_cast<uintptr_t>(p) + bytes); };
  for (uint64_t i = 0; i < count; ++i) {
    const uint64_t bytes = 4 * tensors[i].matrices * tensors[i].rows * tensors[i].cols;
    if (!bytes) continue;
    written.push_back(span(tensors[i].weights, bytes));
    written.push_back(span(tensors[i].momentum, bytes));
    read.push_back(span(tensors[i].gradient, bytes));
  }
  if (schedule) read.push_back(span(schedule, 8));
  std::sort(written.begin(), written.end());
  for (size_t i = 1; i < written.size(); ++i)
    if (written[i].first < written[i - 1].second) return false;
  for (const Span& r : read) {
    const auto next = std::lower_bound(written.begin(), written.end(), Span(r.second, 0));
    if (next != written.begin() && std::prev(next)->second > r.first) return false;
  }
  return true;
}

bool valid(const polar_b200_muon_tensor& t) {
  constexpr uint64_t kLong = 1ull << 20, kShort = 1ull << 15;
  if (!t.matrices || !t.rows || !t.cols) return true;
  return t.rows <= kLong && t.cols <= kLong && std::min(t.rows, t.cols) <= kShort && t.matrices <= 1ull << 20 && t.matrices * t.rows * t.cols <= 1ull << 36;
}

}  // namespace

// Whether the steps may run in any order or at once: no written array overlaps another, a gradient or the schedule.
bool muon_independent(const polar_b200_muon_tensor* tensors, uint64_t count, const float* schedule) { return disjoint(tensors, count, schedule); }

// The argument list of the builtin "fmuon" as the entry point takes it; false where it is none.
bool muon_arguments(const char* name, const polar_b200_arg* a, uint64_t argc, polar_b200_muon_tensor* t, polar_b200_muon_options* o) {
  static const char pattern[] = "TTfffffTT";
  if (std::strcmp(name, "fmuon") || argc != sizeof(pattern) - 1) return false;
  uint64_t n[9] = {};
  for (uint64_t i = 0; i < argc; ++i) {
    if ((pattern[i] == 'T') != (a[i].is_tensor != 0)) return false;
    if (!a[i].is_tensor) continue;
    if (a[i].tensor.dims && !a[i].tensor.shape) return false;
    n[i] = 1;
    for (uint64_t d = 0; d < a[i].tensor.dims; ++d) n[i] *= a[i].tensor.shape[d];
  }
  const polar_b200_tensor& w = a[7].tensor;
  const float steps = a[4].scalar;
  if (w.dims < 2 || n[0] != n[7] || n[8] != n[7] || n[1] != 2 || !a[1].tensor.data || (a[3].scalar != 0.f && a[3].scalar != 1.f) ||
      !(steps >= 1.f && steps <= 32.f) || steps != (float)(uint32_t)steps)
    return false;
  const uint64_t rows = w.shape[w.dims - 2], cols = w.shape[w.dims - 1];
  for (int i : {0, 8}) {                                   // (as many elements of another shape would be other matrices)
    const polar_b200_tensor& x = a[i].tensor;
    if (x.dims < 2 || x.shape[x.dims - 2] != rows || x.shape[x.dims - 1] != cols) return false;
  }
  *t = polar_b200_muon_tensor{w.data, a[0].tensor.data, a[8].tensor.data, rows && cols ? n[7] / (rows * cols) : 0, rows, cols, a[5].scalar, a[6].scalar};
  *o = polar_b200_muon_options{0.f, a[2].scalar, a[3].scalar != 0.f, (uint32_t)steps, 3.4445f, -4.7750f, 2.0315f, a[1].tensor.data};
  return true;
}

}  // namespace polar_b200

using namespace polar_b200;

extern "C" {

uint64_t polar_b200_fmuon_workspace_bytes(const polar_b200_muon_tensor* tensors, uint64_t count) {
  if (!tensors) return 0;
  for (uint64_t i = 0; i < count; ++i)
    if (!valid(tensors[i])) return 0;
  try {
    std::vector<One> all;
    std::vector<size_t> ends;
    matrices_of(tensors, count, &all, &ends, true);
    return workspace_of(all, ends);
  } catch (const std::exception&) {
    return 0;
  }
}

int polar_b200_fmuon(const polar_b200_muon_tensor* tensors, uint64_t count, const polar_b200_muon_options* o, void* workspace, uint64_t workspace_bytes,
                     void* stream) {
  clear_error();
  if (!o || (count && !tensors)) return fail(POLAR_B200_ERR_INVALID, "fmuon: no tensors or options");
  if (!(o->momentum >= 0.f && o->momentum < 1.f)) return fail(POLAR_B200_ERR_INVALID, "fmuon: 0 <= momentum < 1 is needed");
  if (o->steps < 1 || o->steps > 32 || !stays_bounded(o->a, o->b, o->c, o->steps))
    return fail(POLAR_B200_ERR_INVALID, "fmuon: 1 to 32 rounds of a polynomial that lets no singular value pass 1.4");
  const void* some = nullptr;
  for (uint64_t i = 0; i < count; ++i) {
    const polar_b200_muon_tensor& t = tensors[i];
    if (!valid(t)) return fail(POLAR_B200_ERR_INVALID, "fmuon: matrix too large");
    if (!(t.matrices && t.rows && t.cols)) continue;
    if (!t.weights || !t.gradient || !t.momentum) return fail(POLAR_B200_ERR_INVALID, "null device pointer");
    some = t.weights;
  }
  if (!some) return POLAR_B200_OK;
  try {
    if (!muon_independent(tensors, count, o->schedule)) return fail(POLAR_B200_ERR_INVALID, "fmuon: what is written overlaps something else");
    std::vector<One> all;
    std::vector<size_t> ends;
    matrices_of(tensors, count, &all, &ends, false);
    const uint64_t need = workspace_of(all, ends);
    if (workspace && (workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255)))
      return fail(POLAR_B200_ERR_WORKSPACE, "workspace too small or not 256-byte aligned");
    LaunchDeviceScope on(stream, some);
    cudaStream_t st = as_stream(stream);
    void* own = nullptr;
    if (!workspace && need) {
      cudaError_t e = scratch_alloc(&own, need, st);
      if (e != cudaSuccess) return fail(POLAR_B200_ERR_CUDA, "scratch (workspace)", e);
    }
    int rc = POLAR_B200_OK;
    size_t from = 0;
    for (size_t to : ends) {
      rc = run_group(all, from, to, *o, static_cast<char*>(workspace ? workspace : own), st);
      if (rc) break;
      from = to;
    }
    if (rc == POLAR_B200_OK && from < all.size()) {
      int* status = device_status_word(&rc);
      if (!rc) rc = all.size() - from <= kFewSmall ? launch_small<kFewSmall>(all, from, all.size(), *o, status, st)
                                                   : launch_small<kManySmall>(all, from, all.size(), *o, status, st);
    }
    if (own) {
      cudaError_t e = scratch_free(own, st);
      if (rc == POLAR_B200_OK && e != cudaSuccess) rc = fail(POLAR_B200_ERR_CUDA, "returning scratch", e);
    }
    return rc;
  } catch (const std::exception&) {                        // (no exception may leave a C entry)
    return fail(POLAR_B200_ERR_INVALID, "out of host memory");
  }
}

}  // extern "C"
