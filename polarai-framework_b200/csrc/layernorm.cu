// Layer norm of rows and its backward pass.
//
// HBM-bound streams: 8 bytes per element forward (a row is read and written), 12 backward (two rows read, one
// written), and a dozen operations each.  Deviations are summed around the mean, never as the difference of
// two large sums.  A row's sums are taken over two levels and more (32 elements of a thread at most, then lanes, warps, CTAs), so that their rounding stays near
// that of a few dozen additions whatever the row's length.  The weights' gradients are summed over the rows of a team one after the other
// (222 of 65536 x 4096), then over the teams.
#include <algorithm>
#include <atomic>

#include "rows.cuh"

namespace polar_b200 {
namespace {

constexpr int kThreads = 256;

// A load (0 otherwise) and a store where k < live, under predicates: the compiler makes a branch of each, some four instructions more for every
// float (65536 x 1511: 125 us, by branches a third more).
__device__ __forceinline__ float ld_if(const float* p, int k, uint32_t live) {
  float v;
  asm volatile("{.reg .pred q; setp.lt.s32 q, %2, %3; mov.f32 %0, 0f00000000; @q ld.global.f32 %0, [%1];}" : "=f"(v) : "l"(p), "r"(k), "r"(live) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_if(const float4* p, int k, uint32_t live) {
  float4 v;
  asm volatile("{.reg .pred q; setp.lt.s32 q, %5, %6; mov.f32 %0, 0f00000000; mov.f32 %1, 0f00000000; mov.f32 %2, 0f00000000; mov.f32 %3, 0f00000000;"
               " @q ld.global.v4.f32 {%0, %1, %2, %3}, [%4];}"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p), "r"(k), "r"(live) : "memory");
  return v;
}
__device__ __forceinline__ void st_if(float* p, float v, int k, uint32_t live) {
  asm volatile("{.reg .pred q; setp.lt.s32 q, %2, %3; @q st.global.f32 [%0], %1;}" ::"l"(p), "f"(v), "r"(k), "r"(live) : "memory");
}
__device__ __forceinline__ void st_if(float4* p, float4 v, int k, uint32_t live) {
  asm volatile("{.reg .pred q; setp.lt.s32 q, %5, %6; @q st.global.v4.f32 [%0], {%1, %2, %3, %4};}" ::"l"(p), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w),
               "r"(k), "r"(live)
               : "memory");
}

// A thread's share of a row: 4 V elements of it, TEAM threads to a row.  VECTOR: vectors of four, a team's side by side; else single floats.
// Of the V fours, all threads have the first FULL (cols >= 4 TEAM FULL); `live`: how many of the vectors or floats this thread has in all.
template <int TEAM, int V, bool VECTOR, int FULL>
struct Share {
  static constexpr int N = 4 * V, kFull = FULL;
  static __device__ __forceinline__ uint32_t live(uint32_t member, uint32_t cols) {
    const uint32_t first = VECTOR ? 4 * member : member, step = VECTOR ? 4 * TEAM : TEAM;
    return first < cols ? (cols - first + step - 1) / step : 0;
  }
  static __device__ __forceinline__ bool has(uint32_t live, int k) { return k < 4 * FULL || (VECTOR ? k / 4 : k) < (int)live; }
  static __device__ __forceinline__ void load(float (&v)[N], const float* row, uint32_t member, uint32_t live) {
    if (VECTOR) {
      const float4* p = reinterpret_cast<const float4*>(row) + member;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float4 x = i < FULL ? p[TEAM * i] : ld_if(p + TEAM * i, i, live);
        v[4 * i] = x.x, v[4 * i + 1] = x.y, v[4 * i + 2] = x.z, v[4 * i + 3] = x.w;
      }
    } else {
      const float* p = row + member;
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] = k < 4 * FULL ? p[TEAM * k] : ld_if(p + TEAM * k, k, live);
    }
  }
  static __device__ __forceinline__ void store(const float (&v)[N], float* row, uint32_t member, uint32_t live) {
    if (VECTOR) {
      float4* p = reinterpret_cast<float4*>(row) + member;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float4 x = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        if (i < FULL) p[TEAM * i] = x;
        else st_if(p + TEAM * i, x, i, live);
      }
    } else {
      float* p = row + member;
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (k < 4 * FULL) p[TEAM * k] = v[k];
        else st_if(p + TEAM * k, v[k], k, live);
    }
  }
};
// The sum over the threads of a team, in every thread and added in the same order in each: lanes side by side, or the CTA, of whose warps' sums each
// thread reads up to eight as vectors (6000 x 500: 7.0 us, by a second round of exchanges 7.4); more are exchanged (400 x 8192: 6.6 us, as vectors
// 8.0).  `slots`: a float for each warp, aligned to 16 bytes and not in use by anything since the last barrier.
template <int TEAM>
__device__ __forceinline__ float team_sum(float v, float* slots) {
  constexpr int kLanes = TEAM < 32 ? TEAM : 32, kWarps = TEAM / 32;
#pragma unroll
  for (int off = kLanes / 2; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  if (kWarps < 2) return v;
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
  __syncthreads();
  if (kWarps == 2) return slots[0] + slots[1];
  if (kWarps > 8) {
    v = slots[threadIdx.x % (kWarps > 8 ? kWarps : 32)];
#pragma unroll
    for (int off = kWarps / 2; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
  }
  Pair s[2] = {0, 0};
#pragma unroll
  for (int w = 0; w < kWarps; w += 4) {
    const float4 f = *reinterpret_cast<const float4*>(slots + w);
    s[0] = add2(s[0], pair(f.x, f.y)), s[1] = add2(s[1], pair(f.z, f.w));
  }
  s[0] = add2(s[0], s[1]);
  return halves(s[0]).x + halves(s[0]).y;
}
// Two sums over the team: each half of the lanes takes one of them, which takes 6 exchanges in a warp where 10 would do both in every lane.  `slots`: two
// floats for each warp.
template <int TEAM>
__device__ __forceinline__ void team_sums(float (&v)[2], float* slots) {
  constexpr int kLanes = TEAM < 32 ? TEAM : 32, kHalf = kLanes / 2, kWarps = TEAM / 32;
  const bool upper = threadIdx.x & kHalf;
  float s = (upper ? v[1] : v[0]) + __shfl_xor_sync(0xffffffffu, upper ? v[0] : v[1], kHalf);
#pragma unroll
  for (int off = kHalf / 2; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
  if (kWarps > 8) {
    if ((threadIdx.x & 15) == 0) slots[(upper ? kWarps : 0) + (threadIdx.x >> 5)] = s;
    __syncthreads();
    const float* mine = slots + (upper ? kWarps : 0) + (threadIdx.x & 15);
    s = kWarps > 16 ? mine[0] + mine[16] : mine[0];
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
  }
  if (kWarps < 2 || kWarps > 8) {
    const float other = __shfl_xor_sync(0xffffffffu, s, kHalf);
    v[0] = upper ? other : s, v[1] = upper ? s : other;
    return;
  }
  if ((threadIdx.x & 15) == 0) slots[threadIdx.x >> 4] = s;   // (a warp's lanes 0 and 16 have one each)
  __syncthreads();
  Pair t[2] = {0, 0};
#pragma unroll
  for (int w = 0; w < 2 * kWarps; w += 4) {
    const float4 f = *reinterpret_cast<const float4*>(slots + w);
    t[0] = add2(t[0], pair(f.x, f.y)), t[1] = add2(t[1], pair(f.z, f.w));
  }
  t[0] = add2(t[0], t[1]);
  v[0] = halves(t[0]).x, v[1] = halves(t[0]).y;
}

// The sums of one or two values over the CTAs of a cluster, added in the same order in each of them; `mine`: for them, not in use by anything else.
template <int CTAS, int N>
__device__ __forceinline__ void cluster_sums(float (&v)[N], double* mine) {
  if (CTAS == 1) return;
  float* own = reinterpret_cast<float*>(mine);
  if (threadIdx.x == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) own[i] = v[i];
  __syncthreads();
  cluster_arrive();
  cluster_wait();
  float part[N][CTAS];
#pragma unroll
  for (int r = 0; r < CTAS; ++r) {
    if (N == 1) {
      part[0][r] = ld_cluster(own, (uint32_t)r);
    } else {                                               // (both by one load: they are what a row waits for)
      const long long both = __double_as_longlong(ld_cluster(mine, (uint32_t)r));
      part[0][r] = __int_as_float((int)both), part[N - 1][r] = __int_as_float((int)(both >> 32));
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = 0.f;
#pragma unroll
    for (int r = 0; r < CTAS; ++r) v[i] += part[i][r];
  }
}

// What the deviations d = x - m from a first mean m leave to do: the mean is m + c and the variance mean(d^2) - c^2 with c = mean(d), which takes the
// first mean's rounding out of both.  (Of a row of 1000.3, whose sum is rounded, (x - m) / sqrt(eps) is 0.02; x - m is the same whole number of
// steps in all of its columns, so c has to be exactly that: the product with 1 / cols is followed by what its rounding left.)
struct Correction {
  float c, var;
  __device__ __forceinline__ Correction(float squares, float deviations, uint32_t cols, float per_col) {
    c = __fmul_rn(deviations, per_col);
    c = __fmaf_rn(__fmaf_rn(-c, (float)cols, deviations), per_col, c);
    var = squares * per_col - fminf(c * c, 3.402823466e38f);   // (an infinite sum of squares stays that)
    if (var < 0.f) var = 0.f;                              // (NaN stays)
  }
};

template <int N>
__device__ __forceinline__ void unpack(float (&v)[N], const Pair (&x)[N / 2]) {
#pragma unroll
  for (int k = 0; k < N / 2; ++k) v[2 * k] = halves(x[k]).x, v[2 * k + 1] = halves(x[k]).y;
}
// A team's row, as its threads have read it (zeros where a thread has no column), as pairs, and its mean but for rounding.
template <int LANES, int CTAS, class S>
__device__ __forceinline__ float first_mean(const float (&v)[S::N], Pair (&x)[S::N / 2], float per_col, float* slots, double* part) {
  Pair sum = 0;
#pragma unroll
  for (int k = 0; k < S::N / 2; ++k) x[k] = pair(v[2 * k], v[2 * k + 1]), sum = add2(sum, x[k]);
  float s[1] = {team_sum<LANES>(halves(sum).x + halves(sum).y, slots)};
  cluster_sums<CTAS>(s, part);
  return __fmul_rn(s[0], per_col);                         // (rounded by itself, as the mean that the deviations are around)
}
// The row's deviations from it, and what their sums leave to correct.
template <int LANES, int CTAS, class S>
__device__ __forceinline__ Correction deviations(Pair (&x)[S::N / 2], float first, uint32_t live, uint32_t cols, float per_col, float* slots, double* part) {
  const Pair minus = pair(-first, -first);
  Pair squares = 0, sum = 0;
#pragma unroll
  for (int k = 0; k < S::N / 2; ++k) {
    x[k] = add2(x[k], minus);
    const float2 d = halves(x[k]);                         // (no column, no deviation)
    if (2 * k >= 4 * S::kFull) x[k] = pair(S::has(live, 2 * k) ? d.x : 0.f, S::has(live, 2 * k + 1) ? d.y : 0.f);
    squares = fma2(x[k], x[k], squares);
    sum = add2(sum, x[k]);
  }
  float s[2] = {halves(squares).x + halves(squares).y, halves(sum).x + halves(sum).y};
  team_sums<LANES>(s, slots);
  cluster_sums<CTAS>(s, part);
  return Correction(s[0], s[1], cols, per_col);
}
template <int N>
__device__ __forceinline__ void normalized(Pair (&x)[N / 2], float c, float rstd) {
  const Pair minus = pair(-c, -c), r = pair(rstd, rstd);
#pragma unroll
  for (int k = 0; k < N / 2; ++k) x[k] = mul2(add2(x[k], minus), r);
}

// Forward, a row in a team's registers: read once, summed twice.  CTAS > 1: a cluster of so many CTAs, as one team.  A CTA's loads, sums and
// stores take turns, so several CTAs have to share an SM: 2048 threads of them with up to 8 elements per thread (300 x 7830: 7.2 us, in two more registers than
// that allows 8.8), else at least 1024 (512 with 32 elements, but for the widest rows: 16384 x 16384 with one CTA of 512 threads on an SM 452 us, with two, in
// 64 registers, 311).
constexpr int resident(int lanes, int v) {
  const int threads = lanes > 32 ? lanes : kThreads, least = v <= 2 ? 2048 : v > 6 && lanes < 512 ? 512 : 1024;
  return least / threads > 1 ? least / threads : 1;
}
template <int LANES, int V, bool VECTOR, int FULL, int CTAS>
__global__ void __launch_bounds__(LANES > 32 ? LANES : kThreads, resident(LANES, V)) norm_rows_kernel(const float* in, const float* gamma, const float* beta, float eps,
                                                                              uint32_t rows, uint32_t cols, float per_col, float* out,
                                                                              float* mean_out, float* rstd_out) {
  using S = Share<LANES * CTAS, V, VECTOR, FULL>;
  constexpr int kBlock = LANES > 32 ? LANES : kThreads;
  __shared__ __align__(16) float slots[kBlock / 8];        // (a warp's: one of the first sum, two of the others, one that aligns these)
  __shared__ double part[2];
  pdl_enter();
  const uint32_t member = blockIdx.y * LANES + threadIdx.x % LANES;   // (blockIdx.y: the CTA's rank in its cluster)
  const uint64_t r = (uint64_t)blockIdx.x * (kBlock / LANES) + threadIdx.x / LANES;
  const uint32_t live = S::live(member, cols);
  float v[S::N];
  S::load(v, in + (r < rows ? r : rows - 1) * cols, member, live);   // (the lanes of a warp stay together, with a row or without)
  Pair x[S::N / 2];
  const float first = first_mean<LANES, CTAS, S>(v, x, per_col, slots, part);
  const Correction by = deviations<LANES, CTAS, S>(x, first, live, cols, per_col, slots + kBlock / 16, part + 1);
  const float mean = first + by.c, rstd = rsqrtf(by.var + eps);
  if (CTAS > 1) cluster_arrive();                          // (nobody leaves while its part may still be read)
  if (r >= rows) return;                                   // (of a cluster, all or none)
  normalized<S::N>(x, by.c, rstd);
  if (gamma) {
    S::load(v, gamma, member, live);
#pragma unroll
    for (int k = 0; k < S::N / 2; ++k) x[k] = mul2(x[k], pair(v[2 * k], v[2 * k + 1]));
  }
  if (beta) {
    S::load(v, beta, member, live);
#pragma unroll
    for (int k = 0; k < S::N / 2; ++k) x[k] = add2(x[k], pair(v[2 * k], v[2 * k + 1]));
  }
  unpack<S::N>(v, x);
  S::store(v, out + r * cols, member, live);
  if (member == 0) {
    if (mean_out) mean_out[r] = mean;
    if (rstd_out) rstd_out[r] = rstd;
  }
  if (CTAS > 1) cluster_wait();
}

// ---- rows through shared memory -----------------------------------------------------------------------
template <int BYTES>
__device__ __forceinline__ void copy_async(void* to, const float* from, uint32_t bytes) {   // (zeros behind `bytes`)
  const uint32_t dst = (uint32_t)__cvta_generic_to_shared(to);
  if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(from), "r"(bytes) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

// Rows that do not begin on 16-byte boundaries are copied as they lie, vectors from the boundary before their beginning on: how far a row begins
// past a boundary, and the copies that one of LANES threads makes of up to 4 V LANES floats.
__device__ __forceinline__ uint32_t past(const float* p) { return (uint32_t)(reinterpret_cast<uintptr_t>(p) >> 2) & 3; }
template <int LANES, int V>
__device__ __forceinline__ void copy_image(float* to, const float* src, uint32_t count, uint32_t member) {
  const uint32_t shift = past(src);
#pragma unroll
  for (int j = 0; j <= V; ++j) {                           // (a row that begins past a boundary has a vector more)
    const uint32_t i = member + LANES * j;
    const int left = 4 * (int)(shift + count) - 16 * (int)i;
    if (left <= 0 || (j == V && member)) continue;
    if (j == 0 && i == 0 && shift) {
      for (uint32_t k = shift; k < 4 && k < shift + count; ++k) copy_async<4>(to + k, src + (k - shift), 4);
    } else {
      copy_async<16>(to + 4 * i, src + (int64_t)(4 * i) - shift, left < 16 ? left : 16);
    }
  }
}

// Forward, long rows that are not on 16-byte boundaries: an SM's CTAs stay and go through the rows with gamma and beta in their registers; two
// rows are on their way while one is computed (8000 x 9001: 123 us, a cluster of two CTAs per row 271; 16384 x 16383: 362 and
// 681; 8007 x 7830: 90, a CTA per row 101; 60000 x 2101: 173 and 217).
// HELD: gamma and beta are in registers; of rows beyond 16384 columns they are read for each row, and one row is on its way (5294 x 17287: 188 us, a
// cluster of four CTAs per row 412; 300 x 17287 16.6 and 23.1).
template <int LANES, int V, int FULL, bool HELD>
__global__ void __launch_bounds__(LANES, LANES < 512 ? 512 / LANES : 1)
    norm_ring_kernel(const float* in, const float* gamma, const float* beta, float eps, uint32_t rows, uint32_t cols, float per_col, float* out,
                     float* mean_out, float* rstd_out) {
  constexpr int N = 4 * V, kImage = LANES * N + 4, kRing = HELD ? 3 : 2;
  using S = Share<LANES, V, false, FULL>;                  // (cols > 4 LANES FULL)
  extern __shared__ float4 images[];
  __shared__ __align__(16) float slots[LANES / 8];
  pdl_enter();
  float* ring = reinterpret_cast<float*>(images);
  const uint32_t member = threadIdx.x, live = S::live(member, cols);
  uint64_t r = blockIdx.x, fetched = r;
  uint32_t to_stage = 0, stage = 0;
  auto fetch = [&] {
    if (fetched < rows) copy_image<LANES, V>(ring + to_stage * kImage, in + fetched * cols, cols, member);
    copies_end();                                          // (an empty group as well: a group for each row)
    fetched += gridDim.x;
    to_stage = to_stage + 1 == kRing ? 0 : to_stage + 1;
  };
#pragma unroll
  for (int s = 0; s < kRing - 1; ++s) fetch();
  Pair g[HELD ? N / 2 : 1], b[HELD ? N / 2 : 1];
  if constexpr (HELD) {
    float w[N];
#pragma unroll
    for (int k = 0; k < N; ++k) w[k] = 1.f;
    if (gamma) S::load(w, gamma, member, live);
#pragma unroll
    for (int k = 0; k < N / 2; ++k) g[k] = pair(w[2 * k], w[2 * k + 1]);
#pragma unroll
    for (int k = 0; k < N; ++k) w[k] = 0.f;
    if (beta) S::load(w, beta, member, live);
#pragma unroll
    for (int k = 0; k < N / 2; ++k) b[k] = pair(w[2 * k], w[2 * k + 1]);
  }
  for (; r < rows; r += gridDim.x) {
    copies_wait<kRing - 2>();
    __syncthreads();                                       // what other threads have copied is here, and all have read the row before
    float v[N];
    const float* p = ring + stage * kImage + past(in + r * cols) + member;
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = S::has(live, k) ? p[LANES * k] : 0.f;
    fetch();
    Pair x[N / 2];
    const float first = first_mean<LANES, 1, S>(v, x, per_col, slots, nullptr);
    const Correction by = deviations<LANES, 1, S>(x, first, live, cols, per_col, slots + LANES / 16, nullptr);
    const float mean = first + by.c, rstd = rsqrtf(by.var + eps);
    normalized<N>(x, by.c, rstd);
    if constexpr (HELD) {
#pragma unroll
      for (int k = 0; k < N / 2; ++k) x[k] = fma2(x[k], g[k], b[k]);
      unpack<N>(v, x);
    } else {
      unpack<N>(v, x);
      if (gamma) {
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] *= k < 4 * FULL ? gamma[member + LANES * k] : ld_if(gamma + member + LANES * k, k, live);
      }
      if (beta) {
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] += k < 4 * FULL ? beta[member + LANES * k] : ld_if(beta + member + LANES * k, k, live);
      }
    }
    S::store(v, out + r * cols, member, live);
    if (member == 0) {
      if (mean_out) mean_out[r] = mean;
      if (rstd_out) rstd_out[r] = rstd;
    }
    stage = stage + 1 == kRing ? 0 : stage + 1;
  }
}

// The sums of two terms over the elements that a thread has of a row, kThreads apart: up to 32 of them in 32 bits, these sums in 64.  In 32 bits alone the
// rounding would grow with the row (from 2^20 columns on a sum loses a part of each term); in 64 alone the conversions take half as long again as all the rest
// (1000 x 100000: 549 us, so 371).
template <class Terms>
__device__ __forceinline__ void long_sums(uint64_t cols, float (&s)[2], Terms terms) {
  double own[2] = {0., 0.};
  float part[2] = {0.f, 0.f};
  uint64_t c = threadIdx.x;
  for (uint32_t n = 1; c + 3 * kThreads < cols; c += 4 * kThreads, ++n) {
#pragma unroll
    for (int k = 0; k < 4; ++k) terms(c + k * kThreads, part);
    if (n % 8 == 0) {
      own[0] += (double)part[0], own[1] += (double)part[1];
      part[0] = part[1] = 0.f;
    }
  }
  for (; c < cols; c += kThreads) terms(c, part);
  own[0] += (double)part[0], own[1] += (double)part[1];
  s[0] = (float)own[0], s[1] = (float)own[1];
}

// Rows of any length: three passes over a row that the caches hold.
__global__ void __launch_bounds__(kThreads) norm_kernel(const float* in, const float* gamma, const float* beta, float eps,
                                                        uint64_t cols, float* out, float* mean_out, float* rstd_out) {
  pdl_enter();
  __shared__ float slots[2][2 * kThreads / 32];
  const float* x = in + blockIdx.x * cols;
  float s[2];
  long_sums(cols, s, [&](uint64_t c, float (&part)[2]) { part[0] += x[c]; });
  block_sums<kThreads>(s, slots[0]);
  const float first = s[0] / (float)cols;
  long_sums(cols, s, [&](uint64_t c, float (&part)[2]) {
    const float d = x[c] - first;
    part[0] += d * d, part[1] += d;
  });
  block_sums<kThreads>(s, slots[1]);
  const Correction by(s[0], s[1], (uint32_t)cols, 1.f / (float)cols);
  const float mean = first + by.c, rstd = rsqrtf(by.var + eps);
  for (uint64_t c = threadIdx.x; c < cols; c += kThreads)
    out[blockIdx.x * cols + c] = ((x[c] - first) - by.c) * rstd * (gamma ? gamma[c] : 1.f) + (beta ? beta[c] : 0.f);
  if (threadIdx.x == 0) {
    if (mean_out) mean_out[blockIdx.x] = mean;
    if (rstd_out) rstd_out[blockIdx.x] = rstd;
  }
}

// ---- backward ---------------------------------------------------------------------------------------
// One pass over the rows: a team walks over rows (its CTA or cluster, over every gridDim.x-th group of them), the weights' gradients of its
// columns in registers (65536 x 4096: 520 us, 6.2 TB/s; 2001 x 1511, a few rows to a team: 12.5).  The rows come through a ring in shared memory,
// STAGES - 1 of them on their way while one is computed, by asynchronous copies that each thread makes and waits for by itself: what it copies is what it reads, so no barrier is needed but the one of the row's sums.
// The sums over the team's rows go to `partials` [CTAs or clusters][2][cols], which a second kernel adds in order.
// Threads of a CTA: several teams where they are small, as many as an SM's registers take.
constexpr int block_of(int lanes) { return lanes == 96 || lanes == 160 ? 480 : lanes == 224 ? 448 : lanes > kThreads ? lanes : kThreads; }
template <int LANES>
constexpr int kBlockOf = block_of(LANES);
// A barrier of a team and the sums over it, in every thread, where several teams share a CTA (`group`: the team's number; `slots`: 2 for each warp).
template <int LANES>
__device__ __forceinline__ void team_barrier(uint32_t group) {
  if (LANES <= 32) __syncwarp();
  else if (LANES >= kThreads) __syncthreads();
  else asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(LANES) : "memory");
}
template <int LANES>
__device__ __forceinline__ void grad_sums(float (&v)[2], float* slots, uint32_t group) {
  constexpr int kWarps = LANES / 32;
#pragma unroll
  for (int off = (LANES < 32 ? LANES : 32) / 2; off > 0; off >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], off), v[1] += __shfl_xor_sync(0xffffffffu, v[1], off);
  if (LANES <= 32) return;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) slots[2 * warp] = v[0], slots[2 * warp + 1] = v[1];
  team_barrier<LANES>(group);
  const float* mine = slots + 2 * group * kWarps;
  v[0] = lane < kWarps ? mine[2 * lane] : 0.f, v[1] = lane < kWarps ? mine[2 * lane + 1] : 0.f;
#pragma unroll
  for (int off = kWarps > 8 ? 8 : kWarps > 4 ? 4 : kWarps > 2 ? 2 : 1; off > 0; off >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], off), v[1] += __shfl_xor_sync(0xffffffffu, v[1], off);
  v[0] = __shfl_sync(0xffffffffu, v[0], 0), v[1] = __shfl_sync(0xffffffffu, v[1], 0);
}
template <int LANES, int V, bool VECTOR, int CTAS, int STAGES>
__global__ void __launch_bounds__(kBlockOf<LANES>, 512 / kBlockOf<LANES>) norm_grad_rows_kernel(
    const float* gradient, const float* in, const float* gamma, const float* mean, const float* rstd, uint32_t rows, uint32_t cols, float per_col,
    float* din, float* partials) {
  constexpr int kBlock = kBlockOf<LANES>, kGroups = kBlock / LANES, N = 4 * V;
  // (a team has columns for more than half of its places, so half of the fours are full, except for a cluster's last CTA and the shortest rows)
  constexpr int FULL = CTAS == 1 ? V / 2 : 0;
  using S = Share<LANES, V, VECTOR, FULL>;
  // VECTOR: [STAGES][gradient, in][V][kBlock] vectors, of which a thread copies and reads its own.  Else rows are copied as they lie, vectors from
  // the boundary before their beginning on, and read as single floats by other threads than copied them: [STAGES][gradient, in][kGroups][kImage].
  constexpr int kImage = LANES * N + 4;
  extern __shared__ float4 ring4[];
  __shared__ float slots[2][2 * kBlock / 32], part[2][2];
  pdl_enter();
  float* ring = reinterpret_cast<float*>(ring4);
  const uint32_t tid = threadIdx.x, group = tid / LANES, member = tid % LANES;
  // the CTA's part of the columns, and how many this thread has of it
  const uint32_t from = blockIdx.y * (LANES * N), here = from < cols ? min(cols - from, (uint32_t)(LANES * N)) : 0, live = S::live(member, here);
  const uint32_t groups = (rows + kGroups - 1) / kGroups, trips = (groups - blockIdx.x + gridDim.x - 1) / gridDim.x;
  uint64_t r = (uint64_t)blockIdx.x * kGroups + group;
  const uint64_t step = (uint64_t)gridDim.x * kGroups;
  // where the fetches are: the row, its places, the stage
  uint64_t fetched = r;
  const float *src_g = gradient + r * cols + from, *src_x = in + r * cols + from;
  uint32_t to_stage = 0;
  auto image = [&](uint32_t stage, int which) { return ring + ((stage * 2 + which) * kGroups + group) * kImage; };
  auto fetch = [&] {
    if (fetched < rows) {
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        const float* src = which ? src_x : src_g;
        if (VECTOR) {
          src += 4 * member;
#pragma unroll
          for (int i = 0; i < V; ++i)
            copy_async<16>(ring4 + ((to_stage * 2 + which) * V + i) * kBlock + tid, S::has(live, 4 * i) ? src + 4 * LANES * i : gradient,
                           S::has(live, 4 * i) ? 16 : 0);
        } else {
          copy_image<LANES, V>(image(to_stage, which), src, here, member);
        }
      }
    }
    copies_end();                                          // (an empty group as well: the count of groups is the count of trips)
    fetched += step, src_g += step * cols, src_x += step * cols;
    to_stage = to_stage + 1 == STAGES ? 0 : to_stage + 1;
  };
  auto read_stage = [&](float (&v)[N], uint32_t stage, int which) {
    if (r >= rows) {                                       // no row: of a warp's last groups
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] = 0.f;
    } else if (VECTOR) {
#pragma unroll
      for (int i = 0; i < V; ++i) *reinterpret_cast<float4*>(v + 4 * i) = ring4[((stage * 2 + which) * V + i) * kBlock + tid];
    } else {
      const float* p = image(stage, which) + past((which ? in : gradient) + r * cols + from) + member;
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] = S::has(live, k) ? p[LANES * k] : 0.f;
    }
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) fetch();
  float g[N];
#pragma unroll
  for (int k = 0; k < N; ++k) g[k] = 1.f;
  if (gamma) S::load(g, gamma + from, member, live);
  Pair gamma2[N / 2], dgamma[N / 2], dbeta[N / 2];
#pragma unroll
  for (int k = 0; k < N / 2; ++k) gamma2[k] = pair(g[2 * k], g[2 * k + 1]), dgamma[k] = dbeta[k] = 0;
  float m = r < rows ? mean[r] : 0.f, s = r < rows ? rstd[r] : 0.f;
  uint32_t stage = 0;
  const Pair one = pair(1.f, 1.f);
  for (uint32_t trip = 0; trip < trips; ++trip) {
    copies_wait<STAGES - 2>();
    if (!VECTOR) {                                         // what other threads have copied, and their reads of the trip before
      team_barrier<LANES>(group);
    }
    float v[N];
    Pair dy[N / 2], h[N / 2];
    read_stage(v, stage, 0);
#pragma unroll
    for (int k = 0; k < N / 2; ++k) dy[k] = pair(v[2 * k], v[2 * k + 1]);
    read_stage(v, stage, 1);
#pragma unroll
    for (int k = 0; k < N / 2; ++k) h[k] = pair(v[2 * k], v[2 * k + 1]);
    fetch();                                               // (into the stage of the trip before, which has been read)
    const uint64_t next = r + step;
    const float next_m = next < rows ? mean[next] : 0.f, next_s = next < rows ? rstd[next] : 0.f;
    const Pair minus_m = pair(-m, -m), s2 = pair(s, s);
    Pair sum_q = 0, sum_qh = 0;
#pragma unroll
    for (int k = 0; k < N / 2; ++k) {                      // (sums of pairs as 1 * a + b)
      h[k] = mul2(fma2(one, h[k], minus_m), s2);
      dgamma[k] = fma2(dy[k], h[k], dgamma[k]);
      dbeta[k] = fma2(one, dy[k], dbeta[k]);
      dy[k] = mul2(dy[k], gamma2[k]);
      sum_q = fma2(one, dy[k], sum_q);
      sum_qh = fma2(dy[k], h[k], sum_qh);
    }
    float sums[2] = {halves(sum_q).x + halves(sum_q).y, halves(sum_qh).x + halves(sum_qh).y};
    grad_sums<LANES>(sums, slots[trip & 1], group);        // (a barrier lies between the reads of one trip and the writes of the next but one)
    if (CTAS > 1) {
      float* mine = part[trip & 1];
      if (tid == 0) mine[0] = sums[0], mine[1] = sums[1];
      cluster_arrive();
      cluster_wait();
      float p[2][CTAS];
#pragma unroll
      for (int c = 0; c < CTAS; ++c) p[0][c] = ld_cluster(mine, (uint32_t)c), p[1][c] = ld_cluster(mine + 1, (uint32_t)c);
      sums[0] = sums[1] = 0.f;
#pragma unroll
      for (int c = 0; c < CTAS; ++c) sums[0] += p[0][c], sums[1] += p[1][c];
    }
    const float a = sums[0] * per_col, b = sums[1] * per_col;
    const Pair minus_a = pair(-a, -a), minus_b = pair(-b, -b);
#pragma unroll
    for (int k = 0; k < N / 2; ++k) {
      const float2 d = halves(mul2(fma2(h[k], minus_b, fma2(one, dy[k], minus_a)), s2));
      v[2 * k] = d.x, v[2 * k + 1] = d.y;
    }
    if (r < rows) S::store(v, din + r * cols + from, member, live);
    r = next, m = next_m, s = next_s;
    stage = stage + 1 == STAGES ? 0 : stage + 1;
  }
  if (partials) {
    float* to = partials + 2ull * blockIdx.x * cols + from;
    auto unpack = [&](const Pair (&p)[N / 2]) {
#pragma unroll
      for (int k = 0; k < N / 2; ++k) g[2 * k] = halves(p[k]).x, g[2 * k + 1] = halves(p[k]).y;
    };
    if (kGroups == 1) {
      unpack(dgamma);
      S::store(g, to, member, live);
      unpack(dbeta);
      S::store(g, to + cols, member, live);
    } else {                                               // the groups' sums meet in the ring: [dGamma, dBeta][groups][columns]
      constexpr int kWidth = LANES * N;
      copies_wait<0>();
      __syncthreads();
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        unpack(which ? dbeta : dgamma);
#pragma unroll
        for (int k = 0; k < N; ++k)
          ring[(which * kGroups + group) * kWidth + (VECTOR ? 4 * (member + LANES * (k / 4)) + k % 4 : member + LANES * k)] = g[k];
      }
      __syncthreads();
      for (uint32_t c = tid; c < cols; c += kBlock) {
        float sum[2] = {0.f, 0.f};
        for (int q = 0; q < kGroups; ++q) sum[0] += ring[q * kWidth + c], sum[1] += ring[(kGroups + q) * kWidth + c];
        to[c] = sum[0], to[(uint64_t)cols + c] = sum[1];
      }
    }
  }
  if (CTAS > 1) {                                          // nobody leaves while its part may still be read
    cluster_arrive();
    cluster_wait();
  }
}

// Backward, rows of any length: the gradient at the input.
__global__ void __launch_bounds__(kThreads) norm_grad_in_kernel(const float* gradient, const float* in, const float* gamma,
                                                                const float* mean, const float* rstd, uint64_t cols, float* din) {
  pdl_enter();
  __shared__ float slots[2 * kThreads / 32];
  const uint64_t at = blockIdx.x * cols;
  const float m = mean[blockIdx.x], r = rstd[blockIdx.x];
  float s[2];
  long_sums(cols, s, [&](uint64_t c, float (&part)[2]) {
    const float q = gradient[at + c] * (gamma ? gamma[c] : 1.f);
    part[0] += q, part[1] += q * ((in[at + c] - m) * r);
  });
  block_sums<kThreads>(s, slots);
  const float a = s[0] / (float)cols, b = s[1] / (float)cols;
  for (uint64_t c = threadIdx.x; c < cols; c += kThreads) {
    const float q = gradient[at + c] * (gamma ? gamma[c] : 1.f), h = (in[at + c] - m) * r;
    din[at + c] = r * (q - a - h * b);
  }
}

// Backward, rows of any length: the weights' gradients summed over a stretch of rows, a thread per column.
__global__ void __launch_bounds__(kThreads) norm_grad_columns_kernel(const float* gradient, const float* in, const float* mean,
                                                                     const float* rstd, uint64_t rows, uint64_t cols,
                                                                     uint64_t stretch, float* partials) {
  pdl_enter();
  const uint64_t c = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
  if (c >= cols) return;
  float dg = 0.f, db = 0.f;
  const uint64_t first = blockIdx.y * stretch, end = first + stretch < rows ? first + stretch : rows;
  for (uint64_t r = first; r < end; ++r) {
    const float g = gradient[r * cols + c];
    dg += g * ((in[r * cols + c] - mean[r]) * rstd[r]);
    db += g;
  }
  partials[(2ull * blockIdx.y) * cols + c] = dg;
  partials[(2ull * blockIdx.y + 1) * cols + c] = db;
}

// The partial sums of `parts` stretches of rows: COLS columns to a CTA, every (1024 / COLS)th part to a thread, then the threads' sums by columns.
constexpr int kFinishThreads = 1024;
template <int COLS>
__global__ void __launch_bounds__(kFinishThreads) norm_grad_finish_kernel(const float* partials, uint32_t parts, uint64_t cols, float* dgamma,
                                                                          float* dbeta) {
  constexpr int kRows = kFinishThreads / COLS;
  __shared__ float tile[kRows][COLS + 1];
  pdl_enter();
  float* out = blockIdx.y ? dbeta : dgamma;
  if (!out) return;
  const uint32_t row = threadIdx.x / COLS, col = threadIdx.x % COLS;
  const uint64_t c = (uint64_t)blockIdx.x * COLS + col;
  float s = 0.f;
  if (c < cols) {
    const float* q = partials + (2ull * row + blockIdx.y) * cols + c;
    const uint64_t step = 2ull * kRows * cols;             // two rows of sums for each part
#pragma unroll 8
    for (uint32_t p = row; p < parts; p += kRows, q += step) s += *q;   // (eight loads on their way)
  }
  tile[row][col] = s;
  __syncthreads();
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp >= COLS) return;
  s = 0.f;
#pragma unroll
  for (int r = 0; r < kRows; r += 32) s += tile[r + lane][warp];
  s = warp_sum(s);
  if (lane == 0 && (uint64_t)blockIdx.x * COLS + warp < cols) out[(uint64_t)blockIdx.x * COLS + warp] = s;
}

constexpr uint64_t kMaxCols = 1ull << 31, kMaxRows = 0x7fffffffull;

// Stretches of rows whose sums are kept apart, for rows beyond the one-pass kernel.
uint64_t stretches(uint64_t rows) {
  const uint64_t n = (rows + 63) / 64;
  return n < 256 ? n : 256;
}

// How the one-pass kernel runs a shape: lanes and CTAs of a team (lanes 0: not at all), fours per thread, and CTAs or clusters in all.
constexpr int kStages = 3;
constexpr uint64_t kOnePassCols = 65536;
struct GradPlan {
  unsigned lanes, v, ctas, grid;
};
GradPlan grad_plan(uint64_t rows, uint64_t cols, bool vectors) {
  if (cols > kOnePassCols) return GradPlan{0, 0, 0, 0};
  GradPlan p{8, 4, 1, 0};
  if (cols <= 32) p.v = 1;
  else if (cols <= 64) p.v = 2;
  while ((uint64_t)p.lanes * p.v * 4 < cols && p.lanes < 512) p.lanes *= 2;
  // Rows that are read as single floats pay for every place of a team that has no column, so theirs are teams of any number of warps (65536 x 1511:
  // 193 us in five teams of 96 lanes, 222 in four of 128; 30000 x 2101 138 and 193; 10000 x 5001 133 and 155; where rows are vectors smaller CTAs are
  // better: 65536 x 1280 153 and, in teams of 96, 163).  Few rows take more, smaller CTAs (40 x 1511: 5.2, 6.4).
  const uint64_t sms = (uint64_t)sm_count();
  if (!vectors && rows > 2 * sms)
    for (const unsigned lanes : {96u, 160u, 224u, 320u, 384u, 448u})
      if (p.lanes > lanes && p.lanes < 2 * lanes && cols <= lanes * 16) {
        p.lanes = lanes;
        break;
      }
  if (cols > 8192) {
    p.lanes = cols <= 32768 ? 256 : 512;
    p.ctas = (unsigned)((cols + p.lanes * p.v * 4 - 1) / (p.lanes * p.v * 4));
  }
  // 512 threads on an SM, with three stages of up to 64 KB; where there are many rows, some for each CTA, so that the partial sums are few beside
  // them (3 x 7560: 7.2 us with a CTA per row, 8.5 with one for two)
  const uint64_t block = block_of((int)p.lanes), teams = block / p.lanes, groups = (rows + teams - 1) / teams;
  const uint64_t most = sms * (512 / block) / p.ctas, wanted = groups <= sms ? groups : (groups + 1) / 2;
  p.grid = (unsigned)(wanted < most ? wanted : most);
  return p;
}

// How many of a kernel's clusters a device holds at a time: fewer than SMs by CTAs, as a cluster lies within a GPC.  A property of the device and the
// kernel, asked for once.
template <auto KERNEL>
unsigned resident_clusters(unsigned threads, size_t bytes, unsigned ctas, unsigned most) {
  constexpr int kDevices = 64;
  static std::atomic<unsigned> known[kDevices];
  int device = 0, n = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= kDevices) return most * 3 / 4;
  if (const unsigned before = known[device].load(std::memory_order_relaxed)) return before;
  cudaLaunchConfig_t c = {};
  c.gridDim = dim3(most, ctas);
  c.blockDim = dim3(threads);
  c.dynamicSmemBytes = bytes;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = 1, at[0].val.clusterDim.y = ctas, at[0].val.clusterDim.z = 1;
  c.attrs = at;
  c.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(&n, KERNEL, &c) != cudaSuccess || n < 1) {
    cudaGetLastError();
    return most * 3 / 4;
  }
  known[device].store((unsigned)n, std::memory_order_relaxed);
  return (unsigned)n;
}

template <int LANES, int V, bool VECTOR, int CTAS>
int launch_grad_rows(GradPlan& p, cudaStream_t st, const float* gradient, const float* in, const float* gamma, const float* mean,
                     const float* rstd, uint64_t rows, uint64_t cols, float* din, float* partials) {
  constexpr auto kernel = norm_grad_rows_kernel<LANES, V, VECTOR, CTAS, kStages>;
  constexpr size_t bytes = (size_t)kStages * 2 * (4 * V * LANES + (VECTOR ? 0 : 4)) * (kBlockOf<LANES> / LANES) * sizeof(float);
  if (bytes > 48 * 1024 - 1024) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e != cudaSuccess) return fail(POLAR_B200_ERR_CUDA, "cudaFuncSetAttribute(flayernorm_grad)", e);
  }
  if (CTAS > 1) p.grid = std::max(1u, std::min(p.grid, resident_clusters<kernel>(kBlockOf<LANES>, bytes, CTAS, p.grid)));
  return launch_clusters("flayernorm_grad", kernel, dim3(p.grid, CTAS), kBlockOf<LANES>, bytes, st, CTAS, gradient, in, gamma, mean, rstd, (uint32_t)rows,
                         (uint32_t)cols, (float)(1.0 / (double)cols), din, partials);
}

}  // namespace
}  // namespace polar_b200

using namespace polar_b200;

extern "C" {

int polar_b200_flayernorm(const float* in, const float* gamma, const float* beta, float eps, uint64_t rows, uint64_t cols,
                          float* out, float* mean, float* rstd, void* stream) {
  clear_error();
  if (!(eps >= 0.f)) return fail(POLAR_B200_ERR_INVALID, "flayernorm: eps must not be negative");
  if (rows == 0 || cols == 0) return POLAR_B200_OK;
  if (rows > kMaxRows || cols > kMaxCols) return fail(POLAR_B200_ERR_INVALID, "flayernorm: too many rows or columns");
  if (!in || !out) return fail(POLAR_B200_ERR_INVALID, "null device pointer");
  LaunchDeviceScope on(stream, out);
  const bool vectors = (cols & 3) == 0 && aligned16(in) && aligned16(out) && aligned16(gamma) && aligned16(beta);
  cudaStream_t st = as_stream(stream);
  auto go = [&](auto with, auto without, unsigned lanes, unsigned ctas) {
    const unsigned per_cta = lanes > 32 ? 1 : kThreads / lanes;
    return launch_clusters("flayernorm", vectors ? with : without, dim3((unsigned)((rows + per_cta - 1) / per_cta), ctas),
                           lanes > 32 ? lanes : kThreads, 0, st, ctas, in, gamma, beta, eps, (uint32_t)rows, (uint32_t)cols, (float)(1.0 / (double)cols), out, mean, rstd);
  };
#define ROWS(LANES, V, FULL, CTAS) go(norm_rows_kernel<LANES, V, true, FULL, CTAS>, norm_rows_kernel<LANES, V, false, FULL, CTAS>, LANES, CTAS)
#define VECTORS(LANES, V, FULL, CTAS) go(norm_rows_kernel<LANES, V, true, FULL, CTAS>, norm_rows_kernel<LANES, V, true, FULL, CTAS>, LANES, CTAS)
#define FLOATS(LANES, V, FULL, CTAS) go(norm_rows_kernel<LANES, V, false, FULL, CTAS>, norm_rows_kernel<LANES, V, false, FULL, CTAS>, LANES, CTAS)
// (12 and 16 elements to a thread: rows that are vectors are a warp's from 516 to 1024 columns and take 24 or 32 from 4096, so 64 and 512 lanes are
// for single floats; of these, rows of up to 6144 columns that are many enough for 512 lanes are enough for the ring)
#define LANES_OF(V, WITH_64, WITH_512)          \
  switch (lanes) {                              \
    case 8: return ROWS(8, V, V - 1, 1);        \
    case 16: return ROWS(16, V, V - 1, 1);      \
    case 32: return ROWS(32, V, V - 1, 1);      \
    case 64: return WITH_64(64, V, V - 1, 1);   \
    case 128: return ROWS(128, V, V - 1, 1);    \
    case 256: return ROWS(256, V, V - 1, 1);    \
    default: return WITH_512;                   \
  }
  // How many elements a thread takes: 4 where there are few rows, for the shortest chain; 8 while the threads do not fill the SMs; then 16 and,
  // of long rows, 32, whose loads are all in flight at once (20000 x 5000 120 us, with 16 140; 20000 x 8192 189 and
  // 218; at 4096 columns either: 65536 rows 310 and 305, 2048 rows 9.2 and 9.7).
  const uint64_t sms = (uint64_t)sm_count();
  // (The number of elements per thread that a form is made for is its V: FULL fours of every thread are there without asking, so each form serves
  // cols > 4 LANES CTAS FULL only.)
  auto ring = [&](auto kernel, unsigned threads, unsigned v) {
    const size_t bytes = (threads > 512 ? 2 : 3) * (size_t)(threads * v * 4 + 4) * sizeof(float);
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e != cudaSuccess) return fail(POLAR_B200_ERR_CUDA, "cudaFuncSetAttribute(flayernorm)", e);
    const uint64_t most = sms * (threads < 512 ? 512 / threads : 1);
    return launch("flayernorm", kernel, dim3((unsigned)(rows < most ? rows : most)), threads, bytes, st, in, gamma, beta, eps, (uint32_t)rows,
                  (uint32_t)cols, (float)(1.0 / (double)cols), out, mean, rstd);
  };
  // (once every SM has its CTAs, and four rows for each of the smaller ones: 600 x 7830 9.4 us, a CTA per row 9.8; 3000 x 2501 11.5 and 12.2; up to
  // 2048 columns loads into registers do as well)
  if (!vectors && cols > 2048 && cols <= 16384 && rows >= (cols <= 4096 ? 16 : 4) * sms) {
    if (cols <= 4096) return cols <= 128 * 24 ? ring(norm_ring_kernel<128, 6, 4, true>, 128, 6) : ring(norm_ring_kernel<128, 8, 6, true>, 128, 8);
    if (cols <= 8192) return cols <= 256 * 24 ? ring(norm_ring_kernel<256, 6, 4, true>, 256, 6) : ring(norm_ring_kernel<256, 8, 6, true>, 256, 8);
    return cols <= 512 * 24 ? ring(norm_ring_kernel<512, 6, 4, true>, 512, 6) : ring(norm_ring_kernel<512, 8, 6, true>, 512, 8);
  }
  if (!vectors && cols > 16384 && cols <= 1024 * 28 && rows >= 2 * sms)   // (two rows fill the shared memory)
    return cols <= 1024 * 20   ? ring(norm_ring_kernel<1024, 5, 4, false>, 1024, 5)
           : cols <= 1024 * 24 ? ring(norm_ring_kernel<1024, 6, 5, false>, 1024, 6)
                               : ring(norm_ring_kernel<1024, 7, 6, false>, 1024, 7);
  auto any_length = [&] {
    return launch("flayernorm", norm_kernel, dim3((unsigned)rows), kThreads, 0, st, in, gamma, beta, eps, cols, out, mean, rstd);
  };
  const bool few = rows <= 2 * sms, little = rows * cols < (4ull << 20);
  if (cols <= 8192) {
    const unsigned each = few && cols <= 4096 ? 4 : little ? 8 : vectors && cols >= 4096 ? 32 : 16;
    if (vectors && !little && cols > 512 && cols <= 1024) return cols <= 640 ? VECTORS(32, 5, 4, 1) : cols <= 768 ? VECTORS(32, 6, 5, 1) : VECTORS(32, 8, 6, 1);
    unsigned lanes = 8;
    while (lanes * each < cols) lanes *= 2;
    const unsigned v = (unsigned)((cols + lanes - 1) / lanes + 3) / 4;
    if (v > 4) return lanes == 128 ? VECTORS(128, 8, 6, 1) : v > 6 ? VECTORS(256, 8, 6, 1) : VECTORS(256, 6, 4, 1);
    if (lanes == 1024) return v == 1 ? ROWS(1024, 1, 0, 1) : ROWS(1024, 2, 1, 1);
    if (v == 1) LANES_OF(1, ROWS, ROWS(512, 1, 0, 1))
    if (v == 2) LANES_OF(2, ROWS, ROWS(512, 2, 1, 1))
    if (v == 3) LANES_OF(3, FLOATS, any_length())
    LANES_OF(4, FLOATS, FLOATS(512, 4, 3, 1))
  }
  // Longer ones: a large CTA, clusters of CTAs where the row is beyond one or, as single floats, beyond its registers, and smaller shares in
  // larger clusters for up to nine rows, half of the SMs (1 x 32768: 4.0 us, one CTA 6.4; 10 x 32768 5.9 and 6.5; 10 x 20000 5.4 and 5.1; 18 x 32768 8.3
  // and 6.6).
  if (rows * 16 <= sms && cols > 16384 && cols <= 32768) return ROWS(512, 2, 0, 8);
  if (!vectors && cols <= 65536) return cols <= 16384 ? FLOATS(512, 4, 2, 2) : cols <= 32768 ? FLOATS(512, 4, 2, 4) : FLOATS(512, 4, 2, 8);
  if (cols <= 16384) return VECTORS(512, 8, 4, 1);
  if (cols <= 32768) return VECTORS(1024, 8, 4, 1);
  if (cols <= 65536) return VECTORS(1024, 8, 4, 2);
#undef LANES_OF
#undef FLOATS
#undef VECTORS
#undef ROWS
  return any_length();
}

uint64_t polar_b200_flayernorm_grad_workspace_bytes(uint64_t rows, uint64_t cols) {
  if (rows == 0 || cols == 0 || rows > kMaxRows || cols > kMaxCols) return 0;
  const unsigned grid = std::max(grad_plan(rows, cols, true).grid, grad_plan(rows, cols, false).grid);   // (where the tensors lie is not known yet)
  return (grid ? grid : stretches(rows)) * 2 * cols * sizeof(float);
}

int polar_b200_flayernorm_grad(const float* gradient, const float* in, const float* gamma, const float* mean, const float* rstd,
                               uint64_t rows, uint64_t cols, float* din, float* dgamma, float* dbeta, void* workspace,
                               uint64_t workspace_bytes, void* stream) {
  clear_error();
  if (cols == 0) return POLAR_B200_OK;
  if (rows > kMaxRows || cols > kMaxCols) return fail(POLAR_B200_ERR_INVALID, "flayernorm_grad: too many rows or columns");
  if (rows == 0) {                                         // empty sums
    int rc = dgamma ? polar_b200_ffill(0.f, dgamma, cols, stream) : POLAR_B200_OK;
    if (rc == POLAR_B200_OK && dbeta) rc = polar_b200_ffill(0.f, dbeta, cols, stream);
    return rc;
  }
  if (!gradient || !in || !mean || !rstd || !din) return fail(POLAR_B200_ERR_INVALID, "null device pointer");
  LaunchDeviceScope on(stream, din);
  cudaStream_t st = as_stream(stream);
  int rc = POLAR_B200_OK;
  const bool vectors = (cols & 3) == 0 && aligned16(gradient) && aligned16(in) && aligned16(gamma) && aligned16(din);
  GradPlan plan = grad_plan(rows, cols, vectors);
  const uint64_t need = polar_b200_flayernorm_grad_workspace_bytes(rows, cols);
  void* own = nullptr;
  float* partials = nullptr;
  if (dgamma || dbeta) {
    if (workspace && (workspace_bytes < need || !aligned16(workspace)))
      return fail(POLAR_B200_ERR_WORKSPACE, "workspace too small or not 16-byte aligned");
    if (!workspace) {
      cudaError_t e = scratch_alloc(&own, need, st);
      if (e != cudaSuccess) return fail(POLAR_B200_ERR_CUDA, "scratch (sums over rows)", e);
    }
    partials = static_cast<float*>(workspace ? workspace : own);
  }
  uint32_t parts = 0;
  if (plan.lanes) {
    auto go = [&](auto with, auto without) {
      return (vectors ? with : without)(plan, st, gradient, in, gamma, mean, rstd, rows, cols, din, partials);
    };
#define ROWS(LANES, V, CTAS) go(launch_grad_rows<LANES, V, true, CTAS>, launch_grad_rows<LANES, V, false, CTAS>)
#define FLOATS(LANES) launch_grad_rows<LANES, 4, false, 1>(plan, st, gradient, in, gamma, mean, rstd, rows, cols, din, partials)
    switch (plan.lanes) {
      case 8: rc = plan.v == 1 ? ROWS(8, 1, 1) : plan.v == 2 ? ROWS(8, 2, 1) : ROWS(8, 4, 1); break;
      case 16: rc = ROWS(16, 4, 1); break;
      case 32: rc = ROWS(32, 4, 1); break;
      case 64: rc = ROWS(64, 4, 1); break;
      case 128: rc = ROWS(128, 4, 1); break;
      case 96: rc = FLOATS(96); break;
      case 160: rc = FLOATS(160); break;
      case 224: rc = FLOATS(224); break;
      case 320: rc = FLOATS(320); break;
      case 384: rc = FLOATS(384); break;
      case 448: rc = FLOATS(448); break;
      case 256:
        switch (plan.ctas) {
          case 1: rc = ROWS(256, 4, 1); break;
          case 3: rc = ROWS(256, 4, 3); break;
          case 4: rc = ROWS(256, 4, 4); break;
          case 5: rc = ROWS(256, 4, 5); break;
          case 6: rc = ROWS(256, 4, 6); break;
          case 7: rc = ROWS(256, 4, 7); break;
          default: rc = ROWS(256, 4, 8);
        }
        break;
      default:
        switch (plan.ctas) {
          case 1: rc = ROWS(512, 4, 1); break;
          case 5: rc = ROWS(512, 4, 5); break;
          case 6: rc = ROWS(512, 4, 6); break;
          case 7: rc = ROWS(512, 4, 7); break;
          default: rc = ROWS(512, 4, 8);
        }
    }
    parts = plan.grid;                                     // (with clusters what is resident, which is less than planned)
#undef FLOATS
#undef ROWS
  } else if (partials) {
    parts = (uint32_t)stretches(rows);
    rc = launch("flayernorm_grad_columns", norm_grad_columns_kernel, dim3((unsigned)((cols + kThreads - 1) / kThreads), parts), kThreads, 0, st,
                gradient, in, mean, rstd, rows, cols, (rows + parts - 1) / parts, partials);
  }
  if (rc == POLAR_B200_OK && partials) {
    // Few columns: 16 to a CTA, and so half the loads one after the other (4000 x 300 in all 7.6 us, with 32 8.5; 8000 x 1000 21.2 and 20.1, where more
    // CTAs are more rows of 64 bytes at a time)
    auto go = [&](auto kernel, unsigned each) {
      return launch("flayernorm_grad_sum", kernel, dim3((unsigned)((cols + each - 1) / each), 2), kFinishThreads, 0, st, partials, parts, cols, dgamma, dbeta);
    };
    rc = cols <= 5 * (uint64_t)sm_count() ? go(norm_grad_finish_kernel<16>, 16) : go(norm_grad_finish_kernel<32>, 32);
  }
  if (rc == POLAR_B200_OK && !plan.lanes)                  // (last: din may be gradient or in)
    rc = launch("flayernorm_grad", norm_grad_in_kernel, dim3((unsigned)rows), kThreads, 0, st, gradient, in, gamma, mean, rstd, cols, din);
  if (own) {
    cudaError_t e = scratch_free(own, st);
    if (rc == POLAR_B200_OK && e != cudaSuccess) rc = fail(POLAR_B200_ERR_CUDA, "returning scratch", e);
  }
  return rc;
}

}  // extern "C"
