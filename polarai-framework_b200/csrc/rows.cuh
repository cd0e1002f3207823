// Sums and maxima over the threads that share a row.
#pragma once
#include "common.cuh"

namespace polar_b200 {

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}

// The sums of `N` values over the CTA, in every thread; added in the same order in each of them.  `slots`: N values for
// each warp, not in use by anything since the last barrier.
template <int THREADS, int N>
__device__ __forceinline__ void block_sums(float (&v)[N], float* slots) {
  constexpr int kWarps = THREADS / 32;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
  if (kWarps == 1) return;
  if ((threadIdx.x & 31) == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) slots[(threadIdx.x >> 5) * N + i] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = slots[threadIdx.x % kWarps * N + i];            // (a power of two)
#pragma unroll
    for (int off = kWarps / 2; off > 0; off >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], off);
  }
}

// Pairs of floats: one instruction multiplies both, or multiplies and adds; each is rounded as by itself.
using Pair = unsigned long long;
__device__ __forceinline__ Pair pair(float lo, float hi) {
  Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(lo), "f"(hi));
  return p;
}
__device__ __forceinline__ float2 halves(Pair p) {
  float2 v;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(p));
  return v;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

}  // namespace polar_b200
