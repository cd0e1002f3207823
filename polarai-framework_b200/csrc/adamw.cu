// One AdamW step over many tensors.
//
// HBM-bound: with moments in 32 bits a weight reads 16 bytes (weight, gradient, two moments) and writes 12; with moments in
// 8 bits it reads 10 and writes 6, and a block of 128 weights reads and writes two scales.  All tensors of a kind share a launch: a CTA finds
// its chunk's tensor in a table among the kernel's parameters.  One chunk per CTA: loops over several measured 10 to 20 % slower.
// Measured, 235 M weights in 163 tensors: 941 us in 32 bits (7.0 TB/s), 668 us in 8 (5.7 TB/s; 606 in short runs, at higher clocks; issue slots 70 %
// busy); 113 small ones 3.5 us.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <exception>
#include <iterator>
#include <utility>
#include <vector>

#include "rows.cuh"

namespace polar_b200 {
namespace {

constexpr uint32_t kBlock = 128;                           // codes per scale
constexpr float kInvMax = 0.0022321429569274187f;          // 1 / 448 in fp32; 448 is the largest e4m3 value
constexpr float kLeast = 7.888609052210118e-31f;           // 2^-100

// What one step has in common: the powers of beta by number of the step come from the host, or from `schedule`.
struct Common {
  float beta1, beta2, rest1, rest2;                        // rest: 1 - beta
  float eps;
  float lr, inv_correct1, inv_root2;                       // 1 / (1 - beta1^step), 1 / sqrt(1 - beta2^step)
  float log_beta1, log_beta2;
  float one;                                               // 1, in a place where the compiler does not see it (sum_of)
  const float* schedule;
};
struct Tensor {
  float* weights;
  const float* gradient;
  void *first, *second;
  float *first_scales, *second_scales;
  uint64_t count;
  float decay;
};
// The tensors of one launch, in the kernel's parameters (32764 bytes at most), and the chunk at which each begins.
template <int N>
struct Table {
  Common c;
  uint32_t count;
  uint32_t first[N];
  Tensor tensor[N];
};
constexpr int kFewTensors = 16, kMoreTensors = 192, kManyTensors = 448;
static_assert(sizeof(Table<kManyTensors>) <= 32764, "kernel parameters");

struct Rates {
  float keep, rate, inv_root2;                             // 1 - lr * decay, lr / (1 - beta1^step)
};
__device__ __forceinline__ Rates rates_of(const Common& c, float decay) {
  if (!c.schedule) return Rates{1.f - c.lr * decay, c.lr * c.inv_correct1, c.inv_root2};
  // 1 - beta^step = -expm1(step * log beta): no digits are lost at small steps, where beta^step is close to 1
  const float step = c.schedule[0], lr = c.schedule[1];
  return Rates{1.f - lr * decay, lr / -expm1f(step * c.log_beta1), 1.f / sqrtf(-expm1f(step * c.log_beta2))};
}
// The tensor that a chunk belongs to: in each round the begins of seven at a time, which are read together (235 M weights in 163 tensors, moments in 8 bits: 669 us, by
// halving 675).  The places behind the last tensor hold the largest number.
template <int N>
__device__ __forceinline__ uint32_t tensor_of(const Table<N>& t, uint32_t chunk) {
  uint32_t at = 0;
#pragma unroll
  for (uint32_t step = N > 64 ? 64 : 8; step > 0; step /= 8) {
    uint32_t more = 0;
#pragma unroll
    for (uint32_t k = 1; k < 8; ++k)
      if (k * step < N) more += at + k * step < N && t.first[at + k * step] <= chunk;
    at += more * step;
  }
  return at;
}

__device__ __forceinline__ float new_first(const Common& c, float m, float g) {
  return __fadd_rn(__fmul_rn(m, c.beta1), __fmul_rn(g, c.rest1));
}
__device__ __forceinline__ float new_second(const Common& c, float v, float g) {
  return __fadd_rn(__fmul_rn(v, c.beta2), __fmul_rn(__fmul_rn(g, c.rest2), g));
}
__device__ __forceinline__ float new_weight(const Common& c, const Rates& r, float w, float m, float root) {
  return w * r.keep - r.rate * __fdividef(m, root * r.inv_root2 + c.eps);
}

// Moments in 32 bits: a chunk of kThreads vectors of four weights per CTA.
constexpr int kThreads = 256;
__device__ __forceinline__ void step4(const Common& c, const Rates& r, float4& w, const float4& g, float4& m, float4& v) {
  float* wp = &w.x;
  const float* gp = &g.x;
  float *mp = &m.x, *vp = &v.x;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    mp[k] = new_first(c, mp[k], gp[k]);
    vp[k] = new_second(c, vp[k], gp[k]);
    wp[k] = new_weight(c, r, wp[k], mp[k], __fsqrt_rn(vp[k]));
  }
}
template <int N>
__global__ void __launch_bounds__(kThreads, 6) adamw_kernel(const __grid_constant__ Table<N> table) {
  pdl_enter();
  const Common& c = table.c;
  const uint32_t at = tensor_of(table, blockIdx.x);
  const Tensor& t = table.tensor[at];
  float *first = static_cast<float*>(t.first), *second = static_cast<float*>(t.second);
  const uint64_t begin = (uint64_t)(blockIdx.x - table.first[at]) * (kThreads * 4);
  const bool vectors = ((reinterpret_cast<uintptr_t>(t.weights) | reinterpret_cast<uintptr_t>(t.gradient) | reinterpret_cast<uintptr_t>(first) |
                         reinterpret_cast<uintptr_t>(second)) & 15) == 0;
  const uint64_t i = begin + (vectors ? 4 * threadIdx.x : threadIdx.x);
  if (vectors && i + 4 <= t.count) {
    float4 w = ld_stream(reinterpret_cast<const float4*>(t.weights + i));
    const float4 g = ld_stream(reinterpret_cast<const float4*>(t.gradient + i));
    float4 m = ld_stream(reinterpret_cast<const float4*>(first + i)), v = ld_stream(reinterpret_cast<const float4*>(second + i));
    step4(c, rates_of(c, t.decay), w, g, m, v);
    st_stream(reinterpret_cast<float4*>(t.weights + i), w);
    st_stream(reinterpret_cast<float4*>(first + i), m);
    st_stream(reinterpret_cast<float4*>(second + i), v);
    return;
  }
  // the last few of a tensor, or tensors on odd boundaries: four floats of each, eight loads on their way (sixteen take registers that more threads
  // would use: 941 us, 957)
  const Rates r = rates_of(c, t.decay);
  const uint32_t step = vectors ? 1 : kThreads;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    float w[2], g[2], m[2], v[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint64_t e = i + (2 * half + k) * step;
      const bool live = e < t.count;
      w[k] = live ? t.weights[e] : 0.f, g[k] = live ? t.gradient[e] : 0.f, m[k] = live ? first[e] : 0.f, v[k] = live ? second[e] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint64_t e = i + (2 * half + k) * step;
      if (e >= t.count) return;
      first[e] = m[k] = new_first(c, m[k], g[k]);
      second[e] = v[k] = new_second(c, v[k], g[k]);
      t.weights[e] = new_weight(c, r, w[k], m[k], __fsqrt_rn(v[k]));
    }
  }
}

// e4m3 to float and back, a pair at a time.
__device__ __forceinline__ float2 from_e4m3(uint32_t pair) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)pair));
  float2 v;
  asm("{.reg .b16 lo, hi; mov.b32 {lo, hi}, %2; cvt.f32.f16 %0, lo; cvt.f32.f16 %1, hi;}" : "=f"(v.x), "=f"(v.y) : "r"(h));
  return v;
}
__device__ __forceinline__ uint32_t to_e4m3(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// The scale of a block by its largest magnitude (as bits, which order like the magnitudes, NaN above all).
__device__ __forceinline__ float scale_of(uint32_t largest) {
  const float a = __uint_as_float(largest);
  return a < kLeast ? 0.f : __fmul_rn(a, kInvMax);
}

// Moments in 8 bits: a warp per block of codes, four weights per lane; UNROLL blocks of a warp in flight.  Some 60 instructions per weight
// as written one by one kept the issue slots 87 % busy; with packed arithmetic 69 %, and the memory is what is left.
struct Codes {
  uint32_t first, second;                                  // four codes each
  float first_scale, second_scale;
};
__device__ __forceinline__ Pair twice(float v) { return pair(v, v); }
// a + b, each sum rounded: as 1 * a + b, since the assembler makes one fused instruction of a packed product and a packed sum.
__device__ __forceinline__ Pair sum_of(const Common& c, Pair a, Pair b) { return fma2(twice(c.one), a, b); }
__device__ __forceinline__ float reciprocal(float v) {     // 1 ulp
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ void step4(const Common& c, const Rates& r, float4& w, const float4& g, Codes& q) {
  Pair m[2], u[2];
  uint32_t most_m = 0, most_u = 0;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const float2 a = from_e4m3(q.first >> 16 * h & 0xffff), b = from_e4m3(q.second >> 16 * h & 0xffff);
    const Pair gh = h ? pair(g.z, g.w) : pair(g.x, g.y);
    m[h] = sum_of(c, mul2(mul2(pair(a.x, a.y), twice(q.first_scale)), twice(c.beta1)), mul2(gh, twice(c.rest1)));
    const Pair root = mul2(pair(b.x, b.y), twice(q.second_scale));
    const float2 v = halves(sum_of(c, mul2(mul2(root, root), twice(c.beta2)), mul2(mul2(gh, twice(c.rest2)), gh)));
    u[h] = pair(__fsqrt_rn(v.x), __fsqrt_rn(v.y));
    const float2 divisor = halves(fma2(u[h], twice(r.inv_root2), twice(c.eps)));
    const Pair update = mul2(mul2(m[h], twice(-r.rate)), pair(reciprocal(divisor.x), reciprocal(divisor.y)));
    const float2 nw = halves(fma2(h ? pair(w.z, w.w) : pair(w.x, w.y), twice(r.keep), update));
    if (h) w.z = nw.x, w.w = nw.y;
    else w.x = nw.x, w.y = nw.y;
    most_m = max(max(most_m, __float_as_uint(halves(m[h]).x) & 0x7fffffffu), __float_as_uint(halves(m[h]).y) & 0x7fffffffu);
    most_u = max(max(most_u, __float_as_uint(halves(u[h]).x)), __float_as_uint(halves(u[h]).y));   // (no root has a sign)
  }
  q.first_scale = scale_of(__reduce_max_sync(0xffffffffu, most_m));
  q.second_scale = scale_of(__reduce_max_sync(0xffffffffu, most_u));
  // (a block below the least scale is zeros: its values times 0)
  const float by_m = q.first_scale == 0.f ? 0.f : __frcp_rn(q.first_scale), by_u = q.second_scale == 0.f ? 0.f : __frcp_rn(q.second_scale);
  const float2 m0 = halves(mul2(m[0], twice(by_m))), m1 = halves(mul2(m[1], twice(by_m)));
  const float2 u0 = halves(mul2(u[0], twice(by_u))), u1 = halves(mul2(u[1], twice(by_u)));
  q.first = to_e4m3(m0.x, m0.y) | to_e4m3(m1.x, m1.y) << 16;
  uint32_t s = to_e4m3(u0.x, u0.y) | to_e4m3(u1.x, u1.y) << 16;
  uint32_t zeros = ~(((s & 0x7f7f7f7fu) + 0x7f7f7f7fu) | s) & 0x80808080u;   // the top bit of each byte that is zero
  if (zeros && by_u > 0.f) {
    const float2 a = halves(u[0]), b = halves(u[1]);
    zeros &= (a.x > 0.f ? 0x80u : 0u) | (a.y > 0.f ? 0x8000u : 0u) | (b.x > 0.f ? 0x800000u : 0u) | (b.y > 0.f ? 0x80000000u : 0u);
    s |= zeros >> 7;
  }
  q.second = s;
}
template <int N, int UNROLL>
__global__ void __launch_bounds__(kThreads, 5) adamw8_kernel(const __grid_constant__ Table<N> table) {
  pdl_enter();
  const Common& c = table.c;
  const uint32_t at = tensor_of(table, blockIdx.x), lane = threadIdx.x & 31;
  const Tensor& t = table.tensor[at];
  uint8_t *first = static_cast<uint8_t*>(t.first), *second = static_cast<uint8_t*>(t.second);
  // the warp's blocks lie side by side
  const uint64_t block = ((uint64_t)(blockIdx.x - table.first[at]) * (kThreads / 32) + (threadIdx.x >> 5)) * UNROLL;
  if (block * kBlock >= t.count) return;
  const bool vectors = ((reinterpret_cast<uintptr_t>(t.weights) | reinterpret_cast<uintptr_t>(t.gradient)) & 15) == 0 &&
                       ((reinterpret_cast<uintptr_t>(first) | reinterpret_cast<uintptr_t>(second)) & 3) == 0;
  if (vectors && (block + UNROLL) * kBlock <= t.count) {
    const uint64_t i = block * (kBlock / 4) + lane;
    float4 w[UNROLL], g[UNROLL];
    Codes q[UNROLL];
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) {
      w[k] = ld_stream(reinterpret_cast<const float4*>(t.weights) + i + 32 * k);
      g[k] = ld_stream(reinterpret_cast<const float4*>(t.gradient) + i + 32 * k);
      q[k].first = reinterpret_cast<const uint32_t*>(first)[i + 32 * k];
      q[k].second = reinterpret_cast<const uint32_t*>(second)[i + 32 * k];
      q[k].first_scale = t.first_scales[block + k];
      q[k].second_scale = t.second_scales[block + k];
    }
    const Rates r = rates_of(c, t.decay);
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) {
      step4(c, r, w[k], g[k], q[k]);
      st_stream(reinterpret_cast<float4*>(t.weights) + i + 32 * k, w[k]);
      reinterpret_cast<uint32_t*>(first)[i + 32 * k] = q[k].first;
      reinterpret_cast<uint32_t*>(second)[i + 32 * k] = q[k].second;
      if (lane == 0) {
        t.first_scales[block + k] = q[k].first_scale;
        t.second_scales[block + k] = q[k].second_scale;
      }
    }
    return;
  }
  const Rates r = rates_of(c, t.decay);                    // the last blocks of a tensor, or blocks on odd boundaries
  for (uint64_t b = block; b < block + UNROLL && b * kBlock < t.count; ++b) {
    const uint64_t i = b * kBlock + 4 * lane;
    const bool whole = vectors && i + 4 <= t.count;
    float4 w, g;
    Codes q = {0, 0, t.first_scales[b], t.second_scales[b]};
    if (whole) {
      w = *reinterpret_cast<const float4*>(t.weights + i), g = *reinterpret_cast<const float4*>(t.gradient + i);
      q.first = *reinterpret_cast<const uint32_t*>(first + i), q.second = *reinterpret_cast<const uint32_t*>(second + i);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const bool live = i + k < t.count;
        (&w.x)[k] = live ? t.weights[i + k] : 0.f;
        (&g.x)[k] = live ? t.gradient[i + k] : 0.f;
        q.first |= (live ? (uint32_t)first[i + k] : 0u) << 8 * k;
        q.second |= (live ? (uint32_t)second[i + k] : 0u) << 8 * k;
      }
    }
    __syncwarp();
    step4(c, r, w, g, q);
    if (whole) {
      *reinterpret_cast<float4*>(t.weights + i) = w;
      *reinterpret_cast<uint32_t*>(first + i) = q.first, *reinterpret_cast<uint32_t*>(second + i) = q.second;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (whole || i + k >= t.count) continue;
      t.weights[i + k] = (&w.x)[k];
      first[i + k] = (uint8_t)(q.first >> 8 * k);
      second[i + k] = (uint8_t)(q.second >> 8 * k);
    }
    if (lane == 0) {
      t.first_scales[b] = q.first_scale;
      t.second_scales[b] = q.second_scale;
    }
  }
}

// Launches the tensors of one kind, a table's worth at a time.
template <int N, int UNROLL>
int launch_table(const polar_b200_adamw_tensor* tensors, uint64_t count, bool eight, const Common& c, cudaStream_t stream, uint64_t* taken) {
  Table<N> table;
  table.c = c;
  table.count = 0;
  uint64_t chunks = 0, i = 0;
  const uint64_t chunk = (uint64_t)kThreads * UNROLL * 4;
  for (; i < count && table.count < N; ++i) {
    const polar_b200_adamw_tensor& t = tensors[i];
    if (t.count == 0 || (t.first_scales != nullptr) != eight) continue;
    const uint64_t more = (t.count + chunk - 1) / chunk;
    if (chunks + more > 0x7fffffffull) break;
    table.first[table.count] = (uint32_t)chunks;
    table.tensor[table.count++] = Tensor{t.weights, t.gradient, t.first, t.second, t.first_scales, t.second_scales, t.count, t.weight_decay};
    chunks += more;
  }
  *taken = i;
  if (table.count == 0) return POLAR_B200_OK;
  std::fill(table.first + table.count, table.first + N, 0xffffffffu);
  // moments in 8 bits: two blocks per warp in flight (one is a fifth slower, four the same within 3 %); in 32 bits one vector per thread and
  // more threads (941 us, two 949)
  if constexpr (UNROLL == 2) return launch_large("fadamw8", adamw8_kernel<N, 2>, dim3((unsigned)chunks), kThreads, stream, table);
  else return launch_large("fadamw", adamw_kernel<N>, dim3((unsigned)chunks), kThreads, stream, table);
}

// Whether no two of the arrays that a step writes share memory, nor one of them with a gradient: two threads would race on it.  (A tensor's
// weights may be its own gradient: the thread that writes an element has read it.)  Usually each kind of array lies in ascending order in
// memory of its own, which one walk sees; else the spans are sorted.
using Span = std::pair<uintptr_t, uintptr_t>;
constexpr int kWritten = 5;                                // kinds of arrays; the gradients come behind
Span span_of(const polar_b200_adamw_tensor& t, int kind) {
  if (kind == kWritten && t.gradient == t.weights) return Span(0, 0);
  const uint64_t bytes = kind == 0 || kind == kWritten ? 4 * t.count : kind <= 2 ? (t.first_scales ? t.count : 4 * t.count)
                         : t.first_scales ? (t.count + kBlock - 1) / kBlock * 4 : 0;
  const void* p = kind == 0 ? t.weights : kind == 1 ? t.first : kind == 2 ? t.second : kind == 3 ? t.first_scales : kind == 4 ? t.second_scales : t.gradient;
  return Span(reinterpret_cast<uintptr_t>(p), reinterpret_cast<uintptr_t>(p) + bytes);
}
bool disjoint(const polar_b200_adamw_tensor* tensors, uint64_t count) {
  bool ascending = true;
  Span range[kWritten + 1];
  for (int kind = 0; kind <= kWritten; ++kind) {
    Span& r = range[kind] = Span(0, 0);
    for (uint64_t i = 0; i < count; ++i) {
      const Span s = span_of(tensors[i], kind);
      if (s.first == s.second) continue;
      if (r.second == 0) {
        r = s;
        continue;
      }
      ascending = ascending && (s.first >= r.second || kind == kWritten);   // (gradients may lie as they like)
      r = Span(std::min(r.first, s.first), std::max(r.second, s.second));
    }
  }
  if (ascending) {
    bool apart = true;
    for (int a = 0; a <= kWritten; ++a)
      for (int b = 0; b < a; ++b) apart = apart && (range[a].first >= range[b].second || range[b].first >= range[a].second);
    if (apart) return true;
  }
  std::vector<Span> all;
  all.reserve(kWritten * count);
  for (uint64_t i = 0; i < count; ++i)
    for (int kind = 0; kind < kWritten; ++kind) {
      const Span s = span_of(tensors[i], kind);
      if (s.first != s.second) all.push_back(s);
    }
  std::sort(all.begin(), all.end());
  for (size_t i = 1; i < all.size(); ++i)
    if (all[i].first < all[i - 1].second) return false;
  for (uint64_t i = 0; i < count; ++i) {
    const Span s = span_of(tensors[i], kWritten);
    const auto next = std::lower_bound(all.begin(), all.end(), Span(s.second, 0));   // the first one that begins behind the gradient
    if (s.first != s.second && next != all.begin() && std::prev(next)->second > s.first) return false;
  }
  return true;
}

}  // namespace

// Whether the steps may run in any order or at once: no written array overlaps another, a gradient or the schedule.
bool adamw_independent(const polar_b200_adamw_tensor* tensors, uint64_t count, const float* schedule) {
  if (!disjoint(tensors, count)) return false;
  if (!schedule) return true;
  const uintptr_t from = reinterpret_cast<uintptr_t>(schedule);
  for (uint64_t i = 0; i < count; ++i)
    for (int kind = 0; kind < kWritten; ++kind) {
      const Span s = span_of(tensors[i], kind);
      if (s.first != s.second && from < s.second && s.first < from + 8) return false;
    }
  return true;
}

// The argument list of the builtin "fadamw" or "fadamw8" as the entry point takes it; false where it is none.
bool adamw_arguments(const char* name, const polar_b200_arg* a, uint64_t argc, polar_b200_adamw_tensor* t, polar_b200_adamw_options* o) {
  const bool eight = !std::strcmp(name, "fadamw8");
  const char* pattern = eight ? "TTffffTTTTT" : "TTffffTTT";
  if ((!eight && std::strcmp(name, "fadamw")) || argc != std::strlen(pattern)) return false;
  uint64_t n[11] = {};
  for (uint64_t i = 0; i < argc; ++i) {
    if ((pattern[i] == 'T') != (a[i].is_tensor != 0)) return false;
    if (!a[i].is_tensor) continue;
    if (a[i].tensor.dims && !a[i].tensor.shape) return false;
    n[i] = 1;
    for (uint64_t d = 0; d < a[i].tensor.dims; ++d) n[i] *= a[i].tensor.shape[d];
  }
  const uint64_t count = n[6];
  const int second = eight ? 9 : 8;
  if (n[0] != count || n[1] != 2 || !a[1].tensor.data) return false;
  if (eight) {
    const uint64_t codes = (count + 3) / 4, blocks = (count + kBlock - 1) / kBlock;
    if (n[7] < codes || n[8] != blocks || n[9] < codes || n[10] != blocks) return false;
  } else if (n[7] != count || n[8] != count) {
    return false;
  }
  *t = polar_b200_adamw_tensor{a[6].tensor.data, a[0].tensor.data, a[7].tensor.data, a[second].tensor.data,
                               eight ? a[8].tensor.data : nullptr, eight ? a[10].tensor.data : nullptr, count, a[5].scalar};
  *o = polar_b200_adamw_options{0.f, a[2].scalar, a[3].scalar, a[4].scalar, 0, a[1].tensor.data};
  return !eight || count == 0 || (t->first_scales && t->second_scales);
}
}  // namespace polar_b200

using namespace polar_b200;

extern "C" int polar_b200_fadamw(const polar_b200_adamw_tensor* tensors, uint64_t count, const polar_b200_adamw_options* o, void* stream) {
  clear_error();
  if (!o || (count && !tensors)) return fail(POLAR_B200_ERR_INVALID, "fadamw: no tensors or options");
  if (!(o->beta1 >= 0.f && o->beta1 < 1.f && o->beta2 >= 0.f && o->beta2 < 1.f && o->eps >= 0.f))
    return fail(POLAR_B200_ERR_INVALID, "fadamw: 0 <= beta < 1 and eps >= 0 are needed");
  if (!o->schedule && o->step == 0) return fail(POLAR_B200_ERR_INVALID, "fadamw: steps count from 1");
  for (uint64_t i = 0; i < count; ++i) {
    const polar_b200_adamw_tensor& t = tensors[i];
    if (t.count && (!t.weights || !t.gradient || !t.first || !t.second)) return fail(POLAR_B200_ERR_INVALID, "null device pointer");
    if (!t.first_scales != !t.second_scales) return fail(POLAR_B200_ERR_INVALID, "fadamw: both moments are held in 8 bits, or neither");
    if (t.count > 1ull << 37) return fail(POLAR_B200_ERR_INVALID, "fadamw: tensor too large");
  }
  try {
    if (!adamw_independent(tensors, count, o->schedule)) return fail(POLAR_B200_ERR_INVALID, "fadamw: what is written overlaps something else");
  } catch (const std::exception&) {                        // (no exception may leave a C entry)
    return fail(POLAR_B200_ERR_INVALID, "out of host memory");
  }
  const void* some = nullptr;
  for (uint64_t i = 0; i < count && !some; ++i) some = tensors[i].count ? tensors[i].weights : nullptr;
  if (!some) return POLAR_B200_OK;
  LaunchDeviceScope on(stream, some);
  Common c = {};
  c.beta1 = o->beta1, c.beta2 = o->beta2, c.rest1 = 1.f - o->beta1, c.rest2 = 1.f - o->beta2;
  c.eps = o->eps;
  c.schedule = o->schedule;
  c.one = 1.f;
  c.log_beta1 = (float)std::log((double)o->beta1), c.log_beta2 = (float)std::log((double)o->beta2);
  c.lr = o->lr;
  c.inv_correct1 = (float)(1.0 / (1.0 - std::pow((double)o->beta1, (double)o->step)));
  c.inv_root2 = (float)(1.0 / std::sqrt(1.0 - std::pow((double)o->beta2, (double)o->step)));
  for (int eight = 0; eight < 2; ++eight) {
    uint64_t i = 0;
    while (i < count) {
      uint64_t taken = 0;
      // (the table is a kernel's parameters, which the host pays for by their size: 4 tensors 7 us in all, 163 tensors 18, in the largest table 25)
      auto go = [&](auto small, auto medium, auto large) {
        auto f = count - i <= kFewTensors ? small : count - i <= kMoreTensors ? medium : large;
        return f(tensors + i, count - i, eight != 0, c, as_stream(stream), &taken);
      };
      int rc = eight ? go(launch_table<kFewTensors, 2>, launch_table<kMoreTensors, 2>, launch_table<kManyTensors, 2>)
                     : go(launch_table<kFewTensors, 1>, launch_table<kMoreTensors, 1>, launch_table<kManyTensors, 1>);
      if (rc) return rc;
      i += taken;
    }
  }
  return POLAR_B200_OK;
}
