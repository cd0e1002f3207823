// One AdamW step over many tensors.
//
// HBM-bound: with moments in 32 bits a weight reads 16 bytes (weight, gradient, two moments) and writes 12; with moments in
// 8 bits it reads 10 and writes 6, and a block of 128 weights reads and writes two scales.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <exception>
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

struct Rates {
  float keep, rate, inv_root2;                             // 1 - lr * decay, lr / (1 - beta1^step)
};
__device__ __forceinline__ Rates rates_of(const Common& c, float decay) {
  if (!c.schedule) return Rates{1.f - c.lr * decay, c.lr * c.inv_correct1, c.inv_root2};
  // 1 - beta^step = -expm1(step * log beta): no digits are lost at small steps, where beta^step is close to 1
  const float step = c.schedule[0], lr = c.schedule[1];
  return Rates{1.f - lr * decay, lr / -expm1f(step * c.log_beta1), 1.f / sqrtf(-expm1f(step * c.log_beta2))};
}

__device__ __forceinline__ float new_first(const Common& c, float m, float g) {
  return __fadd_rn(__fmul_rn(m, c.beta1), __fmul_rn(g, c.rest1));
}
__device__ __forceinline__ float new_second(const Common& c, float v, float g) {
  return __fadd_rn(__fmul_rn(v, c.beta2), __fmul_rn(__fmul_rn(g, c.rest2), g));
}
__device__ __forceinline__ float new_weight(const Common& c, const Rates& r, float w, float m, float root) {
  return w * r.keep - r.rate * (m / (root * r.inv_root2 + c.eps));
}

__global__ void __launch_bounds__(256) adamw_kernel(const __grid_constant__ Common c, const __grid_constant__ Tensor t) {
  pdl_enter();
  const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= t.count) return;
  const Rates r = rates_of(c, t.decay);
  float *first = static_cast<float*>(t.first), *second = static_cast<float*>(t.second);
  const float g = t.gradient[i], m = new_first(c, first[i], g), v = new_second(c, second[i], g);
  first[i] = m;
  second[i] = v;
  t.weights[i] = new_weight(c, r, t.weights[i], m, __fsqrt_rn(v));
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

// One CTA per block of codes.
__global__ void __launch_bounds__(kBlock) adamw8_kernel(const __grid_constant__ Common c, const __grid_constant__ Tensor t) {
  pdl_enter();
  __shared__ uint32_t largest[2][kBlock / 32];
  const uint64_t i = (uint64_t)blockIdx.x * kBlock + threadIdx.x;
  const bool live = i < t.count;
  uint8_t *first = static_cast<uint8_t*>(t.first), *second = static_cast<uint8_t*>(t.second);
  const Rates r = rates_of(c, t.decay);
  float m = 0.f, v = 0.f, u = 0.f;
  if (live) {
    const float g = t.gradient[i];
    m = __fmul_rn(from_e4m3(first[i]).x, t.first_scales[blockIdx.x]);
    u = __fmul_rn(from_e4m3(second[i]).x, t.second_scales[blockIdx.x]);
    m = new_first(c, m, g);
    v = new_second(c, __fmul_rn(u, u), g);
    u = __fsqrt_rn(v);
    t.weights[i] = new_weight(c, r, t.weights[i], m, u);
  }
  const uint32_t am = __reduce_max_sync(0xffffffffu, __float_as_uint(m) & 0x7fffffffu), au = __reduce_max_sync(0xffffffffu, __float_as_uint(u) & 0x7fffffffu);
  if ((threadIdx.x & 31) == 0) {
    largest[0][threadIdx.x >> 5] = am;
    largest[1][threadIdx.x >> 5] = au;
  }
  __syncthreads();
  uint32_t most[2] = {0, 0};
  for (int w = 0; w < (int)kBlock / 32; ++w)
    for (int k = 0; k < 2; ++k) most[k] = max(most[k], largest[k][w]);
  const float sm = scale_of(most[0]), su = scale_of(most[1]);
  if (threadIdx.x == 0) {
    t.first_scales[blockIdx.x] = sm;
    t.second_scales[blockIdx.x] = su;
  }
  if (!live) return;
  const uint32_t codes = to_e4m3(sm == 0.f ? 0.f : __fmul_rn(m, __fdiv_rn(1.f, sm)), su == 0.f ? 0.f : __fmul_rn(u, __fdiv_rn(1.f, su)));
  first[i] = (uint8_t)codes;
  const uint8_t q = (uint8_t)(codes >> 8);
  second[i] = q == 0 && u > 0.f && su > 0.f ? 1 : q;
}

// Whether no two of the arrays that a step writes share memory: two threads would race on it.  Usually each kind of array lies in
// ascending order in memory of its own, which one walk sees; else the spans are sorted.
using Span = std::pair<uintptr_t, uintptr_t>;
Span span_of(const polar_b200_adamw_tensor& t, int kind) {
  const uint64_t bytes = kind == 0 ? 4 * t.count : kind <= 2 ? (t.first_scales ? t.count : 4 * t.count)
                         : t.first_scales ? (t.count + kBlock - 1) / kBlock * 4 : 0;
  const void* p = kind == 0 ? t.weights : kind == 1 ? t.first : kind == 2 ? t.second : kind == 3 ? t.first_scales : t.second_scales;
  return Span(reinterpret_cast<uintptr_t>(p), reinterpret_cast<uintptr_t>(p) + bytes);
}
bool disjoint(const polar_b200_adamw_tensor* tensors, uint64_t count) {
  bool ascending = true;
  Span range[5];
  for (int kind = 0; kind < 5; ++kind) {
    Span& r = range[kind] = Span(0, 0);
    for (uint64_t i = 0; i < count; ++i) {
      const Span s = span_of(tensors[i], kind);
      if (s.first == s.second) continue;
      if (r.second == 0) {
        r = s;
        continue;
      }
      ascending = ascending && s.first >= r.second;
      r.second = std::max(r.second, s.second);
    }
  }
  if (ascending) {
    bool apart = true;
    for (int a = 0; a < 5; ++a)
      for (int b = 0; b < a; ++b) apart = apart && (range[a].first >= range[b].second || range[b].first >= range[a].second);
    if (apart) return true;
  }
  std::vector<Span> all;
  all.reserve(5 * count);
  for (uint64_t i = 0; i < count; ++i)
    for (int kind = 0; kind < 5; ++kind) {
      const Span s = span_of(tensors[i], kind);
      if (s.first != s.second) all.push_back(s);
    }
  std::sort(all.begin(), all.end());
  for (size_t i = 1; i < all.size(); ++i)
    if (all[i].first < all[i - 1].second) return false;
  return true;
}

}  // namespace

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
    if (!disjoint(tensors, count)) return fail(POLAR_B200_ERR_INVALID, "fadamw: a tensor is named twice, or two overlap");
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
  c.log_beta1 = (float)std::log((double)o->beta1), c.log_beta2 = (float)std::log((double)o->beta2);
  c.lr = o->lr;
  c.inv_correct1 = (float)(1.0 / (1.0 - std::pow((double)o->beta1, (double)o->step)));
  c.inv_root2 = (float)(1.0 / std::sqrt(1.0 - std::pow((double)o->beta2, (double)o->step)));
  for (uint64_t i = 0; i < count; ++i) {
    const polar_b200_adamw_tensor& t = tensors[i];
    if (t.count == 0) continue;
    const Tensor d{t.weights, t.gradient, t.first, t.second, t.first_scales, t.second_scales, t.count, t.weight_decay};
    int rc = t.first_scales ? launch("fadamw8", adamw8_kernel, dim3((unsigned)((t.count + kBlock - 1) / kBlock)), kBlock, 0, as_stream(stream), c, d)
                            : launch("fadamw", adamw_kernel, dim3((unsigned)((t.count + 255) / 256)), 256, 0, as_stream(stream), c, d);
    if (rc) return rc;
  }
  return POLAR_B200_OK;
}
