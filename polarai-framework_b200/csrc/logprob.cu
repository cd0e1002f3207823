// Log probabilities of given classes or tokens, the rows' entropies and likeliest alternatives, and the gradient.
//
// With m the row's maximum, d = x - m, S = sum(exp d) and T = sum(exp(d) * d):
//   logSumExp = m + log S,   logProb = d[id] - log S,   entropy = log S - T / S,
// where no term cancels another: d <= 0, so T <= 0 and log S >= 0.  A -inf logit has exp d = 0 and no part in T.
#include "rows.cuh"

namespace polar_b200 {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kMaxTop = 32;

// The id of a row: whole in 0 .. classes - 1, kPadding below zero, kWrong for anything else.
constexpr int64_t kPadding = -1, kWrong = -2;
__device__ __forceinline__ int64_t read_id(const void* ids, int type, uint64_t row, uint64_t classes) {
  int64_t id;
  if (type == POLAR_B200_IDS_F32) {
    const float f = static_cast<const float*>(ids)[row];
    if (f < 0.f) return kPadding;
    if (!(f < (float)classes) || f != truncf(f)) return kWrong;
    id = (int64_t)f;
  } else {
    id = type == POLAR_B200_IDS_I32 ? static_cast<const int32_t*>(ids)[row] : static_cast<const int64_t*>(ids)[row];
  }
  return id < 0 ? kPadding : (uint64_t)id < classes ? id : kWrong;
}
__device__ __forceinline__ void write_id(void* ids, int type, uint64_t at, uint32_t id) {
  if (type == POLAR_B200_IDS_F32) static_cast<float*>(ids)[at] = (float)id;
  else if (type == POLAR_B200_IDS_I32) static_cast<int32_t*>(ids)[at] = (int32_t)id;
  else static_cast<int64_t*>(ids)[at] = (int64_t)id;
}

// An order over (value, index): larger values first, of equal ones the lower index; NaN above everything, -0 as +0.
// Never 0, which stands for "none".
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);
  return v != v ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t rank_of(float v, uint32_t index) { return (uint64_t)ordered(v) << 32 | (uint32_t)~index; }

struct LogProbOut {
  float *logprob, *entropy, *logsumexp;
  void* top_ids;
  float* top_logprob;
  uint32_t top;
};

__global__ void __launch_bounds__(kThreads) logprob_kernel(const float* logits, uint64_t classes, uint64_t pitch, const void* ids,
                                                           int id_type, LogProbOut o) {
  pdl_enter();
  __shared__ float slots[2 * kThreads / 32], shared_max;
  __shared__ unsigned long long best[kThreads / 32];
  const uint64_t row = blockIdx.x;
  const float* x = logits + row * pitch;
  float m = -INFINITY;
  for (uint64_t c = threadIdx.x; c < classes; c += kThreads) m = fmaxf(m, x[c]);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kThreads / 32; ++w) m = fmaxf(m, slots[w]);
    shared_max = m;
  }
  __syncthreads();
  m = shared_max == -INFINITY ? 0.f : shared_max;          // (a row of NaNs alone as well: its sum is NaN)
  float s[2] = {0.f, 0.f};
  for (uint64_t c = threadIdx.x; c < classes; c += kThreads) {
    const float d = x[c] - m, e = expf(d);
    s[0] += e;
    if (!(e == 0.f)) s[1] += e * d;
  }
  block_sums<kThreads>(s, slots);
  const bool dead = s[0] == 0.f;                           // nothing in the row has any probability
  const float log_sum = logf(s[0]);
  if (threadIdx.x == 0) {
    if (o.logprob) {
      const int64_t id = read_id(ids, id_type, row, classes);
      o.logprob[row] = id == kPadding ? 0.f : id == kWrong ? NAN : dead ? -INFINITY : x[id] - m - log_sum;
    }
    if (o.entropy) o.entropy[row] = dead ? 0.f : log_sum - s[1] / s[0];
    if (o.logsumexp) o.logsumexp[row] = dead ? -INFINITY : m + log_sum;
  }
  unsigned long long last = ~0ull;
  for (uint32_t k = 0; k < o.top; ++k) {                   // the largest below the one before
    unsigned long long mine = 0;
    for (uint64_t c = threadIdx.x; c < classes; c += kThreads) {
      const unsigned long long r = rank_of(x[c], (uint32_t)c);
      if (r < last && r > mine) mine = r;
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, mine, off);
      mine = other > mine ? other : mine;
    }
    if ((threadIdx.x & 31) == 0) best[threadIdx.x >> 5] = mine;
    __syncthreads();
    last = 0;
    for (int w = 0; w < kThreads / 32; ++w) last = best[w] > last ? best[w] : last;
    __syncthreads();
    if (threadIdx.x == 0) {
      const uint32_t at = ~(uint32_t)last;
      if (o.top_ids) write_id(o.top_ids, id_type, row * o.top + k, at);
      if (o.top_logprob) o.top_logprob[row * o.top + k] = dead ? -INFINITY : x[at] - m - log_sum;
    }
  }
}

// The gradient.  What is the same for a row: its logSumExp, -(gLogProb + gEntropy * entropy), gEntropy, the id.
__global__ void __launch_bounds__(kThreads) logprob_grad_kernel(const float* logits, uint64_t classes, uint64_t pitch, const void* ids,
                                                                int id_type, const float* logsumexp, const float* entropy,
                                                                const float* g_logprob, const float* g_entropy, float* dlogits,
                                                                uint64_t dpitch) {
  pdl_enter();
  const uint64_t row = blockIdx.x;
  const float* x = logits + row * pitch;
  float* dx = dlogits + row * dpitch;
  const int64_t id = read_id(ids, id_type, row, classes);
  const float lse = logsumexp[row];
  float g = id == kPadding ? 0.f : g_logprob[row];
  const float ge = g_entropy ? g_entropy[row] : 0.f;
  const bool nothing = lse == -INFINITY || (g == 0.f && ge == 0.f);
  if (id == kWrong && g != 0.f) g = NAN;
  const float h = ge != 0.f ? entropy[row] : 0.f;
  for (uint64_t c = threadIdx.x; c < classes; c += kThreads) {
    float v = 0.f;
    if (!nothing) {
      const float l = x[c] - lse, p = expf(l);
      v = p == 0.f ? 0.f * g : p * (-g - ge * (l + h));
      if ((int64_t)c == id) v += g;
    }
    dx[c] = v;
  }
}

constexpr uint64_t kMaxClasses = 1ull << 31, kMaxRows = 0x7fffffffull;

int check_ids(const char* what, uint64_t rows, uint64_t classes, uint64_t pitch, int id_type) {
  if (id_type != POLAR_B200_IDS_F32 && id_type != POLAR_B200_IDS_I32 && id_type != POLAR_B200_IDS_I64)
    return fail(POLAR_B200_ERR_INVALID, "ids are held in fp32, in 32 or in 64 bits");
  if (rows > kMaxRows || classes > kMaxClasses || pitch < classes || pitch > 1ull << 40) return fail(POLAR_B200_ERR_INVALID, what);
  if (id_type == POLAR_B200_IDS_F32 && classes > 1ull << 24)
    return fail(POLAR_B200_ERR_INVALID, "ids in fp32 reach to 2^24 classes");
  return POLAR_B200_OK;
}

}  // namespace
}  // namespace polar_b200

using namespace polar_b200;

extern "C" {

int polar_b200_flogprob(const float* logits, uint64_t rows, uint64_t classes, uint64_t pitch, const void* ids, int id_type,
                        float* logprob, float* entropy, float* logsumexp, uint64_t top, void* top_ids, float* top_logprob,
                        void* stream) {
  clear_error();
  int rc = check_ids("flogprob: too many rows or classes, or rows closer than their length", rows, classes, pitch, id_type);
  if (rc) return rc;
  if (top > kMaxTop || top > classes) return fail(POLAR_B200_ERR_INVALID, "flogprob: at most 32 alternatives, and no more than classes");
  if (rows == 0) return POLAR_B200_OK;
  if (classes == 0) return fail(POLAR_B200_ERR_INVALID, "flogprob: rows without classes");
  if (!logits || (logprob && !ids)) return fail(POLAR_B200_ERR_INVALID, "null device pointer");
  if (!top_ids && !top_logprob) top = 0;
  const void* some = logprob ? logprob : entropy ? entropy : logsumexp ? logsumexp : top_logprob ? (const void*)top_logprob : top_ids;
  if (!some) return POLAR_B200_OK;                         // nothing is asked for
  LaunchDeviceScope on(stream, some);
  return launch("flogprob", logprob_kernel, dim3((unsigned)rows), kThreads, 0, as_stream(stream), logits, classes, pitch, ids, id_type,
                LogProbOut{logprob, entropy, logsumexp, top_ids, top_logprob, (uint32_t)top});
}

int polar_b200_flogprob_grad(const float* logits, uint64_t rows, uint64_t classes, uint64_t pitch, const void* ids, int id_type,
                             const float* logsumexp, const float* entropy, const float* g_logprob, const float* g_entropy,
                             float* dlogits, uint64_t dpitch, void* stream) {
  clear_error();
  int rc = check_ids("flogprob_grad: too many rows or classes, or rows closer than their length", rows, classes, pitch, id_type);
  if (rc) return rc;
  if (dpitch < classes || dpitch > 1ull << 40) return fail(POLAR_B200_ERR_INVALID, "flogprob_grad: rows of the result closer than their length");
  if (rows == 0 || classes == 0) return POLAR_B200_OK;
  if (!logits || !ids || !logsumexp || !g_logprob || !dlogits || (g_entropy && !entropy))
    return fail(POLAR_B200_ERR_INVALID, "null device pointer");
  if (logits == dlogits && pitch != dpitch) return fail(POLAR_B200_ERR_INVALID, "flogprob_grad: in place the rows lie alike");
  LaunchDeviceScope on(stream, dlogits);
  return launch("flogprob_grad", logprob_grad_kernel, dim3((unsigned)rows), kThreads, 0, as_stream(stream), logits, classes, pitch, ids,
                id_type, logsumexp, entropy, g_logprob, g_entropy, dlogits, dpitch);
}

}  // extern "C"
