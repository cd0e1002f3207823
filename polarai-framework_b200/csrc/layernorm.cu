// Layer norm of rows and its backward pass.
//
// HBM-bound streams: 8 bytes per element forward (a row is read and written), 12 backward (two rows read, one
// written), and a dozen operations each.  Deviations are summed around the mean, never as the difference of
// two large sums, and all sums are taken over two levels (threads, then the CTA), so that their rounding stays near that of a few dozen
// additions whatever the row's length.
#include "rows.cuh"

namespace polar_b200 {
namespace {

constexpr int kThreads = 256;

// Rows of any length, any alignment: three passes over a row that the caches hold.
__global__ void __launch_bounds__(kThreads) norm_kernel(const float* in, const float* gamma, const float* beta, float eps,
                                                        uint64_t cols, float* out, float* mean_out, float* rstd_out) {
  pdl_enter();
  __shared__ float slots[2][kThreads / 32];
  const float* x = in + blockIdx.x * cols;
  float s[1] = {0.f};
  for (uint64_t c = threadIdx.x; c < cols; c += kThreads) s[0] += x[c];
  block_sums<kThreads>(s, slots[0]);
  const float mean = s[0] / (float)cols;
  s[0] = 0.f;
  for (uint64_t c = threadIdx.x; c < cols; c += kThreads) {
    const float d = x[c] - mean;
    s[0] += d * d;
  }
  block_sums<kThreads>(s, slots[1]);
  const float rstd = 1.0f / sqrtf(s[0] / (float)cols + eps);
  for (uint64_t c = threadIdx.x; c < cols; c += kThreads)
    out[blockIdx.x * cols + c] = (x[c] - mean) * rstd * (gamma ? gamma[c] : 1.f) + (beta ? beta[c] : 0.f);
  if (threadIdx.x == 0) {
    if (mean_out) mean_out[blockIdx.x] = mean;
    if (rstd_out) rstd_out[blockIdx.x] = rstd;
  }
}

// Backward, rows of any length: the gradient at the input.
__global__ void __launch_bounds__(kThreads) norm_grad_in_kernel(const float* gradient, const float* in, const float* gamma,
                                                                const float* mean, const float* rstd, uint64_t cols, float* din) {
  pdl_enter();
  __shared__ float slots[2 * kThreads / 32];
  const uint64_t at = blockIdx.x * cols;
  const float m = mean[blockIdx.x], r = rstd[blockIdx.x];
  float s[2] = {0.f, 0.f};
  for (uint64_t c = threadIdx.x; c < cols; c += kThreads) {
    const float q = gradient[at + c] * (gamma ? gamma[c] : 1.f);
    s[0] += q;
    s[1] += q * ((in[at + c] - m) * r);
  }
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

// The partial sums of `parts` stretches of rows, in their order.
__global__ void __launch_bounds__(kThreads) norm_grad_finish_kernel(const float* partials, uint32_t parts, uint64_t cols, float* dgamma,
                                                                    float* dbeta) {
  pdl_enter();
  const uint64_t c = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
  if (c >= cols) return;
  float* out = blockIdx.y ? dbeta : dgamma;
  if (!out) return;
  float s = 0.f;
  for (uint32_t p = 0; p < parts; ++p) s += partials[(2ull * p + blockIdx.y) * cols + c];
  out[c] = s;
}

constexpr uint64_t kMaxCols = 1ull << 31, kMaxRows = 0x7fffffffull;

// Stretches of rows whose sums over the rows are kept apart.
uint64_t stretches(uint64_t rows) {
  const uint64_t n = (rows + 63) / 64;
  return n < 256 ? n : 256;
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
  return launch("flayernorm", norm_kernel, dim3((unsigned)rows), kThreads, 0, as_stream(stream), in, gamma, beta, eps, cols, out, mean,
                rstd);
}

uint64_t polar_b200_flayernorm_grad_workspace_bytes(uint64_t rows, uint64_t cols) {
  if (rows == 0 || cols == 0 || rows > kMaxRows || cols > kMaxCols) return 0;
  return stretches(rows) * 2 * cols * sizeof(float);
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
  if (dgamma || dbeta) {
    const uint64_t need = polar_b200_flayernorm_grad_workspace_bytes(rows, cols);
    if (workspace && (workspace_bytes < need || !aligned16(workspace)))
      return fail(POLAR_B200_ERR_WORKSPACE, "workspace too small or not 16-byte aligned");
    void* own = nullptr;
    if (!workspace) {
      cudaError_t e = scratch_alloc(&own, need, st);
      if (e != cudaSuccess) return fail(POLAR_B200_ERR_CUDA, "scratch (sums over rows)", e);
    }
    float* partials = static_cast<float*>(workspace ? workspace : own);
    const uint64_t parts = stretches(rows), stretch = (rows + parts - 1) / parts;
    const unsigned wide = (unsigned)((cols + kThreads - 1) / kThreads);
    rc = launch("flayernorm_grad_columns", norm_grad_columns_kernel, dim3(wide, (unsigned)parts), kThreads, 0, st, gradient, in, mean, rstd,
                rows, cols, stretch, partials);
    if (rc == POLAR_B200_OK)
      rc = launch("flayernorm_grad_sum", norm_grad_finish_kernel, dim3(wide, 2), kThreads, 0, st, partials, (uint32_t)parts, cols, dgamma,
                  dbeta);
    if (own) {
      cudaError_t e = scratch_free(own, st);
      if (rc == POLAR_B200_OK && e != cudaSuccess) rc = fail(POLAR_B200_ERR_CUDA, "returning scratch", e);
    }
    if (rc) return rc;
  }
  return launch("flayernorm_grad", norm_grad_in_kernel, dim3((unsigned)rows), kThreads, 0, st, gradient, in, gamma, mean, rstd, cols, din);
}

}  // extern "C"
