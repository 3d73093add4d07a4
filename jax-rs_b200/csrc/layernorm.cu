// layernorm.cu -- layer norm over the last axis, forward and backward.
//
//   nn::layer_norm src/nn.rs:712-725 (one vector there; here every row of a
//   matrix, with gamma and beta).  The reference has no gradient for it.
//
//   forward   mean = sum(x) / n, var = sum((x - mean)^2) / n,
//             rstd = 1 / sqrt(var + eps), y = (x - mean) * rstd * gamma + beta
//   backward  xhat = (x - mean) * rstd, g = dy * gamma,
//             dx = (g - mean(g) - xhat * mean(g * xhat)) * rstd,
//             dgamma = sum over rows of dy * xhat, dbeta = sum over rows of dy
#include <math.h>

#include <algorithm>

#include "jx_common.cuh"
#include "nn_common.cuh"

namespace {

using jxn::warp_sum;

constexpr int LN_THREADS = 256;

// Sum over the block; every thread gets it.  sm has one slot per warp and is
// free again at the caller's next block_sum with the other buffer.
__device__ __forceinline__ float block_sum(float v, float* sm) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.0f;
#pragma unroll
  for (int w = 0; w < LN_THREADS / 32; ++w) t += sm[w];
  return t;
}

// One block per row, the row read three times (from L1 or L2 after the first).
__global__ void ln_fwd_kernel(const float* __restrict__ x, const float* __restrict__ gamma,
                              const float* __restrict__ beta, float* y, float* __restrict__ mean_out,
                              float* __restrict__ rstd_out, long long rows, int cols, long long ldx, long long ldy,
                              float eps) {
  __shared__ float sm[2][LN_THREADS / 32];
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const float* in = x + r * ldx;
    float* out = y + r * ldy;
    float s = 0.0f;
    for (int c = threadIdx.x; c < cols; c += LN_THREADS) s += in[c];
    const float mean = block_sum(s, sm[0]) / (float)cols;
    float q = 0.0f;
    for (int c = threadIdx.x; c < cols; c += LN_THREADS) {
      const float d = in[c] - mean;
      q += d * d;
    }
    const float rstd = 1.0f / sqrtf(block_sum(q, sm[1]) / (float)cols + eps);
    for (int c = threadIdx.x; c < cols; c += LN_THREADS) {
      float v = (in[c] - mean) * rstd;
      if (gamma) v *= gamma[c];
      if (beta) v += beta[c];
      out[c] = v;
    }
    if (threadIdx.x == 0) {
      if (mean_out) mean_out[r] = mean;
      if (rstd_out) rstd_out[r] = rstd;
    }
    __syncthreads();
  }
}

__global__ void ln_dx_kernel(const float* dy, const float* __restrict__ x, const float* __restrict__ gamma,
                             const float* __restrict__ mean, const float* __restrict__ rstd, float* dx,
                             long long rows, int cols, long long lddy, long long ldx, long long lddx) {
  __shared__ float sm[2][LN_THREADS / 32];
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const float m = mean[r], rs = rstd[r];
    float s1 = 0.0f, s2 = 0.0f;
    for (int c = threadIdx.x; c < cols; c += LN_THREADS) {
      const float g = dy[r * lddy + c] * (gamma ? gamma[c] : 1.0f);
      s1 += g;
      s2 += g * ((x[r * ldx + c] - m) * rs);
    }
    const float c1 = block_sum(s1, sm[0]) / (float)cols;
    const float c2 = block_sum(s2, sm[1]) / (float)cols;
    for (int c = threadIdx.x; c < cols; c += LN_THREADS) {
      const float g = dy[r * lddy + c] * (gamma ? gamma[c] : 1.0f);
      dx[r * lddx + c] = (g - c1 - (x[r * ldx + c] - m) * rs * c2) * rs;
    }
    __syncthreads();
  }
}

// Column sums over chunks of rows, then over the chunks in order.
__global__ void ln_col_partial_kernel(const float* __restrict__ dy, const float* __restrict__ x,
                                      const float* __restrict__ mean, const float* __restrict__ rstd,
                                      float* __restrict__ part, long long rows, int cols, long long lddy,
                                      long long ldx, long long chunk) {
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= cols) return;
  const long long r0 = (long long)blockIdx.y * chunk, r1 = min(r0 + chunk, rows);
  float a = 0.0f, b = 0.0f;
  for (long long r = r0; r < r1; ++r) {
    const float d = dy[r * lddy + c];
    a += d * ((x[r * ldx + c] - mean[r]) * rstd[r]);
    b += d;
  }
  part[(long long)blockIdx.y * 2 * cols + c] = a;
  part[(long long)blockIdx.y * 2 * cols + cols + c] = b;
}
__global__ void ln_col_final_kernel(const float* __restrict__ part, float* __restrict__ dgamma,
                                    float* __restrict__ dbeta, int chunks, int cols) {
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= 2 * cols) return;
  float acc = 0.0f;
  for (int k = 0; k < chunks; ++k) acc += part[(long long)k * 2 * cols + c];
  float* out = c < cols ? dgamma : dbeta;
  if (out) out[c < cols ? c : c - cols] = acc;
}

}  // namespace

extern "C" {

int jx_layernorm_f32(const float* x, const float* gamma, const float* beta, float* y, float* mean_out, float* rstd_out,
                     int64_t rows, int64_t cols, int64_t ldx, int64_t ldy, float epsilon, jx_stream_t stream) {
  JX_TRACE("jx_layernorm_f32");
  JX_REQUIRE(rows >= 0 && cols >= 1 && cols < (1LL << 31) - 8192, "layernorm: bad size");
  JX_REQUIRE(ldx >= cols && ldy >= cols, "layernorm: row stride smaller than the row");
  JX_REQUIRE(epsilon >= 0.0f, "layernorm: epsilon must not be negative");
  if (rows == 0) return JX_OK;
  JX_REQUIRE(x && y, "layernorm: NULL pointer");
  JX_REQUIRE(y != x || ldy == ldx, "layernorm: in place needs equal row strides");
  const int grid = (int)std::min<long long>(rows, (long long)jx::num_sms() * 8);
  ln_fwd_kernel<<<grid, LN_THREADS, 0, jx::as_stream(stream)>>>(x, gamma, beta, y, mean_out, rstd_out, rows, (int)cols,
                                                                ldx, ldy, epsilon);
  JX_LAUNCH_CHECK("ln_fwd_kernel");
  return JX_OK;
}

int jx_layernorm_bwd_f32(const float* dy, const float* x, const float* gamma, const float* mean, const float* rstd,
                         float* dx, float* dgamma, float* dbeta, int64_t rows, int64_t cols, int64_t lddy, int64_t ldx,
                         int64_t lddx, jx_stream_t stream) {
  JX_TRACE("jx_layernorm_bwd_f32");
  JX_REQUIRE(rows >= 0 && cols >= 1 && cols < (1LL << 30), "layernorm_bwd: bad size");
  JX_REQUIRE(lddy >= cols && ldx >= cols && (!dx || lddx >= cols), "layernorm_bwd: row stride smaller than the row");
  cudaStream_t st = jx::as_stream(stream);
  if (rows == 0) {
    if (dgamma) JX_CUDA(cudaMemsetAsync(dgamma, 0, sizeof(float) * cols, st));
    if (dbeta) JX_CUDA(cudaMemsetAsync(dbeta, 0, sizeof(float) * cols, st));
    return JX_OK;
  }
  JX_REQUIRE(dy && x && mean && rstd, "layernorm_bwd: NULL pointer");
  JX_REQUIRE(dx != x, "layernorm_bwd: dx must not be x");
  JX_REQUIRE(dx != dy || lddx == lddy, "layernorm_bwd: in place needs equal row strides");
  if (dgamma || dbeta) {
    const long long chunk = std::max<long long>(64, (rows + 255) / 256);
    const int chunks = (int)((rows + chunk - 1) / chunk);
    void* part = nullptr;
    if (int rc = jx::scratch_get(sizeof(float) * 2 * (size_t)chunks * cols, &part, st)) return rc;
    float* pp = static_cast<float*>(part);
    ln_col_partial_kernel<<<dim3((unsigned)((cols + 127) / 128), chunks), 128, 0, st>>>(
        dy, x, mean, rstd, pp, rows, (int)cols, lddy, ldx, chunk);
    ln_col_final_kernel<<<(unsigned)((2 * cols + 127) / 128), 128, 0, st>>>(pp, dgamma, dbeta, chunks, (int)cols);
    const cudaError_t e = cudaGetLastError();
    jx::scratch_release(part, st);
    if (e != cudaSuccess) return jx::check_cuda(e, "layernorm_bwd column kernels");
  }
  if (dx) {
    const int grid = (int)std::min<long long>(rows, (long long)jx::num_sms() * 8);
    ln_dx_kernel<<<grid, LN_THREADS, 0, st>>>(dy, x, gamma, mean, rstd, dx, rows, (int)cols, lddy, ldx, lddx);
    JX_LAUNCH_CHECK("ln_dx_kernel");
  }
  return JX_OK;
}

}  // extern "C"
