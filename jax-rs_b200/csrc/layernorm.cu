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
//
// Bound by HBM: 8 bytes an element forward, 12 backward.  A row is read once
// and held in registers, by a warp (narrow rows) or by a block; the variance is
// of the centred values, so that a mean far from zero costs it no more than the
// mean's own rounding in f32 does.  Backward, a
// block keeps its columns' sums over all of its rows in registers and loads the
// next row while it reduces the present one; the blocks' sums are added in
// order by a second kernel.
//
// Forward, 16384 x 4096: 86 us alone, 6.2 TB/s, and 92 in a row of calls, with four vectors in each of 256 threads; two
// in 512 take 122, one in 1024 142, eight in 128 88 (a block waits for its row's
// sums twice, so several blocks per SM must be in different places; where rows are
// few it is the other way).  Backward, 16384 x 2048: 60 us alone, 6.7 TB/s, the join behind it 8 alone,
// and 71 for both in a row of calls (67 in a graph); two blocks
// per SM instead of three take 6 more.  Beyond 8192 columns a cluster shares a row of the
// gradient: 4096 x 16384 take 92 us forward and 172 backward, 4096 x 12000 76 and 152 (floors 82 and 123,
// 60 and 90).  Beyond 16384 a row is read again from L2: 2000 x 20000 take 82 and 221 us (49 and 73).
// Rows that are not aligned are read value by value, and 513 to 640 and 1025 to 1280 columns
// take five of them a thread instead of eight: 30000 x 1111 59 us against 76 forward, 75 against 87 backward, 60000 x 637
// 57 against 71 and 80 against 90.  (No other width has been tried so.)
#include <math.h>

#include <algorithm>

#include "jx_common.cuh"
#include "nn_common.cuh"

namespace {

using jxn::warp_sum;

// Sum over the T threads that share a row (a warp, or the whole block: one slot
// of sm per warp).
template <int T>
__device__ __forceinline__ float row_sum(float v, float* sm) {
  v = warp_sum(v);
  if constexpr (T > 32) {
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sm[threadIdx.x & (T / 32 - 1)];
#pragma unroll
    for (int o = T / 64; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  }
  return v;
}

// This thread's N vectors of V columns of a row: vector i starts at column
// (i * T + t) * V; zeros behind the end.
template <int T, int V, int N>
__device__ __forceinline__ void load_row(float (&x)[N * V], const float* p, int t, int cols) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = (i * T + t) * V;
    if constexpr (V == 4) {
      const float4 f = c < cols ? *reinterpret_cast<const float4*>(p + c) : make_float4(0.f, 0.f, 0.f, 0.f);
      x[4 * i] = f.x;
      x[4 * i + 1] = f.y;
      x[4 * i + 2] = f.z;
      x[4 * i + 3] = f.w;
    } else {
      x[i] = c < cols ? p[c] : 0.0f;
    }
  }
}
template <int T, int V, int N>
__device__ __forceinline__ void store_row(float* p, const float (&x)[N * V], int t, int cols) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = (i * T + t) * V;
    if (c < cols) {
      if constexpr (V == 4)
        *reinterpret_cast<float4*>(p + c) = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
      else
        p[c] = x[i];
    }
  }
}
template <int T, int V, int N>
__device__ __forceinline__ void fill_row(float (&x)[N * V], const float* p, int t, int cols, float value) {
  if (p) {
    load_row<T, V, N>(x, p, t, cols);
  } else {
#pragma unroll
    for (int i = 0; i < N * V; ++i) x[i] = value;
  }
}

constexpr int block_of(int T) { return T == 32 ? 256 : T; }

// T threads per row.
template <int T, int V, int N>
__global__ void __launch_bounds__(block_of(T), T == 512 && N * V >= 16 ? 2 : 1)
    ln_fwd_kernel(const float* x, const float* __restrict__ gamma, const float* __restrict__ beta, float* y,
                  float* __restrict__ mean_out, float* __restrict__ rstd_out, long long rows, int cols, long long ldx,
                  long long ldy, float eps) {
  __shared__ float sm[2][32];
  const int t = threadIdx.x % T;
  const long long r = (long long)blockIdx.x * (block_of(T) / T) + threadIdx.x / T;
  if (r >= rows) return;  // whole warps; a block with T > 32 has one row
  float v[N * V];
  load_row<T, V, N>(v, x + r * ldx, t, cols);
  const float inv = 1.0f / (float)cols;
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < N * V; ++i) s += v[i];
  const float mean = row_sum<T>(s, sm[0]) * inv;
  float q = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const bool in = (i * T + t) * V < cols;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      v[i * V + e] -= mean;
      if (in) q = fmaf(v[i * V + e], v[i * V + e], q);
    }
  }
  const float rstd = 1.0f / sqrtf(row_sum<T>(q, sm[1]) * inv + eps);
#pragma unroll
  for (int i = 0; i < N; ++i) {  // gamma and beta come from L1; loaded earlier they cost the registers of other rows
    const int c = (i * T + t) * V;
    float g[V], b[V], out[V];
    fill_row<1, V, 1>(g, gamma ? gamma + c : nullptr, 0, cols - c, 1.0f);
    fill_row<1, V, 1>(b, beta ? beta + c : nullptr, 0, cols - c, 0.0f);
#pragma unroll
    for (int e = 0; e < V; ++e) out[e] = fmaf(v[i * V + e] * rstd, g[e], b[e]);
    store_row<1, V, 1>(y + r * ldy + c, out, 0, cols - c);
  }
  if (t == 0) {
    if (mean_out) mean_out[r] = mean;
    if (rstd_out) rstd_out[r] = rstd;
  }
}

// Rows too wide for a block's registers: read three times, from L2 after the first.
constexpr int WIDE = 1024;
__global__ void __launch_bounds__(WIDE)
    ln_fwd_wide_kernel(const float* x, const float* __restrict__ gamma, const float* __restrict__ beta, float* y,
                       float* __restrict__ mean_out, float* __restrict__ rstd_out, int cols, long long ldx,
                       long long ldy, float eps) {
  __shared__ float sm[2][32];
  const long long r = blockIdx.x;
  const float* in = x + r * ldx;
  float* out = y + r * ldy;
  float s = 0.0f;
  for (int c = threadIdx.x; c < cols; c += WIDE) s += in[c];
  const float mean = row_sum<WIDE>(s, sm[0]) / (float)cols;
  float q = 0.0f;
  for (int c = threadIdx.x; c < cols; c += WIDE) {
    const float d = in[c] - mean;
    q = fmaf(d, d, q);
  }
  const float rstd = 1.0f / sqrtf(row_sum<WIDE>(q, sm[1]) / (float)cols + eps);
  for (int c = threadIdx.x; c < cols; c += WIDE)
    out[c] = fmaf((in[c] - mean) * rstd, gamma ? gamma[c] : 1.0f, beta ? beta[c] : 0.0f);
  if (threadIdx.x == 0) {
    if (mean_out) mean_out[r] = mean;
    if (rstd_out) rstd_out[r] = rstd;
  }
}

// To the same place in another block of the cluster.
__device__ __forceinline__ void store_remote(float* p, uint32_t rank, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(jxd::mapa_shared(p, rank)), "f"(v) : "memory");
}

// dx (may be NULL) of the rows blockIdx.x * RPB + .., step gridDim.x * RPB, and the
// block's column sums into part[blockIdx.x / CL][2][cols] (may be NULL).  The next row is
// loaded before the present one is reduced.  CL = 2: a row is a cluster's, whose two
// blocks tell each other their warps' sums: 4096 rows of 16384 in 177 us, 4.5 TB/s, against 342
// where the row is read twice and the column sums have a pass of their own, and 280 for
// clusters of four, two to an SM.
template <int T, int V, int N, int PER_SM, int CL>
__global__ void __launch_bounds__(block_of(T), PER_SM)
    ln_bwd_kernel(const float* dy, const float* __restrict__ x, const float* __restrict__ gamma,
                  const float* __restrict__ mean, const float* __restrict__ rstd, float* dx, float* __restrict__ part,
                  long long rows, int cols, long long lddy, long long ldx, long long lddx) {
  constexpr int RPB = block_of(T) / T;  // rows per block at a time
  __shared__ float sm[2][2][32];
  __shared__ float join[T == 32 ? 7 * 2 * 32 * N * V : 1];
  constexpr int COL_T = T * CL, SUMS = COL_T / 32;  // threads and warps of a row
  const uint32_t rank = CL > 1 ? jxd::cluster_ctarank() : 0;
  const unsigned block = blockIdx.x / CL;
  const int t = threadIdx.x % T + (int)rank * T, sub = threadIdx.x / T;
  const long long step = (long long)(gridDim.x / CL) * RPB;
  const float inv = 1.0f / (float)cols;
  if constexpr (CL > 1) jxd::cluster_sync_all();  // the other block runs
  float g[N * V], dg[N * V], db[N * V], xv[N * V], dv[N * V];
  fill_row<COL_T, V, N>(g, gamma, t, cols, 1.0f);
#pragma unroll
  for (int i = 0; i < N * V; ++i) dg[i] = db[i] = 0.0f;
  long long r = (long long)block * RPB + sub;
  float m = 0.0f, rs = 0.0f;
  if (r < rows) {
    load_row<COL_T, V, N>(dv, dy + r * lddy, t, cols);
    load_row<COL_T, V, N>(xv, x + r * ldx, t, cols);
    m = mean[r];
    rs = rstd[r];
  }
  for (int buf = 0; r < rows; r += step, buf ^= 1) {
    float xn[N * V], dn[N * V], mn = 0.0f, rn = 0.0f;
    const long long r1 = r + step;
    if (r1 < rows) {
      load_row<COL_T, V, N>(dn, dy + r1 * lddy, t, cols);
      load_row<COL_T, V, N>(xn, x + r1 * ldx, t, cols);
      mn = mean[r1];
      rn = rstd[r1];
    }
    // Behind the end x is zero, and (0 - m) * rs may be infinite where no column's xhat is.
    // (A select per element instead takes 75.5 us where this takes 71, 16384 x 2048.)
    if (isinf(m * rs)) {
#pragma unroll
      for (int i = 0; i < N * V; ++i)
        if (((i / V) * COL_T + t) * V >= cols) xv[i] = m;
    }
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < N * V; ++i) {  // behind the end dy is zero and xhat finite
      xv[i] = (xv[i] - m) * rs;
      dg[i] = fmaf(dv[i], xv[i], dg[i]);
      db[i] += dv[i];
      dv[i] *= g[i];
      s1 += dv[i];
      s2 = fmaf(dv[i], xv[i], s2);
    }
    if (dx) {
      s1 = warp_sum(s1);
      s2 = warp_sum(s2);
      if constexpr (T > 32) {
        if ((threadIdx.x & 31) == 0) {
          const int w = (int)rank * (T / 32) + (threadIdx.x >> 5);
          sm[buf][0][w] = s1;
          sm[buf][1][w] = s2;
          if constexpr (CL > 1) {
            store_remote(&sm[buf][0][w], rank ^ 1, s1);
            store_remote(&sm[buf][1][w], rank ^ 1, s2);
          }
        }
        // one per row: the other buffer is read before the next one's
        if constexpr (CL > 1) jxd::cluster_sync_all();
        else __syncthreads();
        s1 = sm[buf][0][threadIdx.x & (SUMS - 1)];
        s2 = sm[buf][1][threadIdx.x & (SUMS - 1)];
#pragma unroll
        for (int o = SUMS / 2; o > 0; o >>= 1) {
          s1 += __shfl_xor_sync(0xffffffffu, s1, o);
          s2 += __shfl_xor_sync(0xffffffffu, s2, o);
        }
      }
      const float c1 = s1 * inv, c2 = s2 * inv;
      float out[N * V];
#pragma unroll
      for (int i = 0; i < N * V; ++i) out[i] = (dv[i] - c1 - xv[i] * c2) * rs;
      store_row<COL_T, V, N>(dx + r * lddx, out, t, cols);
    }
#pragma unroll
    for (int i = 0; i < N * V; ++i) {
      xv[i] = xn[i];
      dv[i] = dn[i];
    }
    m = mn;
    rs = rn;
  }
  if (!part) return;
  asm volatile("griddepcontrol.launch_dependents;");
  if constexpr (T == 32) {  // the block's warps have the same columns
    constexpr int W = 2 * 32 * N * V;
    if (sub > 0) {
#pragma unroll
      for (int i = 0; i < N * V; ++i) {
        join[(sub - 1) * W + i * 32 + t] = dg[i];
        join[(sub - 1) * W + (N * V + i) * 32 + t] = db[i];
      }
    }
    __syncthreads();
    if (sub > 0) return;
    for (int w = 0; w < 7; ++w) {
#pragma unroll
      for (int i = 0; i < N * V; ++i) {
        dg[i] += join[w * W + i * 32 + t];
        db[i] += join[w * W + (N * V + i) * 32 + t];
      }
    }
  }
  float* out = part + (long long)block * 2 * cols;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = (i * COL_T + t) * V;
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (c + e < cols) {
        out[c + e] = dg[i * V + e];
        out[cols + c + e] = db[i * V + e];
      }
  }
}

// Rows too wide for registers: dx with the row read twice, and column sums over chunks of rows.
__global__ void __launch_bounds__(WIDE)
    ln_dx_wide_kernel(const float* dy, const float* __restrict__ x, const float* __restrict__ gamma,
                      const float* __restrict__ mean, const float* __restrict__ rstd, float* dx, int cols,
                      long long lddy, long long ldx, long long lddx) {
  __shared__ float sm[2][32];
  const long long r = blockIdx.x;
  const float m = mean[r], rs = rstd[r];
  float s1 = 0.0f, s2 = 0.0f;
  for (int c = threadIdx.x; c < cols; c += WIDE) {
    const float g = dy[r * lddy + c] * (gamma ? gamma[c] : 1.0f);
    s1 += g;
    s2 = fmaf(g, (x[r * ldx + c] - m) * rs, s2);
  }
  const float c1 = row_sum<WIDE>(s1, sm[0]) / (float)cols;
  const float c2 = row_sum<WIDE>(s2, sm[1]) / (float)cols;
  for (int c = threadIdx.x; c < cols; c += WIDE) {
    const float g = dy[r * lddy + c] * (gamma ? gamma[c] : 1.0f);
    dx[r * lddx + c] = (g - c1 - (x[r * ldx + c] - m) * rs * c2) * rs;
  }
}
__global__ void ln_col_partial_kernel(const float* __restrict__ dy, const float* __restrict__ x,
                                      const float* __restrict__ mean, const float* __restrict__ rstd,
                                      float* __restrict__ part, long long rows, int cols, long long lddy,
                                      long long ldx, long long chunk) {
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= cols) return;
  const long long r0 = (long long)blockIdx.y * chunk, r1 = min(r0 + chunk, rows);
  float a = 0.0f, b = 0.0f;
#pragma unroll 4
  for (long long r = r0; r < r1; ++r) {
    const float d = dy[r * lddy + c];
    a = fmaf(d, (x[r * ldx + c] - mean[r]) * rstd[r], a);
    b += d;
  }
  part[(long long)blockIdx.y * 2 * cols + c] = a;
  part[(long long)blockIdx.y * 2 * cols + cols + c] = b;
}

// dgamma and dbeta from part[parts][2 * cols]: 32 columns a block, 32 warps that
// take every 32nd part, then the warps in order.
__global__ void __launch_bounds__(1024) ln_join_kernel(const float* part, float* __restrict__ dgamma,
                                                      float* __restrict__ dbeta, int parts, int cols) {
  __shared__ float sm[32][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const long long c = (long long)blockIdx.x * 32 + lane;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the parts are complete behind it
  float a = 0.0f;
  if (c < 2LL * cols) {
#pragma unroll 8
    for (int p = w; p < parts; p += 32) a += part[(long long)p * 2 * cols + c];
  }
  sm[w][lane] = a;
  __syncthreads();
  // warp w adds column w's 32 sums
  a = warp_sum(sm[lane][w]);
  const long long cc = (long long)blockIdx.x * 32 + w;
  if (lane == 0 && cc < 2LL * cols) {
    float* out = cc < cols ? dgamma : dbeta;
    if (out) out[cc < cols ? cc : cc - cols] = a;
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

struct FwdArgs {
  const float *x, *gamma, *beta;
  float *y, *mean, *rstd;
  long long rows;
  int cols;
  long long ldx, ldy;
  float eps;
};
template <int T, int V, int N>
void fwd(const FwdArgs& a, cudaStream_t st) {
  constexpr int RPB = block_of(T) / T;
  ln_fwd_kernel<T, V, N><<<(unsigned)((a.rows + RPB - 1) / RPB), block_of(T), 0, st>>>(
      a.x, a.gamma, a.beta, a.y, a.mean, a.rstd, a.rows, a.cols, a.ldx, a.ldy, a.eps);
}

struct BwdArgs {
  const float *dy, *x, *gamma, *mean, *rstd;
  float *dx, *dgamma, *dbeta;
  long long rows;
  int cols;
  long long lddy, ldx, lddx;
};

int join(const BwdArgs& a, const float* part, int parts, cudaStream_t st) {
  // its blocks may start while the last rows are summed; they wait before they read
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((2LL * a.cols + 31) / 32));
  cfg.blockDim = dim3(1024);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  JX_CUDA(cudaLaunchKernelEx(&cfg, ln_join_kernel, part, a.dgamma, a.dbeta, parts, a.cols));
  return JX_OK;
}

// PER_SM: blocks per SM that the grid is made for.
template <int T, int V, int N, int PER_SM, int CL = 1>
int bwd(const BwdArgs& a, cudaStream_t st) {
  constexpr int RPB = block_of(T) / T;
  const int parts = (int)std::min<long long>((a.rows + RPB - 1) / RPB, (long long)(jx::num_sms() / CL) * PER_SM);
  const bool sums = a.dgamma || a.dbeta;
  void* part = nullptr;
  if (sums)
    if (int rc = jx::scratch_get(sizeof(float) * 2 * (size_t)parts * a.cols, &part, st)) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(parts * CL));
  cfg.blockDim = dim3(block_of(T));
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = CL;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = CL > 1;
  const cudaError_t e =
      cudaLaunchKernelEx(&cfg, ln_bwd_kernel<T, V, N, PER_SM, CL>, a.dy, a.x, a.gamma, a.mean, a.rstd, a.dx,
                         static_cast<float*>(part), a.rows, a.cols, a.lddy, a.ldx, a.lddx);
  int rc = e == cudaSuccess ? JX_OK : jx::check_cuda(e, "ln_bwd_kernel");
  if (!rc && sums) rc = join(a, static_cast<const float*>(part), parts, st);
  jx::scratch_release(part, st);
  return rc;
}

int bwd_wide(const BwdArgs& a, cudaStream_t st) {
  if (a.dgamma || a.dbeta) {  // before dx, which may be dy
    const long long chunk = std::max<long long>(16, (a.rows + 255) / 256);
    const int chunks = (int)((a.rows + chunk - 1) / chunk);
    void* part = nullptr;
    if (int rc = jx::scratch_get(sizeof(float) * 2 * (size_t)chunks * a.cols, &part, st)) return rc;
    ln_col_partial_kernel<<<dim3((unsigned)((a.cols + 127) / 128), chunks), 128, 0, st>>>(
        a.dy, a.x, a.mean, a.rstd, static_cast<float*>(part), a.rows, a.cols, a.lddy, a.ldx, chunk);
    const cudaError_t e = cudaGetLastError();
    int rc = e == cudaSuccess ? JX_OK : jx::check_cuda(e, "ln_col_partial_kernel");
    if (!rc) rc = join(a, static_cast<const float*>(part), chunks, st);
    jx::scratch_release(part, st);
    if (rc) return rc;
  }
  if (a.dx) {
    ln_dx_wide_kernel<<<(unsigned)a.rows, WIDE, 0, st>>>(a.dy, a.x, a.gamma, a.mean, a.rstd, a.dx, a.cols, a.lddy,
                                                         a.ldx, a.lddx);
    JX_LAUNCH_CHECK("ln_dx_wide_kernel");
  }
  return JX_OK;
}

}  // namespace

extern "C" {

int jx_layernorm_f32(const float* x, const float* gamma, const float* beta, float* y, float* mean_out, float* rstd_out,
                     int64_t rows, int64_t cols, int64_t ldx, int64_t ldy, float epsilon, jx_stream_t stream) {
  JX_TRACE("jx_layernorm_f32");
  JX_REQUIRE(rows >= 0 && rows < (1LL << 31) && cols >= 1 && cols < (1LL << 30), "layernorm: bad size");
  JX_REQUIRE(ldx >= cols && ldy >= cols, "layernorm: row stride smaller than the row");
  JX_REQUIRE(epsilon >= 0.0f, "layernorm: epsilon must not be negative");
  if (rows == 0) return JX_OK;
  JX_REQUIRE(x && y, "layernorm: NULL pointer");
  JX_REQUIRE(y != x || ldy == ldx, "layernorm: in place needs equal row strides");
  cudaStream_t st = jx::as_stream(stream);
  const FwdArgs a = {x, gamma, beta, y, mean_out, rstd_out, rows, (int)cols, ldx, ldy, epsilon};
  const bool vec = !(cols & 3) && !(ldx & 3) && !(ldy & 3) && aligned16(x) && aligned16(y) && aligned16(gamma) &&
                   aligned16(beta);
  // few rows: as many threads to a row as it has vectors, so that one load each covers it
  const bool few = rows < jx::num_sms();
  if (vec) {
    if (cols <= 128) fwd<32, 4, 1>(a, st);
    else if (cols <= 256) fwd<32, 4, 2>(a, st);
    else if (cols <= 512) few ? fwd<128, 4, 1>(a, st) : fwd<32, 4, 4>(a, st);
    else if (cols <= 1024) few ? fwd<256, 4, 1>(a, st) : fwd<64, 4, 4>(a, st);
    else if (cols <= 2048) few ? fwd<512, 4, 1>(a, st) : fwd<128, 4, 4>(a, st);
    else if (cols <= 4096) few ? fwd<1024, 4, 1>(a, st) : fwd<256, 4, 4>(a, st);
    else if (cols <= 8192) few ? fwd<1024, 4, 2>(a, st) : fwd<512, 4, 4>(a, st);
    else if (cols <= 16384) fwd<512, 4, 8>(a, st);
  } else {
    if (cols <= 128) fwd<32, 1, 4>(a, st);
    else if (cols <= 256) fwd<32, 1, 8>(a, st);
    else if (cols <= 512) fwd<64, 1, 8>(a, st);
    else if (cols <= 640) fwd<128, 1, 5>(a, st);
    else if (cols <= 1024) fwd<128, 1, 8>(a, st);
    else if (cols <= 1280) fwd<256, 1, 5>(a, st);
    else if (cols <= 2048) fwd<256, 1, 8>(a, st);
    else if (cols <= 4096) fwd<256, 1, 16>(a, st);
    else if (cols <= 8192) fwd<512, 1, 16>(a, st);
    else if (cols <= 16384) fwd<512, 1, 32>(a, st);
  }
  if (cols > 16384)
    ln_fwd_wide_kernel<<<(unsigned)rows, WIDE, 0, st>>>(x, gamma, beta, y, mean_out, rstd_out, (int)cols, ldx, ldy,
                                                        epsilon);
  JX_LAUNCH_CHECK("ln_fwd_kernel");
  return JX_OK;
}

int jx_layernorm_bwd_f32(const float* dy, const float* x, const float* gamma, const float* mean, const float* rstd,
                         float* dx, float* dgamma, float* dbeta, int64_t rows, int64_t cols, int64_t lddy, int64_t ldx,
                         int64_t lddx, jx_stream_t stream) {
  JX_TRACE("jx_layernorm_bwd_f32");
  JX_REQUIRE(rows >= 0 && rows < (1LL << 31) && cols >= 1 && cols < (1LL << 30), "layernorm_bwd: bad size");
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
  if (!dx && !dgamma && !dbeta) return JX_OK;
  const BwdArgs a = {dy, x, gamma, mean, rstd, dx, dgamma, dbeta, rows, (int)cols, lddy, ldx, lddx};
  const bool vec = !(cols & 3) && !(lddy & 3) && !(ldx & 3) && (!dx || !(lddx & 3)) && aligned16(dy) && aligned16(x) &&
                   aligned16(dx) && aligned16(gamma);
  if (vec) {
    if (cols <= 128) return bwd<32, 4, 1, 3>(a, st);
    if (cols <= 256) return bwd<32, 4, 2, 2>(a, st);
    if (cols <= 512) return bwd<64, 4, 2, 12>(a, st);
    if (cols <= 1024) return bwd<128, 4, 2, 6>(a, st);
    if (cols <= 2048) return bwd<256, 4, 2, 3>(a, st);
    if (cols <= 4096) return bwd<256, 4, 4, 2>(a, st);
    if (cols <= 8192) return bwd<512, 4, 4, 1>(a, st);
    if (cols <= 16384) return bwd<512, 4, 4, 1, 2>(a, st);
  } else {
    if (cols <= 128) return bwd<32, 1, 4, 3>(a, st);
    if (cols <= 256) return bwd<32, 1, 8, 2>(a, st);
    if (cols <= 512) return bwd<64, 1, 8, 12>(a, st);
    if (cols <= 640) return bwd<128, 1, 5, 8>(a, st);
    if (cols <= 1024) return bwd<128, 1, 8, 6>(a, st);
    if (cols <= 1280) return bwd<256, 1, 5, 4>(a, st);
    if (cols <= 2048) return bwd<256, 1, 8, 3>(a, st);
    if (cols <= 4096) return bwd<256, 1, 16, 2>(a, st);
    if (cols <= 8192) return bwd<512, 1, 16, 1>(a, st);
    if (cols <= 16384) return bwd<512, 1, 16, 1, 2>(a, st);
  }
  return bwd_wide(a, st);
}

}  // extern "C"
