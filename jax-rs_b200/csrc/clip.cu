// clip.cu -- the global gradient norm over many tensors, and clipping by it:
// the step before optim::adam_update (src/optim.rs:138-189).  No reference
// counterpart.
//
//   norm = sqrt(sum over tensors and elements of g^2)
//   out  = g * min(1, max_norm / (norm + 1e-6))
//
// Squares are taken and summed in f64: no gradient's square over- or
// underflows, and the sum's order (fixed by the sizes alone) does not matter
// at f32 precision.  The conversions and f64 multiply-adds are far below the
// SM's rate at HBM speed (six elements per SM and clock).
#include <algorithm>

#include "jx_common.cuh"

namespace {

constexpr int CL_THREADS = 256;
constexpr int CL_TENSORS = 128;       // tensors of one launch: the table travels in the launch's parameters
constexpr long long CL_CHUNK = 8192;  // elements of one tensor that a block takes at a time
constexpr int CL_MAX_PARTS = 1 << 20;

struct ClipTable {
  const float* in[CL_TENSORS];
  float* out[CL_TENSORS];
  long long size[CL_TENSORS];
  long long first[CL_TENSORS + 1];  // chunks before this tensor's first
  int count;
};

// The tensor that chunk c belongs to: the last one with first[i] <= c
// (tensors without elements have no chunk: their first equals the next one's).
__device__ __forceinline__ int tensor_of(const ClipTable& t, long long c) {
  int lo = 0, hi = t.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.first[mid] <= c) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ double block_sum_f64(double v) {
  __shared__ double sm[CL_THREADS / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0.0;
#pragma unroll
  for (int w = 0; w < CL_THREADS / 32; ++w) t += sm[w];
  return t;
}

// part[blockIdx.x] = the squares of this block's chunks.
__global__ void __launch_bounds__(CL_THREADS) norm_partial_kernel(const __grid_constant__ ClipTable t,
                                                                 double* __restrict__ part) {
  double acc = 0.0;
  for (long long c = blockIdx.x; c < t.first[t.count]; c += gridDim.x) {
    const int i = tensor_of(t, c);
    const long long at = (c - t.first[i]) * CL_CHUNK;
    const long long n = min(CL_CHUNK, t.size[i] - at);
    const float* in = t.in[i] + at;
    for (long long k = threadIdx.x; k < n; k += CL_THREADS) acc += (double)in[k] * (double)in[k];
  }
  const double s = block_sum_f64(acc);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

__global__ void __launch_bounds__(CL_THREADS) norm_final_kernel(double* __restrict__ part, int parts,
                                                               float* __restrict__ norm_out) {
  double acc = 0.0;
  for (int k = threadIdx.x; k < parts; k += CL_THREADS) acc += part[k];
  const double s = sqrt(block_sum_f64(acc));
  if (threadIdx.x == 0) {
    part[parts] = s;
    if (norm_out) norm_out[0] = (float)s;
  }
}

__global__ void __launch_bounds__(CL_THREADS) clip_scale_kernel(const __grid_constant__ ClipTable t,
                                                               const double* __restrict__ norm, float max_norm) {
  const double f = (double)max_norm / (norm[0] + 1e-6);
  const bool keep = f >= 1.0;  // false for a NaN norm: its NaN goes into the outputs
  const float factor = keep ? 1.0f : (float)f;
  for (long long c = blockIdx.x; c < t.first[t.count]; c += gridDim.x) {
    const int i = tensor_of(t, c);
    if (keep && t.out[i] == t.in[i]) continue;
    const long long at = (c - t.first[i]) * CL_CHUNK;
    const long long n = min(CL_CHUNK, t.size[i] - at);
    const float* in = t.in[i] + at;
    float* out = t.out[i] + at;
    for (long long k = threadIdx.x; k < n; k += CL_THREADS) out[k] = in[k] * factor;
  }
}

// The launch's table for tensors i0 .. min(i0 + CL_TENSORS, count) - 1.
void fill(ClipTable& t, const float* const* in, float* const* out, const int64_t* sizes, int i0, int count) {
  t.count = std::min(CL_TENSORS, count - i0);
  t.first[0] = 0;
  for (int k = 0; k < t.count; ++k) {
    t.in[k] = in[i0 + k];
    t.out[k] = out ? out[i0 + k] : nullptr;
    t.size[k] = sizes[i0 + k];
    t.first[k + 1] = t.first[k] + (sizes[i0 + k] + CL_CHUNK - 1) / CL_CHUNK;
  }
}

int check_tensors(const char* what, const float* const* in, float* const* out, bool want_out, const int64_t* sizes,
                  int count) {
  JX_REQUIRE(count >= 0, "%s: negative tensor count", what);
  JX_REQUIRE(count <= CL_MAX_PARTS, "%s: too many tensors", what);
  if (count == 0) return JX_OK;
  JX_REQUIRE(in && sizes && (!want_out || out), "%s: NULL array", what);
  for (int i = 0; i < count; ++i) {
    JX_REQUIRE(sizes[i] >= 0, "%s: tensor %d has negative size", what, i);
    JX_REQUIRE(sizes[i] == 0 || (in[i] && (!want_out || out[i])), "%s: tensor %d has a NULL pointer", what, i);
  }
  return JX_OK;
}

// Norm of all tensors into part[parts] (f64, device) and norm_out.
int norm_launches(const float* const* in, const int64_t* sizes, int count, float* norm_out, double** part_out,
                  int* parts_out, cudaStream_t st) {
  const int launches = (count + CL_TENSORS - 1) / CL_TENSORS;
  const int cap = jx::num_sms() * 8;
  void* p = nullptr;
  if (int rc = jx::scratch_get(sizeof(double) * ((size_t)launches * cap + 1), &p, st)) return rc;
  double* part = static_cast<double*>(p);
  int parts = 0;
  ClipTable t;
  for (int l = 0; l < launches; ++l) {
    fill(t, in, nullptr, sizes, l * CL_TENSORS, count);
    const int grid = (int)std::min<long long>(t.first[t.count], cap);
    if (grid == 0) continue;
    norm_partial_kernel<<<grid, CL_THREADS, 0, st>>>(t, part + parts);
    parts += grid;
  }
  norm_final_kernel<<<1, CL_THREADS, 0, st>>>(part, parts, norm_out);
  *part_out = part;
  *parts_out = parts;
  return JX_OK;
}

}  // namespace

extern "C" {

int jx_grad_norm_f32(const float* const* grads, const int64_t* sizes, int count, float* norm_out, jx_stream_t stream) {
  JX_TRACE("jx_grad_norm_f32");
  if (int rc = check_tensors("grad_norm", grads, nullptr, false, sizes, count)) return rc;
  JX_REQUIRE(norm_out, "grad_norm: NULL pointer");
  cudaStream_t st = jx::as_stream(stream);
  double* part = nullptr;
  int parts = 0;
  if (int rc = norm_launches(grads, sizes, count, norm_out, &part, &parts, st)) return rc;
  const cudaError_t e = cudaGetLastError();
  jx::scratch_release(part, st);
  return e == cudaSuccess ? JX_OK : jx::check_cuda(e, "grad_norm kernels");
}

int jx_clip_grads_f32(const float* const* grads, float* const* outs, const int64_t* sizes, int count, float max_norm,
                      float* norm_out, jx_stream_t stream) {
  JX_TRACE("jx_clip_grads_f32");
  if (int rc = check_tensors("clip_grads", grads, outs, true, sizes, count)) return rc;
  JX_REQUIRE(max_norm >= 0.0f, "clip_grads: max_norm must not be negative");
  cudaStream_t st = jx::as_stream(stream);
  double* part = nullptr;
  int parts = 0;
  if (int rc = norm_launches(grads, sizes, count, norm_out, &part, &parts, st)) return rc;
  ClipTable t;
  for (int i0 = 0; i0 < count; i0 += CL_TENSORS) {
    fill(t, grads, outs, sizes, i0, count);
    const int grid = (int)std::min<long long>(t.first[t.count], (long long)jx::num_sms() * 8);
    if (grid) clip_scale_kernel<<<grid, CL_THREADS, 0, st>>>(t, part + parts, max_norm);
  }
  const cudaError_t e = cudaGetLastError();
  jx::scratch_release(part, st);
  return e == cudaSuccess ? JX_OK : jx::check_cuda(e, "clip_grads kernels");
}

}  // extern "C"
