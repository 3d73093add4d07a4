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
//
// Bound by HBM: 336M values (1.34 GB) take 194 us for the norm, 6.9 TB/s, and 423 us for the
// scaling, 6.2 TB/s of what it moves.
#include <algorithm>

#include "jx_common.cuh"

namespace {

constexpr int CL_THREADS = 256;
constexpr int CL_TENSORS = 128;  // tensors of one launch: the table travels in the launch's parameters
constexpr int CL_MAX_TENSORS = 1 << 20;
// float4 loads (or loads, where a tensor is not aligned) in flight per thread as it scales: 4, 8 and 16 take 673, 652
// and 642 us for norm and scaling of 336M values
constexpr int CL_VECTORS = 16;

// A block takes a tensor's elements in chunks: long ones where there is much to
// do, short ones so that a small model's few kilobytes still reach every SM.
constexpr long long CL_LONG = 4LL * CL_THREADS * CL_VECTORS, CL_SHORT = 4LL * CL_THREADS;

struct ClipTable {
  const float* in[CL_TENSORS];
  float* out[CL_TENSORS];
  long long size[CL_TENSORS];
  long long first[CL_TENSORS + 1];  // chunks before this tensor's first
  long long chunk;
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

struct Chunk {
  const float* in;
  float* out;
  long long n;
  bool vec;
};
__device__ __forceinline__ Chunk chunk_of(const ClipTable& t, long long c) {
  const int i = tensor_of(t, c);
  const long long at = (c - t.first[i]) * t.chunk;
  Chunk r;
  r.in = t.in[i] + at;
  r.out = t.out[i] ? t.out[i] + at : nullptr;
  r.n = min(t.chunk, t.size[i] - at);
  r.vec = ((reinterpret_cast<uintptr_t>(r.in) | reinterpret_cast<uintptr_t>(r.out)) & 15) == 0;
  return r;
}

// Elements k0 .. of the chunk, CL_VECTORS vectors (or values) per thread; zeros behind the end.
__device__ __forceinline__ void load_vectors(float4 (&x)[CL_VECTORS], const Chunk& c, long long k0) {
#pragma unroll
  for (int e = 0; e < CL_VECTORS; ++e) {
    const long long k = k0 + 4 * (e * CL_THREADS + threadIdx.x);
    x[e] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (k + 4 <= c.n) {
      x[e] = *reinterpret_cast<const float4*>(c.in + k);
    } else {
      if (k < c.n) x[e].x = c.in[k];
      if (k + 1 < c.n) x[e].y = c.in[k + 1];
      if (k + 2 < c.n) x[e].z = c.in[k + 2];
    }
  }
}
__device__ __forceinline__ void load_values(float (&x)[CL_VECTORS], const Chunk& c, long long k0) {
#pragma unroll
  for (int e = 0; e < CL_VECTORS; ++e) {
    const long long k = k0 + e * CL_THREADS + threadIdx.x;
    x[e] = k < c.n ? c.in[k] : 0.0f;
  }
}

// Every thread gets the sum; one call per kernel.
__device__ __forceinline__ double block_sum_f64(double v) {
  __shared__ double sm[CL_THREADS / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0.0;
#pragma unroll
  for (int w = 0; w < CL_THREADS / 32; ++w) t += sm[w];
  return t;
}

__device__ __forceinline__ double square(float x) { return (double)x * (double)x; }

// part[blockIdx.x] = the squares of this block's chunks.  Full occupancy, few loads
// per thread: 0.20 ms for 1.34 GB, against 0.29 ms with CL_VECTORS in flight per
// thread on half the threads.
__global__ void __launch_bounds__(CL_THREADS, 8) norm_partial_kernel(const __grid_constant__ ClipTable t,
                                                                    double* __restrict__ part) {
  double acc = 0.0;
  for (long long i = blockIdx.x; i < t.first[t.count]; i += gridDim.x) {
    const Chunk c = chunk_of(t, i);
    const int n = (int)c.n, n4 = c.vec ? n / 4 : 0;
#pragma unroll 2
    for (int k = threadIdx.x; k < n4; k += CL_THREADS) {
      const float4 x = reinterpret_cast<const float4*>(c.in)[k];
      acc += square(x.x);
      acc += square(x.y);
      acc += square(x.z);
      acc += square(x.w);
    }
#pragma unroll 4
    for (int k = 4 * n4 + threadIdx.x; k < n; k += CL_THREADS) acc += square(c.in[k]);
  }
  const double s = block_sum_f64(acc);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// The norm from all blocks' parts: in every block of a launch the same operations
// in the same order.
__device__ __forceinline__ double norm_of(const double* part, int parts) {
  double acc = 0.0;
#pragma unroll 4
  for (int k = threadIdx.x; k < parts; k += CL_THREADS) acc += part[k];
  return sqrt(block_sum_f64(acc));
}

__global__ void __launch_bounds__(CL_THREADS) norm_final_kernel(const double* part, int parts,
                                                               float* __restrict__ norm_out) {
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the parts are complete behind it
  const double s = norm_of(part, parts);
  if (threadIdx.x == 0) norm_out[0] = (float)s;
}

// The chunks from the last to the first: the norm's pass read those last, and L2 still holds them.
__global__ void __launch_bounds__(CL_THREADS) clip_scale_kernel(const __grid_constant__ ClipTable t, const double* part,
                                                               int parts, float max_norm, float* norm_out) {
  const long long all = t.first[t.count];
  Chunk c = {};
  if (blockIdx.x < all) c = chunk_of(t, all - 1 - blockIdx.x);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const double norm = norm_of(part, parts);
  if (blockIdx.x == 0 && threadIdx.x == 0 && norm_out) norm_out[0] = (float)norm;
  const double f = (double)max_norm / (norm + 1e-6);
  const bool keep = f >= 1.0;  // false for a NaN norm: its NaN goes into the outputs
  const float factor = keep ? 1.0f : (float)f;
  for (long long i = blockIdx.x; i < all; i += gridDim.x) {
    if (i != blockIdx.x) c = chunk_of(t, all - 1 - i);
    if (keep && c.out == c.in) continue;
    if (c.vec) {
      for (long long k0 = 0; k0 < c.n; k0 += CL_LONG) {
        float4 x[CL_VECTORS];
        load_vectors(x, c, k0);
#pragma unroll
        for (int e = 0; e < CL_VECTORS; ++e) {
          const long long k = k0 + 4 * (e * CL_THREADS + threadIdx.x);
          const float4 y = make_float4(x[e].x * factor, x[e].y * factor, x[e].z * factor, x[e].w * factor);
          if (k + 4 <= c.n) {
            *reinterpret_cast<float4*>(c.out + k) = y;
          } else {
            if (k < c.n) c.out[k] = y.x;
            if (k + 1 < c.n) c.out[k + 1] = y.y;
            if (k + 2 < c.n) c.out[k + 2] = y.z;
          }
        }
      }
    } else {
      for (long long k0 = 0; k0 < c.n; k0 += CL_LONG / 4) {
        float x[CL_VECTORS];
        load_values(x, c, k0);
#pragma unroll
        for (int e = 0; e < CL_VECTORS; ++e) {
          const long long k = k0 + e * CL_THREADS + threadIdx.x;
          if (k < c.n) c.out[k] = x[e] * factor;
        }
      }
    }
  }
}

// The launch's table for tensors i0 .. min(i0 + CL_TENSORS, count) - 1.
void fill(ClipTable& t, const float* const* in, float* const* out, const int64_t* sizes, int i0, int count,
          long long chunk) {
  t.count = std::min(CL_TENSORS, count - i0);
  t.chunk = chunk;
  t.first[0] = 0;
  for (int k = 0; k < t.count; ++k) {
    t.in[k] = in[i0 + k];
    t.out[k] = out ? out[i0 + k] : nullptr;
    t.size[k] = sizes[i0 + k];
    t.first[k + 1] = t.first[k] + (sizes[i0 + k] + chunk - 1) / chunk;
  }
}

// Launch whose blocks may start while the launch before finishes (they wait for it before they read its results).
template <class... Params, class... Args>
cudaError_t launch_after(void (*kernel)(Params...), int grid, cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(CL_THREADS);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

int check_tensors(const char* what, const float* const* in, float* const* out, bool want_out, const int64_t* sizes,
                  int count) {
  JX_REQUIRE(count >= 0, "%s: negative tensor count", what);
  JX_REQUIRE(count <= CL_MAX_TENSORS, "%s: too many tensors", what);
  if (count == 0) return JX_OK;
  JX_REQUIRE(in && sizes && (!want_out || out), "%s: NULL array", what);
  for (int i = 0; i < count; ++i) {
    JX_REQUIRE(sizes[i] >= 0, "%s: tensor %d has negative size", what, i);
    JX_REQUIRE(sizes[i] == 0 || (in[i] && (!want_out || out[i])), "%s: tensor %d has a NULL pointer", what, i);
  }
  return JX_OK;
}

int grid_of(const ClipTable& t) { return (int)std::min<long long>(t.first[t.count], (long long)jx::num_sms() * 8); }

// The blocks' parts of the sum of squares, in scratch.
int norm_launches(const float* const* in, const int64_t* sizes, int count, long long chunk, double** part_out,
                  int* parts_out, cudaStream_t st) {
  const int launches = (count + CL_TENSORS - 1) / CL_TENSORS;
  void* p = nullptr;
  if (int rc = jx::scratch_get(sizeof(double) * ((size_t)launches * jx::num_sms() * 8 + 1), &p, st)) return rc;
  double* part = static_cast<double*>(p);
  int parts = 0;
  ClipTable t;
  for (int l = 0; l < launches; ++l) {
    fill(t, in, nullptr, sizes, l * CL_TENSORS, count, chunk);
    const int grid = grid_of(t);
    if (grid == 0) continue;
    norm_partial_kernel<<<grid, CL_THREADS, 0, st>>>(t, part + parts);
    parts += grid;
  }
  *part_out = part;
  *parts_out = parts;
  return JX_OK;
}

long long chunk_for(const int64_t* sizes, int count) {
  long long all = 0;
  for (int i = 0; i < count; ++i) all += sizes[i];
  return all <= CL_SHORT * jx::num_sms() * 8 ? CL_SHORT : CL_LONG;
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
  if (int rc = norm_launches(grads, sizes, count, chunk_for(sizes, count), &part, &parts, st)) return rc;
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) e = launch_after(norm_final_kernel, 1, st, static_cast<const double*>(part), parts, norm_out);
  jx::scratch_release(part, st);
  return e == cudaSuccess ? JX_OK : jx::check_cuda(e, "grad_norm kernels");
}

int jx_clip_grads_f32(const float* const* grads, float* const* outs, const int64_t* sizes, int count, float max_norm,
                      float* norm_out, jx_stream_t stream) {
  JX_TRACE("jx_clip_grads_f32");
  if (int rc = check_tensors("clip_grads", grads, outs, true, sizes, count)) return rc;
  JX_REQUIRE(max_norm >= 0.0f, "clip_grads: max_norm must not be negative");
  cudaStream_t st = jx::as_stream(stream);
  const long long chunk = chunk_for(sizes, count);
  double* part = nullptr;
  int parts = 0;
  if (int rc = norm_launches(grads, sizes, count, chunk, &part, &parts, st)) return rc;
  cudaError_t e = cudaGetLastError();
  // the tensors that the norm's pass read last come first
  ClipTable t;
  const int last = count > 0 ? (count - 1) / CL_TENSORS * CL_TENSORS : 0;
  for (int i0 = last; i0 >= 0 && e == cudaSuccess; i0 -= CL_TENSORS) {
    fill(t, grads, outs, sizes, i0, count, chunk);
    const int grid = grid_of(t);
    // a launch without chunks is left out, but the first one writes norm_out
    if (grid || i0 == last)
      e = launch_after(clip_scale_kernel, std::max(grid, 1), st, t, static_cast<const double*>(part), parts, max_norm,
                       i0 == last ? norm_out : nullptr);
  }
  jx::scratch_release(part, st);
  return e == cudaSuccess ? JX_OK : jx::check_cuda(e, "clip_grads kernels");
}

}  // extern "C"
