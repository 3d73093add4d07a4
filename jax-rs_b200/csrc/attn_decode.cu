// attn_decode.cu -- attention's forward pass for few query rows per key head (a
// decoding step), in plain f32.
//
// Bound by reading K and V once from HBM.  A warp's lanes form groups, LPK lanes
// to a key, each lane with DP / LPK of its columns, so that a load instruction
// reads whole rows; a group keeps a running maximum, sum and output of its own
// for the R query rows that the CTA serves (query rows times heads of the
// group, so that K and V are read once for all of them), and nothing is
// exchanged before the end but the LPK-lane sums of the scores.  The keys are
// cut in chunks over CTAs; attn_join_kernel joins the chunks' results.
#include <algorithm>

#include "attn_common.cuh"

namespace {

using namespace jxa;

constexpr int DC_WARPS = 4;
constexpr int DC_U = 2;  // keys that a group loads at a time

// Rows of a sequence are numbered i * group + head: chunk id of R rows, as seq_of_tile numbers tiles.
__device__ __forceinline__ int seq_of_chunk(const int32_t* cu, int batch, int group, int R, long long id,
                                            long long* j) {
  int lo = 0, hi = batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if ((long long)cu[mid] * group / R + mid <= id) lo = mid;
    else hi = mid;
  }
  *j = id - ((long long)cu[lo] * group / R + lo);
  return lo;
}

__device__ __forceinline__ float exp2_of(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Lane l's columns of a row: vectors of four, LPK vectors apart.
template <int E, int LPK, bool VEC>
__device__ __forceinline__ void load_cols(float (&x)[E], const float* p, int l, int dim) {
#pragma unroll
  for (int c = 0; c < E / 4; ++c) {
    const int col = (c * LPK + l) * 4;
    float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
    if (VEC) {
      if (col < dim) f = *reinterpret_cast<const float4*>(p + col);
    } else {
      if (col < dim) f.x = p[col];
      if (col + 1 < dim) f.y = p[col + 1];
      if (col + 2 < dim) f.z = p[col + 2];
      if (col + 3 < dim) f.w = p[col + 3];
    }
    x[4 * c] = f.x;
    x[4 * c + 1] = f.y;
    x[4 * c + 2] = f.z;
    x[4 * c + 3] = f.w;
  }
}

// grid: (row chunks, key heads, splits).  Split z takes the key chunks z, z +
// gridDim.z, ...; with one split the results go straight to o and lse.
template <int R, int LPK, int DP, bool VEC>
__global__ void __launch_bounds__(32 * DC_WARPS)
    attn_decode_kernel(const __grid_constant__ Shape s, const float* __restrict__ q, const float* __restrict__ k,
                       const float* __restrict__ v, float* o, float* lse, float* __restrict__ part, int chunk) {
  constexpr int E = DP / LPK, G = 32 / LPK;  // columns per lane, groups per warp
  __shared__ float sm_acc[DC_WARPS][R][DP];
  __shared__ float sm_m[DC_WARPS][R], sm_sum[DC_WARPS][R];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane / LPK, l = lane % LPK;
  long long jc;
  const int b = seq_of_chunk(s.cu_q, s.batch, s.group, R, blockIdx.x, &jc);
  const Seq sq = seq_bounds(s, b);
  const long long all_rows = (long long)sq.lq * s.group, row0 = jc * R;
  if (jc < 0 || row0 >= all_rows) return;
  const int rows = (int)min((long long)R, all_rows - row0), hk = blockIdx.y;
  if (blockIdx.z > 0 && (long long)blockIdx.z * chunk >= sq.lk) return;

  float qr[R][E], acc[R][E], m[R], sum[R];
  int vis[R];
  int vis_least = sq.lk;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int i = (int)((row0 + r) / s.group), h = hk * s.group + (int)((row0 + r) % s.group);
    const bool on = r < rows;
    if (on) {
      load_cols<E, LPK, VEC>(qr[r], q + (sq.q0 + i) * s.ldq + (long long)h * s.dim, l, s.dim);
    }
    vis[r] = on ? sq.visible(i, s.causal) : 0;
    if (on) vis_least = min(vis_least, vis[r]);
    m[r] = -INFINITY;
    sum[r] = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      qr[r][e] = on ? qr[r][e] * (s.scale * LOG2E) : 0.0f;
      acc[r][e] = 0.0f;
    }
  }
  const float* kb = k + sq.k0 * s.ldk + (long long)hk * s.dim;
  const float* vb = v + sq.k0 * s.ldv + (long long)hk * s.dim;
  const int vis_most = sq.visible((int)((row0 + rows - 1) / s.group), s.causal);
  for (long long c0 = (long long)blockIdx.z * chunk; c0 < vis_most; c0 += (long long)gridDim.z * chunk) {
    const int end = (int)min(c0 + chunk, (long long)vis_most);
    for (int j0 = (int)c0 + warp * G * DC_U; j0 < end; j0 += DC_WARPS * G * DC_U) {
      // the warp's G * DC_U consecutive keys: u-th load takes keys j0 + u * G + g
      float kr[DC_U][E], vr[DC_U][E];
#pragma unroll
      for (int u = 0; u < DC_U; ++u) {
        const int j = min(j0 + u * G + g, end - 1);
        load_cols<E, LPK, VEC>(kr[u], kb + (long long)j * s.ldk, l, s.dim);
      }
#pragma unroll
      for (int u = 0; u < DC_U; ++u) {
        const int j = min(j0 + u * G + g, end - 1);
        load_cols<E, LPK, VEC>(vr[u], vb + (long long)j * s.ldv, l, s.dim);
      }
      const bool whole = j0 + DC_U * G <= min(end, vis_least);  // every row sees all of these keys
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float x[DC_U];
#pragma unroll
        for (int u = 0; u < DC_U; ++u) {
          float d = 0.0f;
#pragma unroll
          for (int e = 0; e < E; ++e) d = fmaf(qr[r][e], kr[u][e], d);
#pragma unroll
          for (int w = LPK / 2; w > 0; w >>= 1) d += __shfl_xor_sync(0xffffffffu, d, w);
          x[u] = d;
        }
        bool on[DC_U];
#pragma unroll
        for (int u = 0; u < DC_U; ++u) {
          const int j = j0 + u * G + g;
          on[u] = whole || (j < end && j < vis[r]);
          if (!on[u]) x[u] = -INFINITY;
        }
        float top = m[r];
#pragma unroll
        for (int u = 0; u < DC_U; ++u) top = fmaxf(top, x[u]);
        if (__any_sync(0xffffffffu, top > m[r])) {
          const float f = exp2_of(m[r] - (top == -INFINITY ? 0.0f : top));
          sum[r] *= f;
#pragma unroll
          for (int e = 0; e < E; ++e) acc[r][e] *= f;
          m[r] = top;
        }
        const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (int u = 0; u < DC_U; ++u) {
          const float p = exp2_of(x[u] - base);
          sum[r] += p;
          if (whole) {
#pragma unroll
            for (int e = 0; e < E; ++e) acc[r][e] = fmaf(p, vr[u][e], acc[r][e]);
          } else if (on[u]) {  // an unseen key's value may be anything
#pragma unroll
            for (int e = 0; e < E; ++e) acc[r][e] = fmaf(p, vr[u][e], acc[r][e]);
          }
        }
      }
    }
  }
  // the warp's groups, then the warps
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float top = m[r];
#pragma unroll
    for (int w = LPK; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
    const float f = exp2_of(m[r] - (top == -INFINITY ? 0.0f : top));
    float t = sum[r] * f;
#pragma unroll
    for (int w = LPK; w < 32; w <<= 1) t += __shfl_xor_sync(0xffffffffu, t, w);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float a = acc[r][e] * f;
#pragma unroll
      for (int w = LPK; w < 32; w <<= 1) a += __shfl_xor_sync(0xffffffffu, a, w);
      if (g == 0) sm_acc[warp][r][((e / 4) * LPK + l) * 4 + (e & 3)] = a;
    }
    if (lane == 0) {
      sm_m[warp][r] = top;
      sm_sum[warp][r] = t;
    }
  }
  __syncthreads();
  const bool last = gridDim.z == 1;
  for (int r = warp; r < rows; r += DC_WARPS) {
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < DC_WARPS; ++w) top = fmaxf(top, sm_m[w][r]);
    const float base = top == -INFINITY ? 0.0f : top;
    float t = 0.0f, f[DC_WARPS];
#pragma unroll
    for (int w = 0; w < DC_WARPS; ++w) {
      f[w] = exp2_of(sm_m[w][r] - base);
      t += sm_sum[w][r] * f[w];
    }
    const int i = (int)((row0 + r) / s.group), h = hk * s.group + (int)((row0 + r) % s.group);
    const long long tok = sq.q0 + i;
    float* out = last ? o + tok * s.ldo + (long long)h * s.dim
                      : part + ((tok * s.heads + h) * gridDim.z + blockIdx.z) * (MAX_DIM + 2);
    const float inv = !last ? 1.0f : t == 0.0f ? 0.0f : 1.0f / t;
    for (int c = lane; c < s.dim; c += 32) {
      float a = 0.0f;
#pragma unroll
      for (int w = 0; w < DC_WARPS; ++w) a += sm_acc[w][r][c] * f[w];
      out[c] = a * inv;
    }
    if (lane == 0) {
      if (!last) {
        out[MAX_DIM] = top;
        out[MAX_DIM + 1] = t;
      } else if (lse) {
        lse[(long long)h * s.total_q + tok] = t == 0.0f ? -INFINITY : (top + log2f(t)) * LN2;
      }
    }
  }
}

// One warp per (query row, head): the splits' results in order.
__global__ void __launch_bounds__(128) attn_join_kernel(const __grid_constant__ Shape s, const float* __restrict__ part,
                                                       float* o, float* lse, int splits, int chunk) {
  const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const long long tok = w / s.heads;
  const int h = (int)(w - tok * s.heads);
  if (tok >= s.total_q) return;
  const int b = seq_of_row(s.cu_q, s.batch, tok);
  if (b < 0) return;
  const Seq sq = seq_bounds(s, b);
  if (tok < sq.q0 || tok >= sq.q0 + sq.lq) return;
  const int n = max(1, (int)min((long long)splits, ((long long)sq.lk + chunk - 1) / chunk));
  const float* p = part + (tok * s.heads + h) * splits * (MAX_DIM + 2);
  float top = -INFINITY;
  for (int z = lane; z < n; z += 32) top = fmaxf(top, p[(long long)z * (MAX_DIM + 2) + MAX_DIM]);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
  const float base = top == -INFINITY ? 0.0f : top;
  float a[4] = {0.f, 0.f, 0.f, 0.f}, t = 0.0f;
#pragma unroll 4
  for (int z = 0; z < n; ++z) {
    const float* e = p + (long long)z * (MAX_DIM + 2);
    const float f = exp2_of(e[MAX_DIM] - base);
    t += e[MAX_DIM + 1] * f;
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (lane + 32 * c < s.dim) a[c] += e[lane + 32 * c] * f;
  }
  const float inv = t == 0.0f ? 0.0f : 1.0f / t;
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (lane + 32 * c < s.dim) o[tok * s.ldo + (long long)h * s.dim + lane + 32 * c] = a[c] * inv;
  if (lane == 0 && lse) lse[(long long)h * s.total_q + tok] = t == 0.0f ? -INFINITY : (top + log2f(t)) * LN2;
}

using DecodeKernel = void (*)(Shape, const float*, const float*, const float*, float*, float*, float*, int);

template <int R, int L128, int L64>
DecodeKernel kernel_of(int DP, bool vec) {
  if (DP == 128) return vec ? attn_decode_kernel<R, L128, 128, true> : attn_decode_kernel<R, L128, 128, false>;
  return vec ? attn_decode_kernel<R, L64, 64, true> : attn_decode_kernel<R, L64, 64, false>;
}

}  // namespace

namespace jxa {

// rows: query rows per key head of the longest sequence, a hint.
int attention_decode(const Shape& s, const float* q, const float* k, const float* v, float* o, float* lse,
                     long long rows, long long max_k, cudaStream_t st) {
  const int DP = s.dim <= 64 ? 64 : 128;
  auto a16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  const bool vec = !(s.dim & 3) && !(s.ldq & 3) && !(s.ldk & 3) && !(s.ldv & 3) && a16(q) && a16(k) && a16(v);
  const int R = rows <= 1 ? 1 : rows <= 2 ? 2 : rows <= 4 ? 4 : rows <= 8 ? 8 : 16;
  const DecodeKernel kernel = R == 1   ? kernel_of<1, 8, 8>(DP, vec)
                              : R == 2 ? kernel_of<2, 8, 8>(DP, vec)
                              : R == 4 ? kernel_of<4, 8, 8>(DP, vec)
                              : R == 8 ? kernel_of<8, 16, 16>(DP, vec)
                                       : kernel_of<16, 32, 16>(DP, vec);
  const long long chunks = s.total_q * s.group / R + s.batch;
  JX_REQUIRE(chunks < (1LL << 31), "attention: too many rows");
  // keys per CTA: four CTAs per SM over all sequences, 64 keys at least
  const long long even = s.total_k * s.kv_heads / (4LL * jx::num_sms());
  const int chunk = (int)std::min<long long>(1 << 20, std::max<long long>(64, (even + 63) / 64 * 64));
  const int splits = (int)std::max<long long>(1, std::min<long long>(128, (max_k + chunk - 1) / chunk));
  void* part = nullptr;
  if (splits > 1)
    if (int rc = jx::scratch_get(sizeof(float) * (size_t)s.total_q * s.heads * splits * (MAX_DIM + 2), &part, st))
      return rc;
  kernel<<<dim3((unsigned)chunks, (unsigned)s.kv_heads, (unsigned)splits), 32 * DC_WARPS, 0, st>>>(
      s, q, k, v, o, lse, static_cast<float*>(part), chunk);
  if (splits > 1)
    attn_join_kernel<<<(unsigned)((s.total_q * s.heads + 3) / 4), 128, 0, st>>>(s, static_cast<float*>(part), o, lse,
                                                                              splits, chunk);
  const cudaError_t e = cudaGetLastError();
  jx::scratch_release(part, st);
  return e == cudaSuccess ? JX_OK : jx::check_cuda(e, "attn_decode_kernel");
}

}  // namespace jxa
