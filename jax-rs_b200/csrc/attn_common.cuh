// attn_common.cuh -- what the attention kernels share: the call's shape, the
// packed sequences' bounds, and the row-at-a-time forms of the forward pass and
// of both gradients.
#pragma once

#include <math.h>

#include "jx_common.cuh"

namespace jxa {

constexpr int MAX_DIM = 128;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

struct Shape {
  const int32_t* cu_q;
  const int32_t* cu_k;
  int batch, heads, kv_heads, group, dim;
  long long total_q, total_k;
  long long ldq, ldk, ldv, ldo;
  float scale;
  int causal;
  unsigned int* err;
};

struct Seq {
  long long q0, k0;
  int lq, lk;
  // Keys that query row i sees: the first visible(i) ones.
  __device__ __forceinline__ int visible(int i, int causal) const {
    return causal ? max(0, min(lk, i + lk - lq + 1)) : lk;
  }
  // First query row that sees key j.
  __device__ __forceinline__ int first_row(int j, int causal) const { return causal ? max(0, j - (lk - lq)) : 0; }
};

// An offset outside its tensor is taken as the nearest one inside and reported.
__device__ __forceinline__ long long offset_in(const int32_t* cu, int i, long long lo, long long hi,
                                               unsigned int* err) {
  const long long v = cu[i];
  const long long c = v < lo ? lo : v > hi ? hi : v;
  if (c != v) atomicOr(err, JX_DEVERR_RANGE);
  return c;
}
__device__ __forceinline__ Seq seq_bounds(const Shape& s, int b) {
  Seq r;
  r.q0 = offset_in(s.cu_q, b, 0, s.total_q, s.err);
  r.lq = (int)(offset_in(s.cu_q, b + 1, r.q0, s.total_q, s.err) - r.q0);
  r.k0 = offset_in(s.cu_k, b, 0, s.total_k, s.err);
  r.lk = (int)(offset_in(s.cu_k, b + 1, r.k0, s.total_k, s.err) - r.k0);
  return r;
}

// The last b in [0, batch) with at(b) <= x for a function that does not decrease
// (0 if there is none), found by a whole warp: 32 places are tried at a time, so
// that up to 32 sequences cost one load's latency.
template <class At>
__device__ __forceinline__ int last_at_most(int batch, long long x, At at) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = batch;
  while (hi - lo > 1) {
    const int step = (hi - lo + 32) / 33;
    const long long mid = lo + (long long)(lane + 1) * step;
    const bool in = mid < hi && at((int)mid) <= x;
    const int c = __popc(__ballot_sync(0xffffffffu, in));
    lo += c * step;
    hi = min(hi, lo + step);
  }
  return lo;
}
// The sequence that row t belongs to, if t lies within its bounds.  Warp-uniform t.
__device__ __forceinline__ int seq_of_row(const int32_t* cu, int batch, long long t) {
  return last_at_most(batch, t, [&](int b) { return (long long)cu[b]; });
}

// ---- one row by one warp, in plain f32 ------------------------------------------
// The warp's four groups of eight lanes take every fourth key (or query) each;
// lane l of a group holds the elements l, l + 8, l + 16, ... of a row.
constexpr int ROW_E = MAX_DIM / 8;

__device__ __forceinline__ void row_load(float (&r)[ROW_E], const float* p, int dim, int l, bool on) {
#pragma unroll
  for (int e = 0; e < ROW_E; ++e) r[e] = on && l + 8 * e < dim ? p[l + 8 * e] : 0.0f;
}
__device__ __forceinline__ float row_dot(const float (&a)[ROW_E], const float (&b)[ROW_E]) {
  float s = 0.0f;
#pragma unroll
  for (int e = 0; e < ROW_E; ++e) s = fmaf(a[e], b[e], s);
  s += __shfl_xor_sync(0xffffffffu, s, 1);
  s += __shfl_xor_sync(0xffffffffu, s, 2);
  s += __shfl_xor_sync(0xffffffffu, s, 4);
  return s;
}
// Sum over the four groups, stored by the first.
__device__ __forceinline__ void row_store(float* p, const float (&r)[ROW_E], float factor, int dim, int lane) {
#pragma unroll
  for (int e = 0; e < ROW_E; ++e) {
    float v = r[e];
    v += __shfl_xor_sync(0xffffffffu, v, 8);
    v += __shfl_xor_sync(0xffffffffu, v, 16);
    const int c = (lane & 7) + 8 * e;
    if (lane < 8 && c < dim) p[c] = v * factor;
  }
}

// o[0 .. dim) and the log-sum-exp of one query row over nk keys.
static __device__ __noinline__ void row_fwd(const float* q, const float* k, const float* v, float* o, float* lse, int nk,
                                     int dim, long long ldk, long long ldv, float scale) {
  const int lane = threadIdx.x & 31, g = lane >> 3, l = lane & 7;
  float qr[ROW_E], acc[ROW_E];
  row_load(qr, q, dim, l, true);
#pragma unroll
  for (int e = 0; e < ROW_E; ++e) acc[e] = 0.0f;
  float m = -INFINITY, sum = 0.0f;
  for (int j0 = 0; j0 < nk; j0 += 4) {
    const int j = j0 + g;
    const bool on = j < nk;
    float kr[ROW_E];
    row_load(kr, k + (long long)j * ldk, dim, l, on);
    const float x = row_dot(qr, kr) * (scale * LOG2E);
    if (on) {
      const float top = fmaxf(m, x);  // a NaN score leaves the maximum as it is and makes p NaN
      const float safe = top == -INFINITY ? 0.0f : top;
      const float alpha = exp2f(m - safe), p = exp2f(x - safe);
      m = top;
      sum = sum * alpha + p;
      row_load(kr, v + (long long)j * ldv, dim, l, true);
#pragma unroll
      for (int e = 0; e < ROW_E; ++e) acc[e] = acc[e] * alpha + p * kr[e];
    }
  }
  float top = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
  const float f = exp2f(m - (top == -INFINITY ? 0.0f : top));
  sum *= f;
  sum += __shfl_xor_sync(0xffffffffu, sum, 8);
  sum += __shfl_xor_sync(0xffffffffu, sum, 16);
#pragma unroll
  for (int e = 0; e < ROW_E; ++e) acc[e] *= f;
  row_store(o, acc, sum == 0.0f ? 0.0f : 1.0f / sum, dim, lane);
  if (lane == 0 && lse) *lse = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * LN2;
}

// dq of one query row over nk keys.
static __device__ __noinline__ void row_dq(const float* q, const float* k, const float* v, const float* o, const float* dout,
                                    float lse, float* dq, int nk, int dim, long long ldk, long long ldv,
                                    float scale) {
  const int lane = threadIdx.x & 31, g = lane >> 3, l = lane & 7;
  float qr[ROW_E], dor[ROW_E], acc[ROW_E], kr[ROW_E];
  row_load(qr, q, dim, l, true);
  row_load(dor, dout, dim, l, true);
  row_load(kr, o, dim, l, true);
  const float delta = row_dot(dor, kr);
#pragma unroll
  for (int e = 0; e < ROW_E; ++e) acc[e] = 0.0f;
  for (int j0 = 0; j0 < nk; j0 += 4) {
    const int j = j0 + g;
    const bool on = j < nk;
    row_load(kr, v + (long long)j * ldv, dim, l, on);
    const float dp = row_dot(dor, kr);
    row_load(kr, k + (long long)j * ldk, dim, l, on);
    const float x = row_dot(qr, kr) * scale;
    if (on) {
      const float ds = lse == -INFINITY ? 0.0f : expf(x - lse) * (dp - delta);
#pragma unroll
      for (int e = 0; e < ROW_E; ++e) acc[e] = fmaf(ds, kr[e], acc[e]);
    }
  }
  row_store(dq, acc, scale, dim, lane);
}

// dk and dv of one key row: query rows i0 .. lq-1 of the `group` heads that
// share it.  q, o and dout point at the sequence's first row of the group's
// first head, lse at that head's entry of the same row.
static __device__ __noinline__ void row_dkv(const float* q, const float* o, const float* dout, const float* lse,
                                     const float* k, const float* v, float* dk, float* dv, int i0, int lq, int group,
                                     int dim, long long ldq, long long ldo, long long total_q, float scale) {
  const int lane = threadIdx.x & 31, g = lane >> 3, l = lane & 7;
  float kr[ROW_E], vr[ROW_E], ak[ROW_E], av[ROW_E], a[ROW_E], b[ROW_E];
  row_load(kr, k, dim, l, true);
  row_load(vr, v, dim, l, true);
#pragma unroll
  for (int e = 0; e < ROW_E; ++e) ak[e] = av[e] = 0.0f;
  for (int h = 0; h < group; ++h) {
    for (int r = i0; r < lq; r += 4) {
      const int i = r + g;
      const bool on = i < lq;
      row_load(a, o + (long long)i * ldo + h * dim, dim, l, on);
      row_load(b, dout + (long long)i * ldo + h * dim, dim, l, on);
      const float delta = row_dot(a, b), dp = row_dot(b, vr);
      row_load(a, q + (long long)i * ldq + h * dim, dim, l, on);
      const float x = row_dot(a, kr) * scale;
      if (on) {
        const float z = lse[(long long)h * total_q + i];
        const float p = z == -INFINITY ? 0.0f : expf(x - z);
        const float ds = p * (dp - delta);
#pragma unroll
        for (int e = 0; e < ROW_E; ++e) {
          av[e] = fmaf(p, b[e], av[e]);
          ak[e] = fmaf(ds, a[e], ak[e]);
        }
      }
    }
  }
  row_store(dk, ak, scale, dim, lane);
  row_store(dv, av, 1.0f, dim, lane);
}

}  // namespace jxa
