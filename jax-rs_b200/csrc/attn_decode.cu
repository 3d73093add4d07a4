// attn_decode.cu -- attention's forward pass for few query rows per key head (a
// decoding step), in plain f32.
//
// Bound by reading K and V once from HBM.  The keys of all sequences and key heads
// are one line of positions, (sequence, key head, key) in order, cut in equal
// ranges; a ring of shared-memory stages, eight keys each, streams a range with
// TMA, and one to eight warps read it, four query rows each (rows of
// the sequence times heads of the group), so that K and V are read once for all
// rows.  In a warp eight lanes share a key, 16 columns each for dim 128, and the
// four groups of lanes keep a running maximum, sum and output of their own:
// nothing is exchanged per key but the eight-lane sums of the scores.  A range's
// piece of a head goes to scratch unless it is the whole head, and
// attn_join_kernel joins the pieces.
//
// One token behind eight histories, 14.7k keys of 8 heads of 128 (118 MB): 33 us for
// both kernels (30 in a captured graph), 3.6 TB/s, against 18 us of reading at the copy rate.  The
// kernel itself takes 25 us; the rest is the join, which waits for the slowest
// ring.  Copying row by row (one bulk copy of 512 B each) took 37 us, the rate of
// copy instructions being the bound.
//
// 192 KB of stages per SM keep about 128 KB of loads in flight, three times what
// HBM's latency needs at full rate.
#include <algorithm>
#include <atomic>

#include "attn_tc.cuh"

namespace {

using namespace jxa;

constexpr int DC_WARPS = 8;
constexpr int DC_KEYS = 8;  // keys per stage
constexpr int DC_LPK = 8;   // lanes per key
constexpr int DC_GROUPS = 32 / DC_LPK;
constexpr int DC_RING = 192 * 1024;

__host__ __device__ constexpr int dc_stage(int DP) { return DC_KEYS * 2 * DP * 4; }
__host__ __device__ constexpr int dc_stages(int DP) { return DC_RING / dc_stage(DP); }  // of all rings
__host__ __device__ constexpr size_t dc_smem(int DP) { return DC_RING + 2 * 8 * dc_stages(DP) + 128; }

// Every lane for itself: one lane that asks and tells the others takes 150 cycles more.
__device__ __forceinline__ bool ring_wait(uint64_t* bar, uint32_t parity, unsigned int* err) {
  const bool ok = wait_suspended(bar, parity, err);
  return __all_sync(0xffffffffu, ok);
}

// A place in the line of positions.  A head takes lk + VOID of them: starting and
// storing a head costs a ring about as much as VOID keys, so that short heads
// weigh what they cost (8 histories, 3 of them short: 16, 24, 32, 40 and 72 take 40.3, 36.8, 30.2, 30.1 and 30.4 us).
constexpr int VOID = 40;
struct Cursor {
  long long pos;  // line_start(k0, b) + hk * (lk + VOID) + key, as this head was entered
  int b, hk, key, left, entered;  // keys of the head that are left in the range; the key that it was entered at
  Seq sq;
  bool on;

  __device__ __forceinline__ void enter(long long end) {
    on = pos < end;
    entered = key;
    left = on ? (int)min((long long)(sq.lk - key), end - pos) : 0;
  }
  // To the first key at or behind `pos`, in a sequence from b on.
  __device__ __forceinline__ void settle(const Shape& s, long long end, int row_base) {
    on = false;
    left = 0;
    for (; b < s.batch; ++b) {
      sq = seq_bounds(s, b);
      const long long base = (sq.k0 + (long long)b * VOID) * s.kv_heads, in = max(0LL, pos - base);
      if (base >= end) return;  // this sequence and all behind it are other rings'
      if ((long long)sq.lq * s.group <= row_base || sq.lk == 0) continue;
      const int len = sq.lk + VOID;
      if (in >= (long long)s.kv_heads * len) continue;
      hk = (int)(in / len);
      key = (int)(in - (long long)hk * len);
      if (key >= sq.lk) {
        key = 0;
        if (++hk == s.kv_heads) continue;
      }
      pos = base + (long long)hk * len + key;
      enter(end);
      return;
    }
  }
  // Behind the last of the head's keys in the range.
  __device__ __forceinline__ void advance(const Shape& s, long long end, int row_base) {
    pos += key - entered;
    on = false;
    if (key < sq.lk) return;  // the range ends here
    key = 0;
    pos += VOID;
    if (pos >= end) return;
    if (++hk < s.kv_heads) {
      enter(end);
    } else {
      ++b;
      settle(s, end, row_base);
    }
  }
};
__device__ __forceinline__ int seq_of_position(const Shape& s, long long pos) {
  return last_at_most(s.batch, pos, [&](int i) { return (s.cu_k[i] + (long long)i * VOID) * s.kv_heads; });
}

// Lane l's columns of a row of shared memory: vectors of four, DC_LPK vectors apart.
template <int E>
__device__ __forceinline__ void load_cols(float (&x)[E], const float* p, int l) {
#pragma unroll
  for (int c = 0; c < E / 4; ++c) {
    const float4 f = *reinterpret_cast<const float4*>(p + (c * DC_LPK + l) * 4);
    x[4 * c] = f.x;
    x[4 * c + 1] = f.y;
    x[4 * c + 2] = f.z;
    x[4 * c + 3] = f.w;
  }
}

// The same columns of a row of `dim` values in global memory, zeros behind them.
template <int E>
__device__ __forceinline__ void load_row(float (&x)[E], const float* p, int l, int dim, bool vec) {
#pragma unroll
  for (int c = 0; c < E / 4; ++c) {
    const int col = (c * DC_LPK + l) * 4;
    float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
    if (vec) {
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

// Sums of x over the warp's four groups; lane (g, l) is left with four columns
// of it: those of vector g (DP = 128), or of vector g / 2 (DP = 64, held twice).
template <int E>
__device__ __forceinline__ float4 sum_groups(const float (&x)[E], int g) {
  const bool up = g & 2, odd = g & 1;
  float y[E / 2];
#pragma unroll
  for (int e = 0; e < E / 2; ++e) {
    const float mine = up ? x[E / 2 + e] : x[e], other = up ? x[e] : x[E / 2 + e];
    y[e] = mine + __shfl_xor_sync(0xffffffffu, other, 16);
  }
  float z[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (E == 16) {
      const float mine = odd ? y[4 + e] : y[e], other = odd ? y[e] : y[4 + e];
      z[e] = mine + __shfl_xor_sync(0xffffffffu, other, 8);
    } else {
      z[e] = y[e] + __shfl_xor_sync(0xffffffffu, y[e], 8);
    }
  }
  return make_float4(z[0], z[1], z[2], z[3]);
}

// Ring w of `rings` takes the positions w * per .. +per.  warps_per_ring = WR in
// {1, 2, 4, 8}; warp i of a ring has the rows row_base + i * R .. +R of a sequence.
template <int R, int DP, bool VEC>
__global__ void __launch_bounds__(32 * DC_WARPS, 1)
    attn_decode_kernel(const __grid_constant__ Shape s, const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v, const float* __restrict__ q, const float* __restrict__ k,
                       const float* __restrict__ v, float* o, float* lse, float* __restrict__ part, long long per,
                       int WR, int row_base) {
  constexpr int E = DP / DC_LPK, STEPS = DC_KEYS / DC_GROUPS, STAGE = dc_stage(DP);
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane / DC_LPK, l = lane % DC_LPK;
  const int ring = warp / WR, wr = warp % WR, nst = dc_stages(DP) / DC_WARPS * WR;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + DC_RING) + ring * nst;
  uint64_t* empty = full + dc_stages(DP);
  float* stages = reinterpret_cast<float*>(smem + (size_t)ring * nst * STAGE);
  if (wr == 0 && lane == 0) {
    for (int i = 0; i < nst; ++i) {
      jxd::mbar_init(&full[i], VEC ? 1 : 32);
      jxd::mbar_init(&empty[i], WR);
    }
    jxd::fence_mbar_init();
  }
  if (VEC) {
    if (threadIdx.x == 0) {
      jxd::tma_prefetch_desc(&map_k);
      jxd::tma_prefetch_desc(&map_v);
    }
  } else {  // columns behind the head's dim stay zero
    for (int i = threadIdx.x; i < DC_RING / 16; i += 32 * DC_WARPS)
      reinterpret_cast<float4*>(smem)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  jxd::fence_proxy_async_smem();
  __syncthreads();

  const long long w = (long long)ring * gridDim.x + blockIdx.x;  // few rings' worth of work spreads over all SMs
  const long long begin = w * per, end = min(begin + per, (s.total_k + (long long)s.batch * VOID) * s.kv_heads);
  const bool vec_q = !(s.dim & 3) && !(s.ldq & 3) && !(reinterpret_cast<uintptr_t>(q) & 15);
  const bool vec_o = !(s.dim & 3) && !(s.ldo & 3) && !(reinterpret_cast<uintptr_t>(o) & 15);
  Cursor c;
  c.pos = begin;
  c.b = seq_of_position(s, begin);
  c.settle(s, end, row_base);
  Cursor pc = c;  // the copies' place, up to nst stages ahead
  int in_st = 0, out_st = 0, issued = 0;
  bool sends = true;  // lane 0's: if it gives up, the warp finds out when the stage does not come
  uint32_t in_ph = 0, out_ph = 0;
  bool ok = true;
  auto produce = [&]() {  // the ring's first warp: the next stage's rows
    if (!pc.on || !ok) return;
    const int st = in_st, n = min(DC_KEYS, pc.left);
    const long long t = pc.sq.k0 + pc.key;
    float* dst = stages + (size_t)st * (STAGE / 4);
    if constexpr (VEC) {
      // eight rows each, whatever n is: the rest is other sequences' or zeros, and masked
      if (lane == 0) {
        sends = sends && wait_suspended(&empty[st], in_ph ^ 1u, s.err);
        if (sends) {
          jxd::mbar_arrive_expect_tx(&full[st], (uint32_t)STAGE);
          jxd::tma_load_3d(dst, &map_k, &full[st], 0, (int)t, pc.hk);
          jxd::tma_load_3d(dst + DC_KEYS * DP, &map_v, &full[st], 0, (int)t, pc.hk);
          ++issued;
        }
      }
    } else {
      ok = ring_wait(&empty[st], in_ph ^ 1u, s.err);
      if (!ok) return;
      const long long hd = (long long)pc.hk * s.dim;
      for (int r = 0; r < n; ++r)
        for (int col = lane; col < s.dim; col += 32) {
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(jxd::smem_u32(dst + r * DP + col)),
                       "l"(k + (t + r) * s.ldk + hd + col)
                       : "memory");
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(jxd::smem_u32(dst + (8 + r) * DP + col)),
                       "l"(v + (t + r) * s.ldv + hd + col)
                       : "memory");
        }
      asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(jxd::smem_u32(&full[st])) : "memory");
      ++issued;
    }
    if (++in_st == nst) {
      in_st = 0;
      in_ph ^= 1u;
    }
    pc.key += n;
    if ((pc.left -= n) == 0) pc.advance(s, end, row_base);
  };
  if (wr == 0)
    for (int i = 0; i < nst; ++i) produce();

  while (c.on && ok) {
    // one piece of a (sequence, key head)
    const int b = c.b, hk = c.hk, first_key = c.key;
    const Seq sq = c.sq;
    // rows row_base + row0 .. of the sequence
    const int all_rows = (int)min((long long)sq.lq * s.group - row_base, (long long)R * WR), row0 = wr * R;
    float qr[R][E], acc[R][E], m[R], sum[R];
    int vis[R], vis_least = sq.lk;
    {
      int i = (row_base + row0) / s.group, hg = row_base + row0 - i * s.group;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const bool on = row0 + r < all_rows;
        load_row<E>(qr[r], q + (sq.q0 + i) * s.ldq + (long long)(hk * s.group + hg) * s.dim, l, on ? s.dim : 0, vec_q);
        vis[r] = on ? sq.visible(i, s.causal) : 0;
        if (on) vis_least = min(vis_least, vis[r]);
        if (++hg == s.group) {
          hg = 0;
          ++i;
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        m[r] = -INFINITY;
        sum[r] = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          qr[r][e] *= s.scale * LOG2E;
          acc[r][e] = 0.0f;
        }
      }
    }
    while (c.left > 0) {
      const int n = min(DC_KEYS, c.left), st = out_st, j0 = c.key;
      ok = ok && ring_wait(&full[st], out_ph, s.err);
      if (!ok) break;
      const float* base = stages + (size_t)st * (STAGE / 4);
      float x[R][STEPS];
#pragma unroll
      for (int u = 0; u < STEPS; ++u) {
        float kr[E];
        load_cols<E>(kr, base + (u * DC_GROUPS + g) * DP, l);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          float2 d = make_float2(0.0f, 0.0f);
#pragma unroll
          for (int e = 0; e < E; e += 2)
            d = fma2(make_float2(qr[r][e], qr[r][e + 1]), make_float2(kr[e], kr[e + 1]), d);
          x[r][u] = d.x + d.y;
        }
      }
#pragma unroll
      for (int t = DC_LPK / 2; t > 0; t >>= 1)
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int u = 0; u < STEPS; ++u) x[r][u] += __shfl_xor_sync(0xffffffffu, x[r][u], t);
      const bool whole = j0 + DC_KEYS <= vis_least && n == DC_KEYS;  // every row sees all of the stage's keys
      if (!whole) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int u = 0; u < STEPS; ++u)
            if (u * DC_GROUPS + g >= n || j0 + u * DC_GROUPS + g >= vis[r]) x[r][u] = -INFINITY;
      }
      bool grows = false;
      float top[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        top[r] = m[r];
#pragma unroll
        for (int u = 0; u < STEPS; ++u) top[r] = fmaxf(top[r], x[r][u]);
        grows = grows || top[r] > m[r];
      }
      if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float f = exp2_fast(m[r] - (top[r] == -INFINITY ? 0.0f : top[r]));
          sum[r] *= f;
#pragma unroll
          for (int e = 0; e < E; ++e) acc[r][e] *= f;
          m[r] = top[r];
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float z = top[r] == -INFINITY ? 0.0f : top[r];
#pragma unroll
        for (int u = 0; u < STEPS; ++u) {
          x[r][u] = exp2_fast(x[r][u] - z);
          sum[r] += x[r][u];
        }
      }
#pragma unroll
      for (int u = 0; u < STEPS; ++u) {
        float vr[E];
        load_cols<E>(vr, base + (DC_KEYS + u * DC_GROUPS + g) * DP, l);
        if (whole) {
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int e = 0; e < E; e += 2) {
              const float2 a = fma2(make_float2(x[r][u], x[r][u]), make_float2(vr[e], vr[e + 1]),
                                    make_float2(acc[r][e], acc[r][e + 1]));
              acc[r][e] = a.x;
              acc[r][e + 1] = a.y;
            }
        } else {  // an unseen key's value, or what an earlier stage left, may be anything
          const int j = j0 + u * DC_GROUPS + g;
#pragma unroll
          for (int r = 0; r < R; ++r)
            if (u * DC_GROUPS + g < n && j < vis[r]) {
#pragma unroll
              for (int e = 0; e < E; ++e) acc[r][e] = fmaf(x[r][u], vr[e], acc[r][e]);
            }
        }
      }
      __syncwarp();
      if (lane == 0) jxd::mbar_arrive(&empty[st]);
      if (++out_st == nst) {
        out_st = 0;
        out_ph ^= 1u;
      }
      c.key += n;
      c.left -= n;
      if (wr == 0) produce();
    }
    if (!ok) break;
    c.advance(s, end, row_base);
    // join the warp's groups, store
    // the head's first position
    const long long seg = (sq.k0 + (long long)b * VOID) * s.kv_heads + (long long)hk * (sq.lk + VOID);
    const bool last = seg >= begin && seg + sq.lk <= end;
    int i = (row_base + row0) / s.group, hg = row_base + row0 - i * s.group;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float t = m[r];
      t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8));
      t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
      const float f = exp2_fast(m[r] - (t == -INFINITY ? 0.0f : t));
      float a = sum[r] * f;
      a += __shfl_xor_sync(0xffffffffu, a, 8);
      a += __shfl_xor_sync(0xffffffffu, a, 16);
      const float inv = !last ? f : a == 0.0f ? 0.0f : f / a;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[r][e] *= inv;
      const float4 y = sum_groups<E>(acc[r], g);
      if (row0 + r < all_rows) {
        const long long tok = sq.q0 + i;
        const int h = hk * s.group + hg, col = ((E == 16 ? g : g >> 1) * DC_LPK + l) * 4;
        float* out = last ? o + tok * s.ldo + (long long)h * s.dim
                          : part + ((w * 2 + (first_key == 0)) * (R * WR) + row0 + r) * (DP + 4);
        if (E == 16 || !(g & 1)) {
          if (!last || vec_o) {
            if (col < s.dim) *reinterpret_cast<float4*>(out + col) = y;
          } else {
            if (col < s.dim) out[col] = y.x;
            if (col + 1 < s.dim) out[col + 1] = y.y;
            if (col + 2 < s.dim) out[col + 2] = y.z;
            if (col + 3 < s.dim) out[col + 3] = y.w;
          }
        }
        if (lane == 0) {
          if (!last) {
            out[DP] = t;
            out[DP + 1] = a;
          } else if (lse) {
            lse[(long long)h * s.total_q + tok] = a == 0.0f ? -INFINITY : (t + log2f(a)) * LN2;
          }
        }
      }
      if (++hg == s.group) {
        hg = 0;
        ++i;
      }
    }
  }
  // not before: the join's blocks would wait where rings still stream (37.0 us against 33.2 at the start of the kernel)
  asm volatile("griddepcontrol.launch_dependents;");
  if (!ok && wr == 0 && (!VEC || lane == 0)) {  // every copy has landed before the CTA may end
    unsigned long long end = 0;  // for all of them
    for (int u = max(0, issued - nst); u < issued; ++u)
      wait_suspended(&full[u % nst], (uint32_t)(u / nst) & 1u, s.err, end);
  }
}

// One block per (query row, head): the pieces in order; rows without keys; rows
// behind the ones that the rings took (where the caller's hint was too small).
// JN_WARPS warps load JN_AHEAD pieces each at a time: 4 and 8, or 32 and 4 where the
// pieces are many (4 rows, 4 heads, 14400 keys, 257 pieces a head: both kernels 22 us against 39).
template <int JN_WARPS, int JN_AHEAD>
__global__ void __launch_bounds__(32 * JN_WARPS)
    attn_join_kernel(const __grid_constant__ Shape s, const float* __restrict__ q, const float* __restrict__ k,
                     const float* __restrict__ v, const float* part, float* o, float* lse, long long per,
                     int ring_rows, int DP, int row_base, int last_pass) {
  __shared__ float red[2 * JN_WARPS];
  __shared__ float4 acc[JN_WARPS][32];
  const long long tok = blockIdx.x / (unsigned)s.heads;
  const int h = (int)(blockIdx.x % (unsigned)s.heads), hk = h / s.group;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = seq_of_row(s.cu_q, s.batch, tok);
  const Seq sq = seq_bounds(s, b);
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the rings' results are complete and visible behind it
  if (tok < sq.q0 || tok >= sq.q0 + sq.lq) return;
  const int i = (int)(tok - sq.q0);
  const long long row = (long long)i * s.group + h % s.group - row_base;
  if (row < 0 || (row >= ring_rows && !last_pass)) return;  // another pass's
  float* out = o + tok * s.ldo + (long long)h * s.dim;
  if (row >= ring_rows || sq.lk == 0) {
    if (warp == 0)
      row_fwd(q + tok * s.ldq + (long long)h * s.dim, k + sq.k0 * s.ldk + (long long)hk * s.dim,
              v + sq.k0 * s.ldv + (long long)hk * s.dim, out, lse ? lse + (long long)h * s.total_q + tok : nullptr,
              sq.visible(i, s.causal), s.dim, s.ldk, s.ldv, s.scale);
    return;
  }
  const long long seg = (sq.k0 + (long long)b * VOID) * s.kv_heads + (long long)hk * (sq.lk + VOID);
  const long long w0 = seg / per;
  const int n = (int)((seg + sq.lk - 1) / per - w0) + 1;
  if (n == 1) return;
  // piece z lies in ring w0 + z's slot 1 if it starts the head, else in slot 0
  auto piece = [&](int z) { return part + (((w0 + z) * 2 + (z == 0)) * ring_rows + row) * (DP + 4); };
  // each warp takes every JN_WARPS-th piece, a lane four columns; the first ones are loaded before the maximum is known
  const bool in = lane * 4 < DP;
  float4 x[JN_AHEAD];
#pragma unroll
  for (int e = 0; e < JN_AHEAD; ++e) {
    const int z = warp + JN_WARPS * e;
    x[e] = in && z < n ? reinterpret_cast<const float4*>(piece(z))[lane] : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  float top = -INFINITY;
  for (int z = threadIdx.x; z < n; z += 32 * JN_WARPS) top = fmaxf(top, piece(z)[DP]);
#pragma unroll
  for (int e = 16; e > 0; e >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, e));
  if (lane == 0) red[warp] = top;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < JN_WARPS; ++e) top = fmaxf(top, red[e]);
  const float base = top == -INFINITY ? 0.0f : top;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  float t = 0.0f;
  for (int z0 = warp; z0 < n; z0 += JN_WARPS * JN_AHEAD) {
    float f[JN_AHEAD];
#pragma unroll
    for (int e = 0; e < JN_AHEAD; ++e) {
      const int z = z0 + JN_WARPS * e;
      f[e] = z < n ? exp2_fast(piece(z)[DP] - base) : 0.0f;
      t += z < n ? piece(z)[DP + 1] * f[e] : 0.0f;
    }
#pragma unroll
    for (int e = 0; e < JN_AHEAD; ++e) {
      a.x = fmaf(x[e].x, f[e], a.x);
      a.y = fmaf(x[e].y, f[e], a.y);
      a.z = fmaf(x[e].z, f[e], a.z);
      a.w = fmaf(x[e].w, f[e], a.w);
      const int z = z0 + JN_WARPS * (JN_AHEAD + e);
      x[e] = in && z < n ? reinterpret_cast<const float4*>(piece(z))[lane] : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
  acc[warp][lane] = a;
  if (lane == 0) red[JN_WARPS + warp] = t;
  __syncthreads();
  if (warp == 0) {
    t = 0.0f;
    a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int e = 0; e < JN_WARPS; ++e) {
      t += red[JN_WARPS + e];
      a.x += acc[e][lane].x;
      a.y += acc[e][lane].y;
      a.z += acc[e][lane].z;
      a.w += acc[e][lane].w;
    }
    const float inv = t == 0.0f ? 0.0f : 1.0f / t;
    const int c = lane * 4;
    if (c < s.dim) out[c] = a.x * inv;
    if (c + 1 < s.dim) out[c + 1] = a.y * inv;
    if (c + 2 < s.dim) out[c + 2] = a.z * inv;
    if (c + 3 < s.dim) out[c + 3] = a.w * inv;
    if (lane == 0 && lse) lse[(long long)h * s.total_q + tok] = t == 0.0f ? -INFINITY : (top + log2f(t)) * LN2;
  }
}

using DecodeKernel = void (*)(Shape, CUtensorMap, CUtensorMap, const float*, const float*, const float*, float*, float*, float*, long long, int, int);

template <int R>
DecodeKernel kernel_of(int DP, bool vec) {
  if (DP == 128) return vec ? attn_decode_kernel<R, 128, true> : attn_decode_kernel<R, 128, false>;
  return vec ? attn_decode_kernel<R, 64, true> : attn_decode_kernel<R, 64, false>;
}

}  // namespace

namespace jxa {

// rows: query rows per key head of the longest sequence, a hint.
int attention_decode(const Shape& s, const float* q, const float* k, const float* v, float* o, float* lse,
                     long long rows, cudaStream_t st) {
  const int DP = s.dim <= 64 ? 64 : 128;
  auto a16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  const bool vec = s.total_k > 0 && !(s.dim & 3) && !(s.ldk & 3) && !(s.ldv & 3) && a16(k) && a16(v) &&
                   s.ldk < (1LL << 37) && s.ldv < (1LL << 37);  // what a tensor map takes
  const int R = rows <= 1 ? 1 : rows <= 2 ? 2 : 4;
  const int WR = rows <= 4 ? 1 : rows <= 8 ? 2 : rows <= 16 ? 4 : 8;
  const int passes = (int)std::max<long long>(1, (rows + R * WR - 1) / (R * WR));  // K and V are read once a pass
  const DecodeKernel kernel = R == 1 ? kernel_of<1>(DP, vec) : R == 2 ? kernel_of<2>(DP, vec) : kernel_of<4>(DP, vec);
  if (int rc = prepare_kernel((const void*)kernel, 8 + (R >> 1) * 4 + (DP == 128) * 2 + vec, dc_smem(DP), 0)) return rc;
  CUtensorMap map_k = {}, map_v = {};
  if (vec) {
    const uint64_t dims[3] = {(uint64_t)s.dim, (uint64_t)s.total_k, (uint64_t)s.kv_heads};
    const uint64_t in_k[2] = {(uint64_t)s.ldk * 4, (uint64_t)s.dim * 4}, in_v[2] = {(uint64_t)s.ldv * 4, in_k[1]};
    const uint32_t box[2] = {(uint32_t)DP, DC_KEYS};
    if (int rc = jx::tensor_map_f32_3d(&map_k, k, dims, in_k, box)) return rc;
    if (int rc = jx::tensor_map_f32_3d(&map_v, v, dims, in_v, box)) return rc;
  }
  // positions per ring: an equal share, 32 at least
  const int max_rings = jx::num_sms() * (DC_WARPS / WR);
  const long long all = (s.total_k + (long long)s.batch * VOID) * s.kv_heads;
  const long long per = std::max<long long>(32, ((all + max_rings - 1) / max_rings + 7) / 8 * 8);
  const int rings = (int)((all + per - 1) / per);
  const int grid = std::min(jx::num_sms(), rings);
  void* part = nullptr;
  if (int rc = jx::scratch_get(sizeof(float) * (size_t)grid * (DC_WARPS / WR) * 2 * R * WR * (DP + 4), &part, st))
    return rc;
  const bool wide = rings > 32LL * s.batch * s.kv_heads;  // more pieces a head, on average, than four warps load at once
  cudaError_t e = cudaSuccess;
  for (int p = 0; p < passes && e == cudaSuccess; ++p) {
    const int row_base = p * R * WR;
    kernel<<<grid, 32 * DC_WARPS, dc_smem(DP), st>>>(s, map_k, map_v, q, k, v, o, lse, static_cast<float*>(part), per,
                                                     WR, row_base);
    // the join's blocks may start while the last rings finish; they wait for them before they read
    e = cudaGetLastError();
    if (e == cudaSuccess) {
      const auto join = wide ? attn_join_kernel<32, 4> : attn_join_kernel<4, 8>;
      e = launch_overlapped(join, s.total_q * s.heads, wide ? 1024 : 128, 0, st, s, q, k, v,
                            static_cast<const float*>(part), o, lse, per, R * WR, DP, row_base, (int)(p == passes - 1));
    }
  }
  jx::scratch_release(part, st);
  return e == cudaSuccess ? JX_OK : jx::check_cuda(e, "attn_decode_kernel");
}

}  // namespace jxa
