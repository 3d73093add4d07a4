// attn_bwd.cu -- attention's gradients on the tensor cores (operands and sums as
// in attn_tc.cuh).
//
// Two kernels, each with its sums in registers, so that every sum has a fixed
// order and nothing is added atomically; the price is that the scores and
// dout v^T are computed in both (seven products a tile instead of five).
//
// dq: one CTA per (128 query rows, head), streaming K and V tiles.
//   S = Q K^T, dP = dO V^T        Q and dO in tensor memory
//   dS = P (dP - delta)           P = exp2(S f - lse2)
//   dQ += dS K                    dS in tensor memory, over S's columns
// dk, dv: one CTA per (128 keys, key head, part of the query rows), streaming
// blocks of 64 rows of Q and dO of every head of the group.
//   S^T = K Q^T, dP^T = V dO^T    K and V in tensor memory
//   dV += P^T dO, dK += dS^T Q    P^T over S^T's columns, dS^T over dP^T's
// An operand computed here needs its scale before its largest value is known:
// P <= 1 and |dP - delta| <= |dout row| |v row| + |delta| (norms) bound dS; it
// overestimates by some bits of the 39 there are (a row of 2^14 keys with equal
// weights keeps 21 bits of each dS).
#include <algorithm>

#include "attn_tc.cuh"

namespace {

using namespace jxa;
using jxg::wait_bounded;

constexpr int BW_THREADS = 384;  // warp 0 copies, warp 1 MMA, warps 4..11 the rest
constexpr int BW_FIRST = 4;
constexpr int BW_LAUNCH_REGS = 168;
constexpr int BW_LOW_REGS = 56;
constexpr int BW_HIGH_REGS = 216;
static_assert(128 * BW_LOW_REGS + 256 * BW_HIGH_REGS <= BW_THREADS * BW_LAUNCH_REGS,
              "register split exceeds the launch allocation");

struct BwdTiles {
  const uint8_t *q, *k, *v, *d;  // tiles; d is dout
  const float *inv_q, *inv_k, *inv_v, *inv_d;
  const int *bad_q, *bad_k, *bad_v, *bad_d;
  const float *norm_v, *norm_d, *lse2, *delta, *delta_top;
  int q_tiles, k_tiles, parts;
  const int *order_q, *order_k;
  float *part_k, *part_v;  // [parts][total_k * kv_heads * dim], used where parts > 1
};

// 1 / f of a power of two.
__device__ __forceinline__ float inverse_pow2(float f) { return __uint_as_float((254u << 23) - __float_as_uint(f)); }

// Scale for a computed operand of magnitude <= bound, at most 2^100.
__device__ __forceinline__ float bound_scale(float bound) {
  const int e = (int)(__float_as_uint(bound) >> 23);
  return __uint_as_float((uint32_t)(268 - min(max(e, 41), 254)) << 23);
}

// The largest of a row's two halves; `xch` is [2][128].
__device__ __forceinline__ float row_max(float v, float* xch, int half, int row, int id) {
  xch[half * 128 + row] = v;
  pair_sync(id);
  v = fmaxf(v, xch[(half ^ 1) * 128 + row]);
  pair_sync(id);
  return v;
}

// A row's half from an area into tensor memory; returns its scale's exponent and, with `norm`, the row's norm.
template <int DP>
__device__ __forceinline__ int stay_row(const uint8_t* area, int half, int row, bool negate, uint32_t taddr, float* xch,
                                        int id, float* norm) {
  float x[DP / 2];
  const float t = __uint_as_float(half_from_area<DP>(x, area, row, half));
  const int e = (int)(__float_as_uint(row_max(t, xch, half, row, id)) >> 23);
  const float f = scale_of(e);
  if (norm) {
    float n = 0.0f;
#pragma unroll
    for (int c = 0; c < DP / 2; ++c) n = fmaf(x[c] * f, x[c] * f, n);
    xch[half * 128 + row] = n;
    pair_sync(id);
    *norm = sqrtf(n + xch[(half ^ 1) * 128 + row]) * inverse_of(e);
    pair_sync(id);
  }
  row_half_store<DP>(x, negate ? -f : f, taddr, half);
  return e;
}

// acc += part * factor for this thread's DP/2 columns of a tensor-memory sum.
template <int DP>
__device__ __forceinline__ void drain(float (&acc)[DP / 2], uint32_t taddr, float factor) {
  const float2 f2 = make_float2(factor, factor);
#pragma unroll
  for (int c = 0; c < DP / 2; c += 16) {
    uint32_t r[16];
    jxd::tmem_ld16(taddr + c, r);
    jxd::tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      const float2 v = fma2(make_float2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), f2,
                            make_float2(acc[c + i], acc[c + i + 1]));
      acc[c + i] = v.x;
      acc[c + i + 1] = v.y;
    }
  }
}

// ---- dq ------------------------------------------------------------------------
// Tensor memory: Q, dO, X (scores), Y (dP) and the sum's part D.  At DP = 128 the
// first four fill it: dS goes over X and D over Y, and S(j+1) has to wait for
// dS(j) K.  At DP = 64 D has its own columns: dS goes over Y, and S(j+1) runs
// while dS(j) is computed.
template <int DP>
struct DqLayout {
  static constexpr bool AHEAD = DP == 64;
  static constexpr uint32_t Q = 0, DO = AHEAD ? 64 : 128, X = AHEAD ? 128 : 256, Y = AHEAD ? 256 : 384;
  static constexpr uint32_t DS = AHEAD ? Y : X, D = AHEAD ? 384 : Y;
};
__host__ __device__ constexpr int dq_k_stages(int DP) { return DP == 128 ? 2 : 3; }
__host__ __device__ constexpr int dq_v_stages(int DP) { return DP == 128 ? 1 : 2; }
__host__ __device__ constexpr size_t dq_smem(int DP) {
  return (size_t)(dq_k_stages(DP) + dq_v_stages(DP)) * tile_bytes(DP) + 1024 + 2 * 128 * 4 + 256;
}

template <int DP>
__global__ void __launch_bounds__(BW_THREADS, 1)
    attn_dq_kernel(const __grid_constant__ Shape s, const __grid_constant__ BwdTiles bt, const float* __restrict__ q,
                   const float* __restrict__ k, const float* __restrict__ v, const float* __restrict__ o,
                   const float* __restrict__ lse, const float* __restrict__ dout, float* dq) {
  using L = DqLayout<DP>;
  constexpr int KS = dq_k_stages(DP), VS = dq_v_stages(DP), STAGE = tile_bytes(DP), PART = tile_part(DP);
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = jxd::smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
  float* xch = reinterpret_cast<float*>(smem + (KS + VS) * STAGE);
  uint64_t* kfull = reinterpret_cast<uint64_t*>(xch + 2 * 128);
  uint64_t* kempty = kfull + KS;
  uint64_t* vfull = kempty + KS;
  uint64_t* vempty = vfull + VS;
  uint64_t* stayfull = vempty + VS;
  uint64_t* sfull = stayfull + 1;
  uint64_t* dpfull = sfull + 1;
  uint64_t* dsfull = dpfull + 1;
  uint64_t* dqfull = dsfull + 1;
  uint64_t* dfree = dqfull + 1;  // D is drained
  uint64_t* xfree = dfree + 1;   // X is read
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(xfree + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int id = bt.order_q[blockIdx.x / (unsigned)s.heads], h = (int)(blockIdx.x % (unsigned)s.heads);
  int jt;
  const int b = seq_of_tile(s.cu_q, s.batch, id, &jt);
  const Seq sq = seq_bounds(s, b);
  if (jt < 0 || (long long)jt * TILE >= sq.lq) return;
  const int i0 = jt * TILE, rows = min(TILE, sq.lq - i0);
  const int hk = h / s.group;
  const int nb = (sq.visible(i0 + rows - 1, s.causal) + TILE - 1) / TILE;
  const long long slot0 = (long long)first_tile(sq.k0, b) * s.kv_heads + hk;
  const long long qslot = ((long long)first_tile(sq.q0, b) + jt) * s.heads + h;

  const long long hd = (long long)h * s.dim;
  // Q passes through K's last stage, dout through V's last one; the copies for the first stages start at once
  uint8_t *area_q = smem + (KS - 1) * STAGE, *area_d = smem + (KS + VS - 1) * STAGE;
  auto copy_k = [&](int j) {
    jxd::mbar_arrive_expect_tx(&kfull[j % KS], STAGE);
    bulk_load(jxd::smem_u32(smem + j % KS * STAGE), bt.k + (slot0 + (long long)j * s.kv_heads) * STAGE, STAGE,
              &kfull[j % KS]);
  };
  auto copy_v = [&](int j) {
    jxd::mbar_arrive_expect_tx(&vfull[j % VS], STAGE);
    bulk_load(jxd::smem_u32(smem + (KS + j % VS) * STAGE), bt.v + (slot0 + (long long)j * s.kv_heads) * STAGE, STAGE,
              &vfull[j % VS]);
  };
  bool bad = false;
  if (warp == 0 && lane == 0) {
    for (int i = 0; i < KS; ++i) {
      jxd::mbar_init(&kfull[i], 1);
      jxd::mbar_init(&kempty[i], 1);
    }
    for (int i = 0; i < VS; ++i) {
      jxd::mbar_init(&vfull[i], 1);
      jxd::mbar_init(&vempty[i], 1);
    }
    jxd::mbar_init(stayfull, 8);
    jxd::mbar_init(sfull, 1);
    jxd::mbar_init(dpfull, 1);
    jxd::mbar_init(dsfull, 8);
    jxd::mbar_init(dqfull, 1);
    jxd::mbar_init(dfree, 8);
    jxd::mbar_init(xfree, 8);
    *abort_flag = 0;
    jxd::fence_mbar_init();
    jxd::fence_proxy_async_smem();
    if (nb > 0) copy_k(0);
  } else if (warp == 1) {
    jxd::tmem_alloc(tmem_slot, 512);
    jxd::tmem_relinquish();
  } else if (warp >= BW_FIRST) {
    const int tid = threadIdx.x - 32 * BW_FIRST;
    float4 f[DP / 8], g[DP / 8];
    rows_load<DP>(f, q + (sq.q0 + i0) * s.ldq + hd, s.ldq, rows, s.dim, aligned16(q, s.dim, s.ldq), tid);
    rows_load<DP>(g, dout + (sq.q0 + i0) * s.ldo + hd, s.ldo, rows, s.dim, aligned16(dout, s.dim, s.ldo), tid);
    rows_to_area<DP>(area_q, f, tid);
    rows_to_area<DP>(area_d, g, tid);
  } else if (warp >= 2) {
    if (threadIdx.x == 64) bad = bt.bad_q[qslot] || bt.bad_d[qslot];
    for (int j = (int)threadIdx.x - 64; j < nb; j += 64)
      bad = bad || bt.bad_k[slot0 + (long long)j * s.kv_heads] || bt.bad_v[slot0 + (long long)j * s.kv_heads];
  }
  jxd::tc_fence_before();
  bad = __syncthreads_or(bad);
  jxd::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (bad) {
    // row by row, in plain f32
    for (int r = warp; r < rows; r += BW_THREADS / 32) {
      const long long t = sq.q0 + i0 + r;
      row_dq(q + t * s.ldq + hd, k + sq.k0 * s.ldk + (long long)hk * s.dim, v + sq.k0 * s.ldv + (long long)hk * s.dim,
             o + t * s.ldo + hd, dout + t * s.ldo + hd, lse[(long long)h * s.total_q + t], dq + t * s.ldq + hd,
             sq.visible(i0 + r, s.causal), s.dim, s.ldk, s.ldv, s.scale);
    }
    if (warp == 0 && lane == 0 && nb > 0) wait_bounded(&kfull[0], 0, s.err);  // the copy has landed
    if (warp == 1) {
      __syncwarp();
      jxd::tmem_dealloc(tmem, 512);
    }
    return;
  }

  if (warp < BW_FIRST) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(BW_LOW_REGS));
    if (warp == 0 && jxd::elect_one()) {
      int j = 0, nv = 0;
      bool ok = wait_bounded(stayfull, 0, s.err);  // the areas are free again
      for (; ok && j < nb; ++j) {
        if (j > 0) {
          if (!(ok = !*abort_flag && wait_bounded(&kempty[j % KS], (uint32_t)(j / KS + 1) & 1u, s.err))) break;
          copy_k(j);
        }
        if (!(ok = !*abort_flag && wait_bounded(&vempty[j % VS], (uint32_t)(j / VS + 1) & 1u, s.err))) { ++j; break; }
        copy_v(j);
        ++nv;
      }
      if (!ok) j = max(j, min(nb, 1));  // the first K is under way in any case
      if (nv < nb) *abort_flag = 1;
      // every copy has landed before the CTA may end
      for (int u = max(0, j - KS); u < j; ++u) wait_bounded(&kfull[u % KS], (uint32_t)(u / KS) & 1u, s.err);
      for (int u = max(0, nv - VS); u < nv; ++u) wait_bounded(&vfull[u % VS], (uint32_t)(u / VS) & 1u, s.err);
    }
    if (warp == 1 && nb > 0 && jxd::elect_one()) {
      constexpr uint32_t id_s = idesc_f16(128, false), id_o = idesc_f16(DP, true);
      const uint32_t sbase = jxd::smem_u32(smem);
      bool ok = wait_bounded(stayfull, 0, s.err);
      // 128 x 128 scores of a row operand in tensor memory and a streamed tile
      auto scores = [&](uint32_t d, uint32_t a0, uint32_t tile) {
        auto step = [&](int ks, uint32_t a, uint32_t part, uint32_t acc) {
          mma_f16_ts(d, a0 + a + ks * 8, jxd::smem_desc_k_sw128(tile + part + (ks >> 2) * PANEL + (ks & 3) * 32), id_s,
                     acc);
        };
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) {
          step(ks, DP / 2, 0, ks > 0);
          step(ks, 0, PART, 1);
        }
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) step(ks, 0, 0, 1);
      };
      auto ready = [&](uint64_t* bar, int n) {
        ok = ok && !*abort_flag && wait_bounded(bar, (uint32_t)n & 1u, s.err);
        jxd::tc_fence_after();
        return ok;
      };
      auto q_scores = [&](int j) {
        if (!ready(&kfull[j % KS], j / KS)) return;
        if (L::AHEAD && j > 0 && !ready(xfree, j - 1)) return;
        scores(tmem + L::X, tmem + L::Q, sbase + (j % KS) * STAGE);
        jxd::mma_commit(sfull);
      };
      q_scores(0);
      for (int j = 0; ok && j < nb; ++j) {
        if (!ready(&vfull[j % VS], j / VS)) break;
        if (!L::AHEAD && !ready(dfree, j + 1)) break;  // D is Y
        scores(tmem + L::Y, tmem + L::DO, sbase + (KS + j % VS) * STAGE);
        jxd::mma_commit(dpfull);
        jxd::mma_commit(&vempty[j % VS]);
        if (L::AHEAD && j + 1 < nb) q_scores(j + 1);
        if (!ready(dsfull, j)) break;
        if (L::AHEAD && !ready(dfree, j + 1)) break;
        const uint32_t kt = sbase + (j % KS) * STAGE;
        auto step = [&](int ks, uint32_t a, uint32_t part, uint32_t acc) {
          mma_f16_ts(tmem + L::D, tmem + L::DS + a + (ks >> 1) * 32 + (ks & 1) * 8,
                     smem_desc_mn_sw128(kt + part + ks * 2048, PANEL), id_o, acc);
        };
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          step(ks, 16, 0, ks > 0);
          step(ks, 0, PART, 1);
        }
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) step(ks, 0, 0, 1);
        jxd::mma_commit(dqfull);
        jxd::mma_commit(&kempty[j % KS]);
        if (!L::AHEAD && j + 1 < nb) q_scores(j + 1);
      }
      if (!ok) *abort_flag = 1;
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(BW_HIGH_REGS));
    const int quarter = warp & 3, half = (warp - BW_FIRST) >> 2, row = quarter * 32 + lane, bar = 1 + quarter;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    float norm_d;
    const int e_q = stay_row<DP>(area_q, half, row, s.scale < 0.0f, tmem + lanes + L::Q, xch, bar, nullptr);
    const int e_d = stay_row<DP>(area_d, half, row, false, tmem + lanes + L::DO, xch, bar, &norm_d);
    tmem_st_wait();
    jxd::fence_proxy_async_smem();  // the areas become copies' destinations
    jxd::tc_fence_before();
    __syncwarp();
    if (lane == 0) jxd::mbar_arrive(stayfull);
    const float f_row = inverse_of(e_q) * (fabsf(s.scale) * LOG2E), inv_d = inverse_of(e_d);
    const float lse2 = bt.lse2[qslot * TILE + row], delta = bt.delta[qslot * TILE + row];
    const int vis = row < rows ? sq.visible(i0 + row, s.causal) : 0;
    const int vis_all = sq.visible(i0, s.causal);

    float acc[DP / 2];
#pragma unroll
    for (int c = 0; c < DP / 2; ++c) acc[c] = 0.0f;
    float g_prev = 0.0f;
    bool ok = true;
    auto done = [&](uint64_t* b8) {
      jxd::tc_fence_before();
      __syncwarp();
      if (lane == 0) jxd::mbar_arrive(b8);
    };
    auto add_part = [&](int j) {
      ok = ok && warp_wait(dqfull, (uint32_t)j & 1u, abort_flag, s.err);
      jxd::tc_fence_after();
      drain<DP>(acc, tmem + lanes + L::D + half * (DP / 2), g_prev);
      done(dfree);
    };
    for (int j = 0; j < nb; ++j) {
      const long long slot = slot0 + (long long)j * s.kv_heads;
      const float inv_k = bt.inv_k[slot], inv_v = bt.inv_v[slot], norm_v = bt.norm_v[slot];
      if (!L::AHEAD && j > 0) add_part(j - 1);
      ok = ok && warp_wait(sfull, (uint32_t)j & 1u, abort_flag, s.err);
      jxd::tc_fence_after();
      const float f = f_row * inv_k;
      const float2 f2 = make_float2(f, f), l2 = make_float2(-lse2, -lse2);
      float2 p[32];
#pragma unroll
      for (int c = 0; c < 64; c += 32) {
        uint32_t r[32];
        jxd::tmem_ld32(tmem + lanes + L::X + half * 64 + c, r);
        jxd::tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          const float2 z = fma2(make_float2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), f2, l2);
          p[(c + i) / 2] = make_float2(exp2_fast(z.x), exp2_fast(z.y));
        }
      }
      if (L::AHEAD) done(xfree);
      if (j * TILE + TILE > vis_all) {  // some row does not see all of the tile's keys
        const int key0 = j * TILE + half * 64;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          if (key0 + 2 * i >= vis) p[i].x = 0.0f;
          if (key0 + 2 * i + 1 >= vis) p[i].y = 0.0f;
        }
      }
      // P is at most 2^14
      const float fd = inv_d * inv_v, sc = bound_scale(16384.0f * (norm_d * norm_v + fabsf(delta)));
      const float pf = sc * fd, dl = -delta * inverse_pow2(fd);
      const float2 pf2 = make_float2(pf, pf), one2 = make_float2(1.0f, 1.0f), dl2 = make_float2(dl, dl);
#pragma unroll
      for (int i = 0; i < 32; ++i) p[i] = mul2(p[i], pf2);
      if (L::AHEAD && j > 0) add_part(j - 1);
      ok = ok && warp_wait(dpfull, (uint32_t)j & 1u, abort_flag, s.err);
      jxd::tc_fence_after();
#pragma unroll
      for (int c = 0; c < 64; c += 32) {
        uint32_t r[32], hi[16], lo[16];
        jxd::tmem_ld32(tmem + lanes + L::Y + half * 64 + c, r);
        jxd::tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float2 e = fma2(make_float2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), one2, dl2);
          const float2 ds = mul2(p[c / 2 + i], e);
          split_half(ds.x, ds.y, hi[i], lo[i]);
        }
        tmem_st16(tmem + lanes + L::DS + half * 64 + c, hi);
        tmem_st16(tmem + lanes + L::DS + half * 64 + c + 16, lo);
      }
      tmem_st_wait();
      done(dsfull);
      g_prev = inv_k * inverse_pow2(sc) * 6.103515625e-05f;  // P's 2^14
    }
    if (nb > 0) add_part(nb - 1);
    // every MMA has retired: the stages are free
    half_to_area<DP>(smem, acc, s.scale, row, half);
    movers_sync();
    rows_store<DP>(dq + (sq.q0 + i0) * s.ldq + hd, s.ldq, smem, rows, s.dim, aligned16(dq, s.dim, s.ldq),
                   threadIdx.x - 32 * BW_FIRST);
  }
  jxd::tc_fence_before();
  __syncthreads();
  jxd::tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    jxd::tmem_dealloc(tmem, 512);
  }
}

// ---- dk, dv --------------------------------------------------------------------
// Query rows per step: 128 at DP = 64, where the parts of dV and dK have columns of
// their own (Z and W); 64 at DP = 128, where they share Z.  (An MMA of 64 columns
// takes 45 cycles where half of one of 128 would be 32.)
template <int DP>
struct KvLayout {
  static constexpr bool APART = DP == 64;
  static constexpr int BLK = APART ? 128 : 64;
  static constexpr uint32_t K = 0, V = APART ? 64 : 128, X = APART ? 128 : 256, Y = APART ? 256 : 320, Z = 384,
                            W = APART ? 448 : 384;
  static constexpr int PANEL_BYTES = BLK * 128;             // of a block
  static constexpr int STAGE = DP / 64 * 2 * PANEL_BYTES;   // one block of Q or of dout: 32 KB
};
constexpr int KV_STAGES = 3;  // of Q and of dout each
__host__ __device__ constexpr size_t kv_smem(int DP) {
  return (size_t)2 * KV_STAGES * (DP == 64 ? KvLayout<64>::STAGE : KvLayout<128>::STAGE) + 1024 +
         KV_STAGES * 1024 /*lse2, delta*/ + 2 * 128 * 4 + 256;
}

template <int DP>
__global__ void __launch_bounds__(BW_THREADS, 1)
    attn_dkv_kernel(const __grid_constant__ Shape s, const __grid_constant__ BwdTiles bt, const float* __restrict__ q,
                    const float* __restrict__ k, const float* __restrict__ v, const float* __restrict__ o,
                    const float* __restrict__ lse, const float* __restrict__ dout, float* dk, float* dv) {
  using L = KvLayout<DP>;
  constexpr int ST = KV_STAGES, BLK = L::BLK, STAGE = L::STAGE, PART = STAGE / 2, HPANEL = L::PANEL_BYTES;
  constexpr int PER_TILE = TILE / BLK;  // blocks of a tile
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = jxd::smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
  float* stats = reinterpret_cast<float*>(smem + 2 * ST * STAGE);  // [ST][lse2 BLK, delta BLK]
  float* xch = stats + ST * 2 * BLK;
  uint64_t* qfull = reinterpret_cast<uint64_t*>(xch + 2 * 128);
  uint64_t* qempty = qfull + ST;
  uint64_t* dfull = qempty + ST;
  uint64_t* dempty = dfull + ST;
  uint64_t* stayfull = dempty + ST;
  uint64_t* sfull = stayfull + 1;
  uint64_t* pfull = sfull + 1;
  uint64_t* dpfull = pfull + 1;
  uint64_t* dsfull = dpfull + 1;
  uint64_t* zfull = dsfull + 1;
  uint64_t* zfree = zfull + 1;  // dV's part
  uint64_t* wfull = zfree + 1;  // dK's
  uint64_t* wfree = wfull + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(wfree + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // the keys that the most rows see start first
  unsigned w = blockIdx.x;
  const int part = (int)(w % (unsigned)bt.parts);
  w /= (unsigned)bt.parts;
  const int hk = (int)(w % (unsigned)s.kv_heads), id = bt.order_k[w / (unsigned)s.kv_heads];
  int jt;
  const int b = seq_of_tile(s.cu_k, s.batch, id, &jt);
  const Seq sq = seq_bounds(s, b);
  if (jt < 0 || (long long)jt * TILE >= sq.lk) return;
  const int j0 = jt * TILE, rows = min(TILE, sq.lk - j0);
  const int blk0 = sq.first_row(j0, s.causal) / BLK;
  const int nblk = max(0, (sq.lq + BLK - 1) / BLK - blk0);
  const long long steps = (long long)s.group * nblk;
  const int it0 = (int)(steps * part / bt.parts), it1 = (int)(steps * (part + 1) / bt.parts);
  const long long qslot0 = (long long)first_tile(sq.q0, b) * s.heads + (long long)hk * s.group;
  const long long kslot = ((long long)first_tile(sq.k0, b) + jt) * s.kv_heads + hk;
  const int h0 = hk * s.group;
  const long long kd = (long long)hk * s.dim;
  // where this part's sums go
  float* out_k = bt.parts > 1 ? bt.part_k + (long long)part * s.total_k * s.kv_heads * s.dim : dk;
  float* out_v = bt.parts > 1 ? bt.part_v + (long long)part * s.total_k * s.kv_heads * s.dim : dv;
  const long long ld_k = bt.parts > 1 ? (long long)s.kv_heads * s.dim : s.ldk;
  const long long ld_v = bt.parts > 1 ? (long long)s.kv_heads * s.dim : s.ldv;

  const int n = it1 - it0;
  // K passes through the last stages of Q's ring, V through those of dout's; the first stages' copies start at once
  constexpr int AREA_STAGES = area_bytes(DP) / STAGE;
  uint8_t *area_k = smem + (ST - AREA_STAGES) * STAGE, *area_v = smem + (2 * ST - AREA_STAGES) * STAGE;
  // a block: its rows of each part's panels
  auto load = [&](uint8_t* dst, const uint8_t* tile, int hb, uint64_t* bar) {
#pragma unroll
    for (int e = 0; e < 2 * (DP / 64); ++e)
      bulk_load(jxd::smem_u32(dst + e * HPANEL), tile + (long long)e * PANEL + hb * HPANEL, HPANEL, bar);
  };
  auto copy_q = [&](int u) {
    const int g = (it0 + u) / nblk, blk = blk0 + (it0 + u) % nblk, st = u % ST;
    const long long slot = qslot0 + (long long)(blk / PER_TILE) * s.heads + g;
    jxd::mbar_arrive_expect_tx(&qfull[st], STAGE + 2 * BLK * 4);
    load(smem + st * STAGE, bt.q + slot * tile_bytes(DP), blk % PER_TILE, &qfull[st]);
    bulk_load(jxd::smem_u32(stats + st * 2 * BLK), bt.lse2 + slot * TILE + blk % PER_TILE * BLK, BLK * 4, &qfull[st]);
    bulk_load(jxd::smem_u32(stats + st * 2 * BLK + BLK), bt.delta + slot * TILE + blk % PER_TILE * BLK, BLK * 4,
              &qfull[st]);
  };
  auto copy_d = [&](int u) {
    const int g = (it0 + u) / nblk, blk = blk0 + (it0 + u) % nblk, st = u % ST;
    const long long slot = qslot0 + (long long)(blk / PER_TILE) * s.heads + g;
    jxd::mbar_arrive_expect_tx(&dfull[st], STAGE);
    load(smem + (ST + st) * STAGE, bt.d + slot * tile_bytes(DP), blk % PER_TILE, &dfull[st]);
  };
  bool bad = false;
  if (warp == 0 && lane == 0) {
    for (int i = 0; i < ST; ++i) {
      jxd::mbar_init(&qfull[i], 1);
      jxd::mbar_init(&qempty[i], 1);
      jxd::mbar_init(&dfull[i], 1);
      jxd::mbar_init(&dempty[i], 1);
    }
    jxd::mbar_init(stayfull, 8);
    jxd::mbar_init(sfull, 1);
    jxd::mbar_init(pfull, 8);
    jxd::mbar_init(dpfull, 1);
    jxd::mbar_init(dsfull, 8);
    jxd::mbar_init(zfull, 1);
    jxd::mbar_init(zfree, 8);
    jxd::mbar_init(wfull, 1);
    jxd::mbar_init(wfree, 8);
    *abort_flag = 0;
    jxd::fence_mbar_init();
    jxd::fence_proxy_async_smem();
    if (n > 0) {
      copy_q(0);
      copy_d(0);
    }
  } else if (warp == 1) {
    jxd::tmem_alloc(tmem_slot, 512);
    jxd::tmem_relinquish();
  } else if (warp >= BW_FIRST) {
    const int tid = threadIdx.x - 32 * BW_FIRST;
    float4 f[DP / 8], g[DP / 8];
    rows_load<DP>(f, k + (sq.k0 + j0) * s.ldk + kd, s.ldk, rows, s.dim, aligned16(k, s.dim, s.ldk), tid);
    rows_load<DP>(g, v + (sq.k0 + j0) * s.ldv + kd, s.ldv, rows, s.dim, aligned16(v, s.dim, s.ldv), tid);
    rows_to_area<DP>(area_k, f, tid);
    rows_to_area<DP>(area_v, g, tid);
  } else if (warp >= 2) {
    if (threadIdx.x == 64) bad = bt.bad_k[kslot] || bt.bad_v[kslot];
    const int t0 = blk0 / PER_TILE, nt = nblk > 0 ? (sq.lq + TILE - 1) / TILE - t0 : 0;
    for (long long e = (int)threadIdx.x - 64; e < (long long)nt * s.group; e += 64) {
      const long long slot = qslot0 + (t0 + e / s.group) * s.heads + e % s.group;
      bad = bad || bt.bad_q[slot] || bt.bad_d[slot];
    }
  }
  jxd::tc_fence_before();
  bad = __syncthreads_or(bad);
  jxd::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (bad) {
    // row by row, in plain f32: the first part computes every row whole, the others add zeros
    for (int r = warp; r < rows; r += BW_THREADS / 32) {
      const long long t = sq.k0 + j0 + r;
      row_dkv(q + sq.q0 * s.ldq + (long long)h0 * s.dim, o + sq.q0 * s.ldo + (long long)h0 * s.dim,
              dout + sq.q0 * s.ldo + (long long)h0 * s.dim, lse + (long long)h0 * s.total_q + sq.q0,
              k + t * s.ldk + kd, v + t * s.ldv + kd, out_k + t * ld_k + kd, out_v + t * ld_v + kd,
              part == 0 ? sq.first_row(j0 + r, s.causal) : sq.lq, sq.lq, s.group, s.dim, s.ldq, s.ldo, s.total_q,
              s.scale);
    }
    if (warp == 0 && lane == 0 && n > 0) {  // the copies have landed
      wait_bounded(&qfull[0], 0, s.err);
      wait_bounded(&dfull[0], 0, s.err);
    }
    if (warp == 1) {
      __syncwarp();
      jxd::tmem_dealloc(tmem, 512);
    }
    return;
  }

  if (warp < BW_FIRST) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(BW_LOW_REGS));
    if (warp == 0 && jxd::elect_one()) {
      int u = min(n, 1), nd = u;
      bool ok = wait_bounded(stayfull, 0, s.err);  // the areas are free again
      for (; ok && u < n; ++u) {
        if (!(ok = !*abort_flag && wait_bounded(&qempty[u % ST], (uint32_t)(u / ST + 1) & 1u, s.err))) break;
        copy_q(u);
        if (!(ok = !*abort_flag && wait_bounded(&dempty[u % ST], (uint32_t)(u / ST + 1) & 1u, s.err))) { ++u; break; }
        copy_d(u);
        ++nd;
      }
      if (!ok) *abort_flag = 1;
      // every copy has landed before the CTA may end
      for (int e = max(0, u - ST); e < u; ++e) wait_bounded(&qfull[e % ST], (uint32_t)(e / ST) & 1u, s.err);
      for (int e = max(0, nd - ST); e < nd; ++e) wait_bounded(&dfull[e % ST], (uint32_t)(e / ST) & 1u, s.err);
    }
    if (warp == 1 && n > 0 && jxd::elect_one()) {
      constexpr uint32_t id_s = idesc_f16(BLK, false), id_o = idesc_f16(DP, true);
      const uint32_t sbase = jxd::smem_u32(smem);
      bool ok = wait_bounded(stayfull, 0, s.err);
      auto ready = [&](uint64_t* bar, int u) {
        return !*abort_flag && wait_bounded(bar, (uint32_t)u & 1u, s.err);
      };
      // 128 x BLK scores
      auto scores = [&](uint32_t d, uint32_t a0, uint32_t tile) {
        auto step = [&](int ks, uint32_t a, uint32_t p, uint32_t acc) {
          mma_f16_ts(d, a0 + a + ks * 8, jxd::smem_desc_k_sw128(tile + p + (ks >> 2) * HPANEL + (ks & 3) * 32), id_s,
                     acc);
        };
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) {
          step(ks, DP / 2, 0, ks > 0);
          step(ks, 0, PART, 1);
        }
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) step(ks, 0, 0, 1);
      };
      // 128 x DP sums over the block's rows; a0 holds 16 columns of hi, 16 of lo for every 32 rows
      auto sums = [&](uint32_t d, uint32_t a0, uint32_t tile) {
        auto step = [&](int ks, uint32_t a, uint32_t p, uint32_t acc) {
          mma_f16_ts(d, a0 + a + (ks >> 1) * 32 + (ks & 1) * 8, smem_desc_mn_sw128(tile + p + ks * 2048, HPANEL), id_o,
                     acc);
        };
#pragma unroll
        for (int ks = 0; ks < BLK / 16; ++ks) {
          step(ks, 16, 0, ks > 0);
          step(ks, 0, PART, 1);
        }
#pragma unroll
        for (int ks = 0; ks < BLK / 16; ++ks) step(ks, 0, 0, 1);
      };
      auto q_scores = [&](int u) {
        if (!ok || !(ok = ready(&qfull[u % ST], u / ST))) return;
        jxd::tc_fence_after();
        scores(tmem + L::X, tmem + L::K, sbase + (u % ST) * STAGE);
        jxd::mma_commit(sfull);
      };
      auto d_scores = [&](int u) {
        if (!ok || !(ok = ready(&dfull[u % ST], u / ST))) return;
        jxd::tc_fence_after();
        scores(tmem + L::Y, tmem + L::V, sbase + (ST + u % ST) * STAGE);
        jxd::mma_commit(dpfull);
      };
      q_scores(0);
      d_scores(0);
      for (int u = 0; ok && u < n; ++u) {
        // the sums' columns are drained: dV's of the step before, and dK's where they share them
        if (!(ok = ready(pfull, u) && ready(L::APART ? zfree : wfree, u + 1))) break;
        jxd::tc_fence_after();
        sums(tmem + L::Z, tmem + L::X, sbase + (ST + u % ST) * STAGE);
        jxd::mma_commit(zfull);
        jxd::mma_commit(&dempty[u % ST]);
        if (u + 1 < n) q_scores(u + 1);
        if (!ok || !(ok = ready(dsfull, u) && (L::APART ? ready(wfree, u + 1) : ready(zfree, u)))) break;
        jxd::tc_fence_after();
        sums(tmem + L::W, tmem + L::Y, sbase + (u % ST) * STAGE);
        jxd::mma_commit(wfull);
        jxd::mma_commit(&qempty[u % ST]);
        if (u + 1 < n) d_scores(u + 1);
      }
      if (!ok) *abort_flag = 1;
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(BW_HIGH_REGS));
    const int quarter = warp & 3, half = (warp - BW_FIRST) >> 2, row = quarter * 32 + lane, bar = 1 + quarter;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    float norm_v;
    const int e_k = stay_row<DP>(area_k, half, row, s.scale < 0.0f, tmem + lanes + L::K, xch, bar, nullptr);
    const int e_v = stay_row<DP>(area_v, half, row, false, tmem + lanes + L::V, xch, bar, &norm_v);
    tmem_st_wait();
    jxd::fence_proxy_async_smem();  // the areas become copies' destinations
    jxd::tc_fence_before();
    __syncwarp();
    if (lane == 0) jxd::mbar_arrive(stayfull);
    const float f_row = inverse_of(e_k) * (fabsf(s.scale) * LOG2E), inv_v = inverse_of(e_v);
    const int first = row < rows ? sq.first_row(j0 + row, s.causal) : 0x7fffffff;  // first query row that sees this key
    const int first_all = sq.first_row(j0 + rows - 1, s.causal);

    float ak[DP / 2], av[DP / 2];
#pragma unroll
    for (int c = 0; c < DP / 2; ++c) ak[c] = av[c] = 0.0f;
    float g_prev = 0.0f;
    bool ok = true;
    auto ready = [&](uint64_t* b8, int u) {
      ok = ok && warp_wait(b8, (uint32_t)u & 1u, abort_flag, s.err);
      jxd::tc_fence_after();
    };
    auto done = [&](uint64_t* b8) {
      jxd::tc_fence_before();
      __syncwarp();
      if (lane == 0) jxd::mbar_arrive(b8);
    };
    constexpr int C = BLK / 2;  // columns of the scores that this thread has
    for (int u = 0; u < n; ++u) {
      const int g = (it0 + u) / nblk, blk = blk0 + (it0 + u) % nblk, st = u % ST;
      const long long slot = qslot0 + (long long)(blk / PER_TILE) * s.heads + g;
      const float inv_q = bt.inv_q[slot], inv_d = bt.inv_d[slot], norm_d = bt.norm_d[slot], top_d = bt.delta_top[slot];
      const float* lse2 = stats + st * 2 * BLK + half * C;
      const float* delta = lse2 + BLK;
      ready(&qfull[st], u / ST);  // landed before the scores were issued: its statistics are visible here too
      ready(sfull, u);
      const float f = f_row * inv_q;
      const float2 f2 = make_float2(f, f);
      const bool edge = blk * BLK < first_all || rows < TILE;  // some key is not seen by all of the block's rows
      float2 p[C / 2];
#pragma unroll
      for (int c = 0; c < C; c += 32) {
        uint32_t r[32];
        jxd::tmem_ld32(tmem + lanes + L::X + half * C + c, r);
        jxd::tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const float4 l = *reinterpret_cast<const float4*>(lse2 + c + i);
          const float2 z0 = fma2(make_float2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), f2,
                                 make_float2(-l.x, -l.y));
          const float2 z1 = fma2(make_float2(__uint_as_float(r[i + 2]), __uint_as_float(r[i + 3])), f2,
                                 make_float2(-l.z, -l.w));
          p[(c + i) / 2] = make_float2(exp2_fast(z0.x), exp2_fast(z0.y));
          p[(c + i) / 2 + 1] = make_float2(exp2_fast(z1.x), exp2_fast(z1.y));
        }
      }
      if (edge) {
        const int i0 = blk * BLK + half * C;
#pragma unroll
        for (int i = 0; i < C / 2; ++i) {
          if (i0 + 2 * i < first) p[i].x = 0.0f;
          if (i0 + 2 * i + 1 < first) p[i].y = 0.0f;
        }
      }
#pragma unroll
      for (int c = 0; c < C; c += 32) {
        uint32_t hi[16], lo[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) split_half(p[c / 2 + i].x, p[c / 2 + i].y, hi[i], lo[i]);
        tmem_st16(tmem + lanes + L::X + half * C + c, hi);
        tmem_st16(tmem + lanes + L::X + half * C + c + 16, lo);
      }
      tmem_st_wait();
      done(pfull);
      if (u > 0) {
        ready(wfull, u - 1);
        drain<DP>(ak, tmem + lanes + L::W + half * (DP / 2), g_prev);
        done(wfree);
      }
      // P is at most 2^14
      const float fd = inv_v * inv_d, sc = bound_scale(16384.0f * (norm_v * norm_d + top_d));
      const float pf = sc * fd, nf = -inverse_pow2(fd);
      const float2 pf2 = make_float2(pf, pf), nf2 = make_float2(nf, nf);
      ready(dpfull, u);
#pragma unroll
      for (int c = 0; c < C; c += 32) {
        uint32_t r[32], hi[16], lo[16];
        jxd::tmem_ld32(tmem + lanes + L::Y + half * C + c, r);
        jxd::tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const float4 d = *reinterpret_cast<const float4*>(delta + c + i);
          const float2 e0 = fma2(make_float2(d.x, d.y), nf2, make_float2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])));
          const float2 e1 =
              fma2(make_float2(d.z, d.w), nf2, make_float2(__uint_as_float(r[i + 2]), __uint_as_float(r[i + 3])));
          const float2 a0 = mul2(mul2(p[(c + i) / 2], pf2), e0), a1 = mul2(mul2(p[(c + i) / 2 + 1], pf2), e1);
          split_half(a0.x, a0.y, hi[i / 2], lo[i / 2]);
          split_half(a1.x, a1.y, hi[i / 2 + 1], lo[i / 2 + 1]);
        }
        tmem_st16(tmem + lanes + L::Y + half * C + c, hi);
        tmem_st16(tmem + lanes + L::Y + half * C + c + 16, lo);
      }
      tmem_st_wait();
      done(dsfull);
      ready(zfull, u);
      drain<DP>(av, tmem + lanes + L::Z + half * (DP / 2), inv_d * 6.103515625e-05f);  // P's 2^14
      done(zfree);
      g_prev = inv_q * inverse_pow2(sc) * 6.103515625e-05f;
    }
    if (n > 0) {
      ready(wfull, n - 1);
      drain<DP>(ak, tmem + lanes + L::W + half * (DP / 2), g_prev);
    }
    // every MMA has retired: the stages are free
    const int tid = threadIdx.x - 32 * BW_FIRST;
    half_to_area<DP>(smem, ak, s.scale, row, half);
    half_to_area<DP>(smem + ST * STAGE, av, 1.0f, row, half);
    movers_sync();
    rows_store<DP>(out_k + (sq.k0 + j0) * ld_k + kd, ld_k, smem, rows, s.dim, aligned16(out_k, s.dim, ld_k), tid);
    rows_store<DP>(out_v + (sq.k0 + j0) * ld_v + kd, ld_v, smem + ST * STAGE, rows, s.dim,
                   aligned16(out_v, s.dim, ld_v), tid);
  }
  jxd::tc_fence_before();
  __syncthreads();
  jxd::tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    jxd::tmem_dealloc(tmem, 512);
  }
}

// The parts' sums in order, 16 key rows of one key head per block.
constexpr int JOIN_ROWS = 16;
template <bool VEC>
__global__ void __launch_bounds__(256) attn_dkv_join_kernel(const __grid_constant__ Shape s,
                                                           const __grid_constant__ BwdTiles bt, float* dk, float* dv) {
  int jt;
  const int b = seq_of_tile(s.cu_k, s.batch, blockIdx.x / (TILE / JOIN_ROWS), &jt);
  const Seq sq = seq_bounds(s, b);
  const long long j0 = (long long)jt * TILE + blockIdx.x % (TILE / JOIN_ROWS) * JOIN_ROWS;
  if (jt < 0 || j0 >= sq.lk) return;
  const int rows = (int)min((long long)JOIN_ROWS, sq.lk - j0);
  const long long t0 = sq.k0 + j0, hd = (long long)blockIdx.y * s.dim;
  const long long ld = (long long)s.kv_heads * s.dim, all = s.total_k * ld;
  constexpr int V = VEC ? 4 : 1;
  const int cols = s.dim / V, half = rows * cols;  // the rows of dk, then those of dv
  for (int e = threadIdx.x; e < 2 * half; e += 256) {
    const bool is_v = e >= half;
    const int f = is_v ? e - half : e, r = f / cols, c = (f - r * cols) * V;
    const float* p = (is_v ? bt.part_v : bt.part_k) + (t0 + r) * ld + hd + c;
    float* out = (is_v ? dv + (t0 + r) * s.ldv : dk + (t0 + r) * s.ldk) + hd + c;
    if constexpr (VEC) {
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int i = 0; i < bt.parts; ++i) {
        const float4 x = *reinterpret_cast<const float4*>(p + i * all);
        a.x += x.x;
        a.y += x.y;
        a.z += x.z;
        a.w += x.w;
      }
      *reinterpret_cast<float4*>(out) = a;
    } else {
      float a = 0.0f;
#pragma unroll 4
      for (int i = 0; i < bt.parts; ++i) a += p[i * all];
      *out = a;
    }
  }
}

template <int DP>
int launch(const Shape& s, const BwdTiles& bt, const float* q, const float* k, const float* v, const float* o,
           const float* lse, const float* dout, float* dq, float* dk, float* dv, cudaStream_t st) {
  if (int rc = prepare_kernel((const void*)attn_dq_kernel<DP>, DP == 128 ? 2 : 3, dq_smem(DP), BW_LAUNCH_REGS))
    return rc;
  if (int rc = prepare_kernel((const void*)attn_dkv_kernel<DP>, DP == 128 ? 4 : 5, kv_smem(DP), BW_LAUNCH_REGS))
    return rc;
  attn_dq_kernel<DP><<<(unsigned)((long long)bt.q_tiles * s.heads), BW_THREADS, dq_smem(DP), st>>>(
      s, bt, q, k, v, o, lse, dout, dq);
  attn_dkv_kernel<DP><<<(unsigned)((long long)bt.k_tiles * s.kv_heads * bt.parts), BW_THREADS, kv_smem(DP), st>>>(
      s, bt, q, k, v, o, lse, dout, dk, dv);
  if (bt.parts > 1) {
    const dim3 grid((unsigned)(bt.k_tiles * (TILE / JOIN_ROWS)), (unsigned)s.kv_heads);
    const bool vec = !(s.dim & 3) && !(s.ldk & 3) && !(s.ldv & 3) &&
                     !((reinterpret_cast<uintptr_t>(dk) | reinterpret_cast<uintptr_t>(dv)) & 15);
    if (vec) attn_dkv_join_kernel<true><<<grid, 256, 0, st>>>(s, bt, dk, dv);
    else attn_dkv_join_kernel<false><<<grid, 256, 0, st>>>(s, bt, dk, dv);
  }
  JX_LAUNCH_CHECK("attention_bwd kernels");
  return JX_OK;
}

}  // namespace

namespace jxa {

int attention_bwd_tiles(const Shape& s, const float* q, const float* k, const float* v, const float* o,
                        const float* lse, const float* dout, float* dq, float* dk, float* dv, cudaStream_t st) {
  const int DP = s.dim <= 64 ? 64 : 128;
  const long long kt = tile_count(s.total_k, s.batch), qt = tile_count(s.total_q, s.batch);
  // key tiles are few where heads are shared: enough parts of the query rows for four CTAs per SM
  const long long ctas = kt * s.kv_heads;
  const int parts = (int)std::max<long long>(1, std::min<long long>(8, 4LL * jx::num_sms() / std::max(1LL, ctas)));
  JX_REQUIRE(qt * s.heads < (1LL << 31) && kt * s.kv_heads * parts < (1LL << 31) && kt < (1LL << 27),
             "attention_bwd: too many rows");
  const size_t ks = (size_t)kt * s.kv_heads, qs = (size_t)qt * s.heads, tb = tile_bytes(DP);
  const size_t part_floats = parts > 1 ? (size_t)parts * s.total_k * s.kv_heads * s.dim : 0;
  // tiles first, then arrays whose pieces the copies read 16-byte aligned, then the rest
  const size_t bytes = (2 * ks + 2 * qs) * tb + 2 * qs * TILE * 4 + (5 * ks + 6 * qs + qt + kt) * 4 + 2 * part_floats * 4;
  void* p = nullptr;
  if (int rc = jx::scratch_get(bytes + 64, &p, st)) return rc;
  uint8_t* at = static_cast<uint8_t*>(p);
  auto take = [&](size_t n) {
    uint8_t* r = at;
    at += n;
    return r;
  };
  uint8_t *tk = take(ks * tb), *tv = take(ks * tb), *tq = take(qs * tb), *td = take(qs * tb);
  float* lse2 = (float*)take(qs * TILE * 4);
  float* delta = (float*)take(qs * TILE * 4);
  float* part_k = (float*)take(part_floats * 4);
  float* part_v = (float*)take(part_floats * 4);
  float *inv_k = (float*)take(ks * 4), *inv_v = (float*)take(ks * 4), *norm_v = (float*)take(ks * 4);
  float *inv_q = (float*)take(qs * 4), *inv_d = (float*)take(qs * 4), *norm_d = (float*)take(qs * 4);
  float* delta_top = (float*)take(qs * 4);
  int *bad_k = (int*)take(ks * 4), *bad_v = (int*)take(ks * 4), *bad_q = (int*)take(qs * 4), *bad_d = (int*)take(qs * 4);
  int *order_q = (int*)take(qt * 4), *order_k = (int*)take(kt * 4);
  TileSources kv = {}, qd = {};
  kv.t[0] = {k, s.ldk, tk, inv_k, bad_k};
  kv.t[1] = {v, s.ldv, tv, inv_v, bad_v, norm_v};
  qd.t[0] = {q, s.ldq, tq, inv_q, bad_q};
  qd.t[1] = {dout, s.ldo, td, inv_d, bad_d, norm_d, o, lse, lse2, delta, delta_top};
  const BwdTiles bt = {tq,     tk,     tv,    td,    inv_q, inv_k,     inv_v,   inv_d,   bad_q, bad_k,  bad_v,
                       bad_d,  norm_v, norm_d, lse2, delta, delta_top, (int)qt, (int)kt, parts, order_q, order_k, part_k, part_v};
  kv.order = order_k;
  kv.order_other = order_q;
  int rc = split_tiles(s, false, kv, 2, s.kv_heads, DP, st);
  if (!rc) rc = split_tiles(s, true, qd, 2, s.heads, DP, st);
  if (!rc)
    rc = DP == 128 ? launch<128>(s, bt, q, k, v, o, lse, dout, dq, dk, dv, st)
                   : launch<64>(s, bt, q, k, v, o, lse, dout, dq, dk, dv, st);
  jx::scratch_release(p, st);
  return rc;
}

}  // namespace jxa
