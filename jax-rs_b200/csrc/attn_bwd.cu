// attn_bwd.cu -- attention's gradients on the tensor cores (operands and sums as
// in attn_tc.cuh).
//
// Two kinds of CTAs, each with its sums in registers, so that every sum has a fixed
// order and nothing is added atomically; the price is that the scores and
// dout v^T are computed in both (seven products a tile instead of five).  All
// four operands are split into tiles once, and each kind streams two of them.
//
// dq: one CTA per (128 query rows, head), streaming K and V tiles.
//   S = Q K^T, dP = dO V^T,  dS = P (dP - delta),  dQ += dS K
// dk, dv: one CTA per (128 keys, key head, part of the query rows), streaming
// blocks of Q and dO of every head of the group.
//   S^T = K Q^T, dP^T = V dO^T,  dV += P^T dO, dK += dS^T Q
// with P = exp2(S f - lse2), computed operands in tensor memory.
//
// The products of a step wait for each other through the registers (S -> P -> dV,
// dP -> dS -> dK), 900 to 1800 cycles each way, so scores are issued a step
// ahead where tensor memory has the room; the layouts below say where that is.
// An MMA of 64 columns takes 44 to 48 cycles, not the 32 that half of one of 128 is, so
// that a tile's seven products of three parts each take 2600 (dq) and 3650 cycles (dk and dv) at dim 64;
// the steps take 3200 and 5000, the mean of 16 with the first one's latencies.  What stands between two products on the MMA thread's
// way counts in full: its waits look at the barrier and at nothing else (an abort
// flag read there cost 3% to 10% of the whole).
//
// 4096 packed tokens in 5 sequences, 16 heads, dim 64, causal: 195 us (178 to 185 in a
// captured graph on a cool GPU), of which the split 31 and the products 159; each of the four
// CTAs in a row on an SM spends 4.6 us on its start, its first tiles' latency and its
// stores.  4096 tokens, 16 heads on 4, dim 128: 690 to 710 us with the power limit's clock.
//
// A computed operand needs its scale before its largest value is known: P <= 1
// and |dP - delta| <= |dout row| |v row| + |delta| (norms) bound dS.  The norms
// are the row's own for dq, and for dk and dv the largest among the block's rows
// that see the key: rows of dout may differ in size, and one scale for all would
// leave small ones few bits.  The bound overestimates by log2 of the keys that
// share a row's weight and some bits more, of the 28 that there are above the
// last value with 22 bits.
#include <algorithm>

#include "attn_tc.cuh"

namespace {

using namespace jxa;

constexpr int BW_THREADS = 384;  // warp 0 copies, warp 1 MMA, warps 4..11 the rest
constexpr int BW_FIRST = 4;
constexpr int BW_LAUNCH_REGS = 168;
constexpr int BW_LOW_REGS = 56;
constexpr int BW_HIGH_REGS = 216;
static_assert(128 * BW_LOW_REGS + 256 * BW_HIGH_REGS <= BW_THREADS * BW_LAUNCH_REGS,
              "register split exceeds the launch allocation");

struct BwdTiles {
  const uint8_t *q, *k, *v, *d;  // tiles; d is dout
  const float4* num_q;  // of a tile of query rows: what undoes Q's scale and dout's, dout's largest row norm
  const float4* num_k;  // of a tile of keys: what undoes K's scale and V's, V's largest row norm
  const int *bad_q, *bad_k, *bad_v, *bad_d;
  const float *lse2, *delta, *row_norm;
  const float2* later;
  int q_tiles, k_tiles, parts;
  const TileRef *order_q, *order_k;
  float *part_k, *part_v;  // [parts][total_k * kv_heads * dim], used where parts > 1
};

// 1 / f of a power of two.
__device__ __forceinline__ float inverse_pow2(float f) { return __uint_as_float((254u << 23) - __float_as_uint(f)); }

// Scale for a computed operand of magnitude <= bound, at most 2^100.
__device__ __forceinline__ float bound_scale(float bound) {
  const int e = (int)(__float_as_uint(bound) >> 23);
  return __uint_as_float((uint32_t)(268 - min(max(e, 41), 254)) << 23);
}
// A row's norm is taken as this part of its tile's at least, so that the scale of an
// all but empty row stays finite: rows of less than 2^-20 are zeros (or the tile is marked).
constexpr float LEAST_NORM = 1.4901161e-08f;  // 2^-26
// Scale of dS over that of dP: below 2^40 but for a bound of zero, whose dS is zero under any finite one.
__device__ __forceinline__ float scale_ratio(float sc, float fd) { return fminf(sc * fd, 1.2676506e+30f); }  // 2^100

// acc += part * factor for this thread's DP/2 columns of a tensor-memory sum.
template <int DP>
__device__ __forceinline__ void drain(float (&acc)[DP / 2], uint32_t taddr, float factor) {
  const float2 f2 = make_float2(factor, factor);
#pragma unroll
  for (int c = 0; c < DP / 2; c += 32) {
    uint32_t r[32];
    jxd::tmem_ld32(taddr + c, r);
    jxd::tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      const float2 v = fma2(make_float2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), f2,
                            make_float2(acc[c + i], acc[c + i + 1]));
      acc[c + i] = v.x;
      acc[c + i + 1] = v.y;
    }
  }
}

// A tile from shared memory into tensor memory: hi in DP/2 columns, lo in the next
// DP/2; this thread has half of row `row`.
template <int DP>
__device__ __forceinline__ void tile_to_tmem(const uint8_t* tile, int row, int half, uint32_t taddr) {
  constexpr int CHUNKS = DP / 16;  // of 16 bytes, per half row
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    const uint8_t* p = tile + part * tile_part(DP) + (DP == 128 ? half * PANEL : 0) + row * 128;
    uint32_t r[4 * CHUNKS];
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      const int c = DP == 128 ? i : half * CHUNKS + i;
      const uint4 x = *reinterpret_cast<const uint4*>(p + ((c ^ (row & 7)) << 4));
      r[4 * i] = x.x;
      r[4 * i + 1] = x.y;
      r[4 * i + 2] = x.z;
      r[4 * i + 3] = x.w;
    }
    const uint32_t to = taddr + part * (DP / 2) + half * (DP / 4);
    if constexpr (DP == 128) tmem_st32(to, r);
    else tmem_st16(to, r);
  }
}

// Scores: D[128 x N] = A B^T over DP columns, small parts first.  A's tile lies in
// tensor memory at `a` (TS), or in shared memory at `a`; B's has `panel` bytes a
// panel and `part` a part.
template <int DP, int N, bool TS>
__device__ __forceinline__ void mma_scores(uint32_t d, uint32_t a, uint32_t b, uint32_t panel, uint32_t part) {
  constexpr uint32_t id = idesc_f16(N, false);
  auto step = [&](int ks, bool a_lo, bool b_lo, uint32_t acc) {
    const uint64_t bd = jxd::smem_desc_k_sw128(b + (b_lo ? part : 0) + (ks >> 2) * panel + (ks & 3) * 32);
    const bool shrink = !a_lo && !b_lo && ks == 0;
    if constexpr (TS) {
      const uint32_t ad = a + (a_lo ? DP / 2 : 0) + ks * 8;
      if (shrink) mma_f16_ts_shrink(d, ad, bd, id);
      else mma_f16_ts(d, ad, bd, id, acc);
    } else {
      const uint64_t ad = jxd::smem_desc_k_sw128(a + (a_lo ? tile_part(DP) : 0) + (ks >> 2) * PANEL + (ks & 3) * 32);
      if (shrink) mma_f16_ss_shrink(d, ad, bd, id);
      else mma_f16_ss(d, ad, bd, id, acc);
    }
  };
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks) {
    step(ks, true, false, ks > 0);
    step(ks, false, true, 1);
  }
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks) step(ks, false, false, 1);
}

// Sums: D[128 x DP] = A B over ROWS rows of B; A in tensor memory, 16 columns of
// hi and 16 of lo for every 32 rows.
template <int DP, int ROWS>
__device__ __forceinline__ void mma_sums(uint32_t d, uint32_t a, uint32_t b, uint32_t panel, uint32_t part) {
  constexpr uint32_t id = idesc_f16(DP, true);
  auto step = [&](int ks, bool a_lo, bool b_lo, uint32_t acc) {
    const uint32_t ad = a + (ks >> 1) * 32 + (ks & 1) * 8 + (a_lo ? 16 : 0);
    const uint64_t bd = smem_desc_mn_sw128(b + (b_lo ? part : 0) + ks * 2048, panel);
    if (!a_lo && !b_lo && ks == 0) mma_f16_ts_shrink(d, ad, bd, id);
    else mma_f16_ts(d, ad, bd, id, acc);
  };
#pragma unroll
  for (int ks = 0; ks < ROWS / 16; ++ks) {
    step(ks, true, false, ks > 0);
    step(ks, false, true, 1);
  }
#pragma unroll
  for (int ks = 0; ks < ROWS / 16; ++ks) step(ks, false, false, 1);
}

// ---- dq ------------------------------------------------------------------------
// Tensor memory at DP = 128: Q and dO (from shared memory they would not leave room
// for K and V), X for S, then dS, and Y for dP, then the sum's part D: S(j+1)
// follows dS(j) K.  At DP = 64 Q stays in shared memory, S alternates between two
// X, dS goes over its S and D has its own columns: S runs two tiles ahead and dP
// one.
template <int DP>
struct DqLayout {
  static constexpr bool AHEAD = DP == 64;
  static constexpr int KS = AHEAD ? 4 : 2, VS = AHEAD ? 2 : 1;  // stages
  static constexpr uint32_t Q = 0, DO = AHEAD ? 448 : 128;      // (Q: DP = 128)
  static constexpr uint32_t X = AHEAD ? 0 : 256, X_STEP = AHEAD ? 128 : 0, Y = AHEAD ? 256 : 384, D = 384;
  static constexpr int STAY = AHEAD ? tile_bytes(DP) : 0;       // shared memory for Q
  static constexpr size_t SMEM = STAY + (size_t)(KS + VS) * tile_bytes(DP) + 1024 + 256;
};

template <int DP>
__device__ __forceinline__ void dq_tile(const Shape& s, const BwdTiles& bt, uint8_t* smem_raw, unsigned w,
                                        const float* __restrict__ q, const float* __restrict__ k,
                                        const float* __restrict__ v, const float* __restrict__ o,
                                        const float* __restrict__ lse, const float* __restrict__ dout, float* dq) {
  using L = DqLayout<DP>;
  constexpr int KS = L::KS, VS = L::VS, STAGE = tile_bytes(DP), PART = tile_part(DP);
  const uint32_t raw_addr = jxd::smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
  uint8_t* ring = smem + L::STAY;  // K's stages, then V's
  uint64_t* kfull = reinterpret_cast<uint64_t*>(ring + (KS + VS) * STAGE);
  uint64_t* kempty = kfull + KS;
  uint64_t* vfull = kempty + KS;
  uint64_t* vempty = vfull + VS;
  uint64_t* stayfull = vempty + VS;  // Q's and dO's tiles have landed
  uint64_t* moved = stayfull + 1;    // and those that go there are in tensor memory
  uint64_t* sfull = moved + 1;       // [2]
  uint64_t* dpfull = sfull + 2;
  uint64_t* dsfull = dpfull + 1;
  uint64_t* dqfull = dsfull + 1;
  uint64_t* dfree = dqfull + 1;  // D is drained
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(dfree + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const TileRef ref = load_ref(bt.order_q + w / (unsigned)s.heads);
  const int h = (int)(w % (unsigned)s.heads), b = ref.b, jt = ref.jt;
  const Seq sq = seq_of(ref);
  if (jt < 0) return;
  const int i0 = jt * TILE, rows = min(TILE, sq.lq - i0);
  const int hk = h / s.group;
  const int nb = (sq.visible(i0 + rows - 1, s.causal) + TILE - 1) / TILE;
  const long long slot0 = (long long)first_tile(sq.k0, b) * s.kv_heads + hk;
  const long long qslot = ((long long)first_tile(sq.q0, b) + jt) * s.heads + h;
  const long long hd = (long long)h * s.dim;

  // dO passes through V's last stage, Q (at DP = 128) through K's
  uint8_t* at_q = L::AHEAD ? smem : ring + (KS - 1) * STAGE;
  uint8_t* at_d = ring + (KS + VS - 1) * STAGE;
  constexpr int K_FIRST = L::AHEAD ? KS : KS - 1, V_FIRST = VS - 1;  // stages that are free at once
  auto copy_k = [&](int j) {
    jxd::mbar_arrive_expect_tx(&kfull[j % KS], STAGE);
    bulk_load(jxd::smem_u32(ring + j % KS * STAGE), bt.k + (slot0 + (long long)j * s.kv_heads) * STAGE, STAGE,
              &kfull[j % KS]);
  };
  auto copy_v = [&](int j) {
    jxd::mbar_arrive_expect_tx(&vfull[j % VS], STAGE);
    bulk_load(jxd::smem_u32(ring + (KS + j % VS) * STAGE), bt.v + (slot0 + (long long)j * s.kv_heads) * STAGE, STAGE,
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
    jxd::mbar_init(stayfull, 1);
    jxd::mbar_init(moved, 8);
    jxd::mbar_init(&sfull[0], 1);
    jxd::mbar_init(&sfull[1], 1);
    jxd::mbar_init(dpfull, 1);
    jxd::mbar_init(dsfull, 8);
    jxd::mbar_init(dqfull, 1);
    jxd::mbar_init(dfree, 8);
    *abort_flag = 0;
    jxd::fence_mbar_init();
    jxd::fence_proxy_async_smem();
    if (nb > 0) {
      jxd::mbar_arrive_expect_tx(stayfull, 2 * STAGE);
      bulk_load(jxd::smem_u32(at_q), bt.q + qslot * STAGE, STAGE, stayfull);
      copy_k(0);
      bulk_load(jxd::smem_u32(at_d), bt.d + qslot * STAGE, STAGE, stayfull);
      for (int j = 1; j < min(nb, K_FIRST); ++j) copy_k(j);
      for (int j = 0; j < min(nb, V_FIRST); ++j) copy_v(j);
    }
  } else if (warp == 1) {
    jxd::tmem_alloc(tmem_slot, 512);
    jxd::tmem_relinquish();
  } else if (warp >= 2) {
    if (threadIdx.x == 64) bad = bt.bad_q[qslot] || bt.bad_d[qslot];
    for (int j = (int)threadIdx.x - 64; j < nb; j += BW_THREADS - 64)
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
    if (warp == 0 && lane == 0 && nb > 0) {  // the copies have landed
      unsigned long long end = 0;  // for all of them
      wait_suspended(stayfull, 0, s.err, end);
      for (int j = 0; j < min(nb, K_FIRST); ++j) wait_suspended(&kfull[j], 0, s.err, end);
      for (int j = 0; j < min(nb, V_FIRST); ++j) wait_suspended(&vfull[j], 0, s.err, end);
    }
    if (warp == 1) {
      __syncwarp();
      jxd::tmem_dealloc(tmem, 512);
    }
    return;
  }

  if (warp < BW_FIRST) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(BW_LOW_REGS));
    if (warp == 0 && nb > 0 && jxd::elect_one()) {
      // ---- the remaining copies
      int nk = min(nb, K_FIRST), nv = min(nb, V_FIRST);
      bool ok = wait_suspended(moved, 0, s.err);  // the stages that Q and dO passed through are free
      auto free_stage = [&](uint64_t* bar, int use) {
        return ok = ok && !*abort_flag && wait_suspended(bar, (uint32_t)(use + 1) & 1u, s.err);
      };
      while (ok && (nk < nb || nv < nb)) {
        if (nv < nb && nv < nk) {
          if (!free_stage(&vempty[nv % VS], nv / VS)) break;
          copy_v(nv++);
        } else {
          if (!free_stage(&kempty[nk % KS], nk / KS)) break;
          copy_k(nk++);
        }
      }
      if (!ok) *abort_flag = 1;
      // every copy has landed before the CTA may end
      unsigned long long end = 0;  // for all of them
      wait_suspended(stayfull, 0, s.err, end);
      for (int u = max(0, nk - KS); u < nk; ++u) wait_suspended(&kfull[u % KS], (uint32_t)(u / KS) & 1u, s.err, end);
      for (int u = max(0, nv - VS); u < nv; ++u) wait_suspended(&vfull[u % VS], (uint32_t)(u / VS) & 1u, s.err, end);
    }
    if (warp == 1 && nb > 0 && jxd::elect_one()) {
      // ---- MMA (its waits stand between products: nothing is looked at there but the barrier)
      const uint32_t kbase = jxd::smem_u32(ring), vbase = kbase + KS * STAGE;
      bool ok = wait_polling(stayfull, 0, s.err);
      auto ready = [&](uint64_t* bar, int n) {
        ok = ok && wait_polling(bar, (uint32_t)n & 1u, s.err);
        jxd::tc_fence_after();
        return ok;
      };
      auto q_scores = [&](int j) {
        if (!ready(&kfull[j % KS], j / KS)) return;
        mma_scores<DP, 128, !L::AHEAD>(tmem + L::X + (j & 1) * L::X_STEP, L::AHEAD ? jxd::smem_u32(at_q) : tmem + L::Q,
                                       kbase + (j % KS) * STAGE, PANEL, PART);
        jxd::mma_commit(&sfull[j & 1]);
      };
      auto d_scores = [&](int j) {
        if (!ready(&vfull[j % VS], j / VS)) return;
        mma_scores<DP, 128, true>(tmem + L::Y, tmem + L::DO, vbase + (j % VS) * STAGE, PANEL, PART);
        jxd::mma_commit(dpfull);
        jxd::mma_commit(&vempty[j % VS]);
      };
      if (!L::AHEAD) ready(moved, 0);
      if (ok) q_scores(0);
      if (L::AHEAD && ok && nb > 1) q_scores(1);
      if (L::AHEAD) ready(moved, 0);
      if (ok) d_scores(0);
      for (int j = 0; ok && j < nb; ++j) {
        if (!ready(dsfull, j)) break;
        if (L::AHEAD && j + 1 < nb) d_scores(j + 1);    // Y is read
        if (L::AHEAD && !ready(dfree, j + 1)) break;
        mma_sums<DP, 128>(tmem + L::D, tmem + L::X + (j & 1) * L::X_STEP, kbase + (j % KS) * STAGE, PANEL, PART);
        jxd::mma_commit(dqfull);
        jxd::mma_commit(&kempty[j % KS]);
        if (L::AHEAD) {
          if (j + 2 < nb) q_scores(j + 2);
        } else if (j + 1 < nb) {
          q_scores(j + 1);
          if (!ready(dfree, j)) break;  // D is Y
          d_scores(j + 1);
        }
      }
      if (!ok) *abort_flag = 1;
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(BW_HIGH_REGS));
    const int quarter = warp & 3, half = (warp - BW_FIRST) >> 2, row = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    bool ok = true;
    auto ready = [&](uint64_t* bar, int n) {
      warp_wait(bar, (uint32_t)n & 1u, ok, abort_flag, s.err);
      jxd::tc_fence_after();
    };
    auto done = [&](uint64_t* bar) {
      jxd::tc_fence_before();
      __syncwarp();
      if (lane == 0) jxd::mbar_arrive(bar);
    };
    if (nb > 0) {
      ready(stayfull, 0);
      if constexpr (!L::AHEAD) tile_to_tmem<DP>(at_q, row, half, tmem + lanes + L::Q);
      tile_to_tmem<DP>(at_d, row, half, tmem + lanes + L::DO);
      tmem_st_wait();
      done(moved);
    }
    const float4 num = bt.num_q[qslot];
    const float f_tile = num.x * (s.scale * LOG2E), inv_d = num.y;
    const float norm_d = fmaxf(bt.row_norm[qslot * TILE + row], num.z * LEAST_NORM);
    const float lse2 = bt.lse2[qslot * TILE + row], delta = bt.delta[qslot * TILE + row];
    const int vis = row < rows ? sq.visible(i0 + row, s.causal) : 0;
    const int vis_all = sq.visible(i0, s.causal);

    float acc[DP / 2];
#pragma unroll
    for (int c = 0; c < DP / 2; ++c) acc[c] = 0.0f;
    float g_prev = 0.0f;
    float2 p[32];
    // P of tile j, scaled for dS, and what undoes dS's scale; the next tile's numbers are loaded a tile ahead
    float dl = 0.0f, g = 0.0f;
    const float4* num_k = bt.num_k + slot0;
    float4 next = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (nb > 0) next = *num_k;
    auto weights = [&](int j) {
      const float inv_k = next.x, inv_v = next.y, norm_v = next.z;
      if (j + 1 < nb) next = *(num_k += s.kv_heads);
      // P is at most 2^14
      const float fd = inv_d * inv_v, sc = bound_scale(16384.0f * (norm_d * norm_v + fabsf(delta)));
      const float f = f_tile * inv_k, pf = scale_ratio(sc, fd);
      dl = -delta * inverse_pow2(fd);
      g = inv_k * inverse_pow2(sc) * 6.103515625e-05f;  // P's 2^14
      const float2 f2 = make_float2(f, f), l2 = make_float2(-lse2, -lse2), pf2 = make_float2(pf, pf);
      ready(&sfull[j & 1], j >> 1);
#pragma unroll
      for (int c = 0; c < 64; c += 32) {
        uint32_t r[32];
        jxd::tmem_ld32(tmem + lanes + L::X + (j & 1) * L::X_STEP + half * 64 + c, r);
        jxd::tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          const float2 z = fma2(make_float2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), f2, l2);
          p[(c + i) / 2] = make_float2(exp2_fast(z.x), exp2_fast(z.y));
        }
      }
      if (j * TILE + TILE > vis_all) {  // some row does not see all of the tile's keys
        const int key0 = j * TILE + half * 64;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          if (key0 + 2 * i >= vis) p[i].x = 0.0f;
          if (key0 + 2 * i + 1 >= vis) p[i].y = 0.0f;
        }
      }
#pragma unroll
      for (int i = 0; i < 32; ++i) p[i] = mul2(p[i], pf2);
    };
    auto add_part = [&](int j) {
      ready(dqfull, j);
      drain<DP>(acc, tmem + lanes + L::D + half * (DP / 2), g_prev);
      done(dfree);
    };
    if (L::AHEAD && nb > 0) weights(0);
    for (int j = 0; j < nb; ++j) {
      if (!L::AHEAD) {
        if (j > 0) add_part(j - 1);
        weights(j);
      }
      ready(dpfull, j);
      const float2 one2 = make_float2(1.0f, 1.0f), dl2 = make_float2(dl, dl);
      const uint32_t ds = tmem + lanes + L::X + (j & 1) * L::X_STEP + half * 64;
#pragma unroll
      for (int c = 0; c < 64; c += 32) {
        uint32_t r[32], hi[16], lo[16];
        jxd::tmem_ld32(tmem + lanes + L::Y + half * 64 + c, r);
        jxd::tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float2 e = fma2(make_float2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), one2, dl2);
          const float2 x = mul2(p[c / 2 + i], e);
          split_half(x.x, x.y, hi[i], lo[i]);
        }
        tmem_st16(ds + c, hi);
        tmem_st16(ds + c + 16, lo);
      }
      tmem_st_wait();
      done(dsfull);
      if (L::AHEAD) {
        if (j > 0) add_part(j - 1);
        g_prev = g;
        if (j + 1 < nb) weights(j + 1);
      } else {
        g_prev = g;
      }
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
// DP = 64: blocks of 128 query rows, K and V in shared memory; two X for S^T, Y
// for dP^T (dS^T over it), the parts of dV and dK in Z and W:
//   S(u+1), dV(u), dK(u), dP(u+1)
// DP = 128: blocks of 64 rows, K in shared memory, V in tensor memory; two X, two
// Y, and Z for both sums' parts, each drained while the scores after it run:
//   dV(u), dP(u+1), dK(u), S(u+2)
// (An MMA of 64 columns takes 45 cycles where half of one of 128 would be 32, which
// is what the block of 64 rows costs.)
template <int DP>
struct KvLayout {
  static constexpr bool APART = DP == 64;
  static constexpr int BLK = kv_block(DP);
  static constexpr int QS = 3, DS = 2;  // stages of Q and of dout
  static constexpr uint32_t V = 0;      // DP = 128
  static constexpr uint32_t X = APART ? 0 : 128, X_STEP = BLK, Y = 256, Y_STEP = APART ? 0 : BLK;
  static constexpr uint32_t Z = 384, W = APART ? 448 : 384;
  static constexpr int PANEL_BYTES = BLK * 128;                                    // of a block
  static constexpr int STAGE = DP / 64 * 2 * PANEL_BYTES;                          // one block: 32 KB
  static constexpr int STAY = APART ? 2 * tile_bytes(DP) : tile_bytes(DP);         // shared memory for K (and V)
  static constexpr int STATS = 2 * BLK + 4;  // floats of a block's lse2, delta and its tile's numbers; two blocks
  // What is left of an SM's 227 KB for aligning the tiles to 1024 bytes.  The array is
  // declared so aligned; a base that were not would be refused.
  static constexpr int SPARE = 768;
  static constexpr size_t SMEM = STAY + (size_t)(QS + DS) * STAGE + 2 * STATS * 4 + 208 + SPARE;
};
static_assert(KvLayout<64>::SMEM <= 232448 && KvLayout<128>::SMEM <= 232448, "shared memory of an SM");

template <int DP>
__device__ __forceinline__ void dkv_tile(const Shape& s, const BwdTiles& bt, uint8_t* smem_raw, unsigned w,
                                         const float* __restrict__ q, const float* __restrict__ k,
                                         const float* __restrict__ v, const float* __restrict__ o,
                                         const float* __restrict__ lse, const float* __restrict__ dout, float* dk,
                                         float* dv) {
  using L = KvLayout<DP>;
  constexpr int QS = L::QS, DS = L::DS, BLK = L::BLK, STAGE = L::STAGE, PART = STAGE / 2, HPANEL = L::PANEL_BYTES;
  constexpr int PER_TILE = TILE / BLK;  // blocks of a tile
  const uint32_t raw_addr = jxd::smem_u32(smem_raw), shift = ((raw_addr + 1023u) & ~1023u) - raw_addr;
  if (shift > (uint32_t)L::SPARE) {
    if (threadIdx.x == 0) atomicOr(s.err, JX_DEVERR_TIMEOUT);
    return;
  }
  uint8_t* smem = smem_raw + shift;
  uint8_t* ring = smem + L::STAY;  // Q's stages, then dout's
  float* stats = reinterpret_cast<float*>(ring + (QS + DS) * STAGE);  // [2][lse2 BLK, delta BLK, numbers 4]
  uint64_t* qfull = reinterpret_cast<uint64_t*>(stats + 2 * L::STATS);
  uint64_t* qempty = qfull + QS;
  uint64_t* dfull = qempty + QS;
  uint64_t* dempty = dfull + DS;
  uint64_t* stayfull = dempty + DS;  // K's and V's tiles have landed
  uint64_t* moved = stayfull + 1;    // V's is in tensor memory (DP = 128)
  uint64_t* sfull = moved + 1;       // [2]
  uint64_t* dpfull = sfull + 2;      // [2]
  uint64_t* pfull = dpfull + 2;
  uint64_t* dsfull = pfull + 1;
  uint64_t* zfull = dsfull + 1;
  uint64_t* zfree = zfull + 1;  // dV's part
  uint64_t* wfull = zfree + 1;  // dK's
  uint64_t* wfree = wfull + 1;
  uint64_t* tfull = wfree + 1;  // [2] statistics
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tfull + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // the keys that the most rows see start first
  const int part = (int)(w % (unsigned)bt.parts);
  w /= (unsigned)bt.parts;
  const TileRef ref = load_ref(bt.order_k + w / (unsigned)s.kv_heads);
  const int hk = (int)(w % (unsigned)s.kv_heads), b = ref.b, jt = ref.jt;
  const Seq sq = seq_of(ref);
  if (jt < 0) return;
  const int j0 = jt * TILE, rows = min(TILE, sq.lk - j0);
  const int blk0 = sq.first_row(j0, s.causal) / BLK;
  const int nblk = max(0, (sq.lq + BLK - 1) / BLK - blk0);
  const long long steps = (long long)s.group * nblk;
  const int it0 = (int)(steps * part / bt.parts), n = (int)(steps * (part + 1) / bt.parts) - it0;
  const long long qslot0 = (long long)first_tile(sq.q0, b) * s.heads + (long long)hk * s.group;
  const long long kslot = ((long long)first_tile(sq.k0, b) + jt) * s.kv_heads + hk;
  const int h0 = hk * s.group;
  const long long kd = (long long)hk * s.dim;
  // where this part's sums go
  float* out_k = bt.parts > 1 ? bt.part_k + (long long)part * s.total_k * s.kv_heads * s.dim : dk;
  float* out_v = bt.parts > 1 ? bt.part_v + (long long)part * s.total_k * s.kv_heads * s.dim : dv;
  const long long ld_k = bt.parts > 1 ? (long long)s.kv_heads * s.dim : s.ldk;
  const long long ld_v = bt.parts > 1 ? (long long)s.kv_heads * s.dim : s.ldv;

  // at DP = 128 V passes through Q's last two stages
  uint8_t* at_v = L::APART ? smem + tile_bytes(DP) : ring + (QS - 2) * STAGE;
  constexpr int Q_FIRST = L::APART ? QS : QS - 2;  // stages that are free at once
  // step u's block, as its tile's slot and its place in the tile
  auto slot_of = [&](int u, int* place) {
    const int g = (it0 + u) / nblk, blk = blk0 + (it0 + u) % nblk;
    *place = blk % PER_TILE;
    return qslot0 + (long long)(blk / PER_TILE) * s.heads + g;
  };
  // a block: its rows of each part's panels
  auto load = [&](uint8_t* dst, const uint8_t* tile, int place, uint64_t* bar) {
    jxd::mbar_arrive_expect_tx(bar, STAGE);
#pragma unroll
    for (int e = 0; e < 2 * (DP / 64); ++e)
      bulk_load(jxd::smem_u32(dst + e * HPANEL), tile + (long long)e * PANEL + place * HPANEL, HPANEL, bar);
  };
  auto copy_q = [&](int u) {
    int place;
    const long long slot = slot_of(u, &place);
    load(ring + u % QS * STAGE, bt.q + slot * tile_bytes(DP), place, &qfull[u % QS]);
  };
  auto copy_d = [&](int u) {
    int place;
    const long long slot = slot_of(u, &place);
    load(ring + (QS + u % DS) * STAGE, bt.d + slot * tile_bytes(DP), place, &dfull[u % DS]);
  };
  auto copy_stats = [&](int u) {
    int place;
    const long long slot = slot_of(u, &place);
    float* dst = stats + (u & 1) * L::STATS;
    jxd::mbar_arrive_expect_tx(&tfull[u & 1], L::STATS * 4);
    bulk_load(jxd::smem_u32(dst), bt.lse2 + slot * TILE + place * BLK, BLK * 4, &tfull[u & 1]);
    bulk_load(jxd::smem_u32(dst + BLK), bt.delta + slot * TILE + place * BLK, BLK * 4, &tfull[u & 1]);
    bulk_load(jxd::smem_u32(dst + 2 * BLK), bt.num_q + slot, 16, &tfull[u & 1]);
  };
  bool bad = false;
  if (warp == 0 && lane == 0) {
    for (int i = 0; i < QS; ++i) {
      jxd::mbar_init(&qfull[i], 1);
      jxd::mbar_init(&qempty[i], 1);
    }
    for (int i = 0; i < DS; ++i) {
      jxd::mbar_init(&dfull[i], 1);
      jxd::mbar_init(&dempty[i], 1);
    }
    jxd::mbar_init(stayfull, 1);
    jxd::mbar_init(moved, 8);
    for (int i = 0; i < 2; ++i) {
      jxd::mbar_init(&sfull[i], 1);
      jxd::mbar_init(&dpfull[i], 1);
      jxd::mbar_init(&tfull[i], 1);
    }
    jxd::mbar_init(pfull, 8);
    jxd::mbar_init(dsfull, 8);
    jxd::mbar_init(zfull, 1);
    jxd::mbar_init(zfree, 8);
    jxd::mbar_init(wfull, 1);
    jxd::mbar_init(wfree, 8);
    *abort_flag = 0;
    jxd::fence_mbar_init();
    jxd::fence_proxy_async_smem();
    if (n > 0) {
      jxd::mbar_arrive_expect_tx(stayfull, 2 * tile_bytes(DP));
      bulk_load(jxd::smem_u32(smem), bt.k + kslot * tile_bytes(DP), tile_bytes(DP), stayfull);
      bulk_load(jxd::smem_u32(at_v), bt.v + kslot * tile_bytes(DP), tile_bytes(DP), stayfull);
      for (int u = 0; u < min(n, Q_FIRST); ++u) copy_q(u);
      for (int u = 0; u < min(n, 2); ++u) copy_stats(u);
      for (int u = 0; u < min(n, DS); ++u) copy_d(u);
    }
  } else if (warp == 1) {
    jxd::tmem_alloc(tmem_slot, 512);
    jxd::tmem_relinquish();
  } else if (warp >= 2) {
    if (threadIdx.x == 64) bad = bt.bad_k[kslot] || bt.bad_v[kslot];
    const int t0 = blk0 / PER_TILE, nt = nblk > 0 ? (sq.lq + TILE - 1) / TILE - t0 : 0;
    for (long long e = (int)threadIdx.x - 64; e < (long long)nt * s.group; e += BW_THREADS - 64) {
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
      unsigned long long end = 0;  // for all of them
      wait_suspended(stayfull, 0, s.err, end);
      for (int u = 0; u < min(n, Q_FIRST); ++u) wait_suspended(&qfull[u], 0, s.err, end);
      for (int u = 0; u < min(n, DS); ++u) wait_suspended(&dfull[u], 0, s.err, end);
      for (int u = 0; u < min(n, 2); ++u) wait_suspended(&tfull[u], 0, s.err, end);
    }
    if (warp == 1) {
      __syncwarp();
      jxd::tmem_dealloc(tmem, 512);
    }
    return;
  }

  if (warp < BW_FIRST) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(BW_LOW_REGS));
    if (warp == 0 && n > 0 && jxd::elect_one()) {
      // ---- the remaining copies
      // Q(0) Q(1) dout(0) statistics(0) Q(2) dout(1) statistics(1) ...: dK(u), which the copies of
      // block u+3 of Q and u+2 of the statistics wait for, needs nothing behind dout(u+1) in this order
      int nq = min(n, Q_FIRST), nd = min(n, DS), nt = min(n, 2);
      bool ok = L::APART || wait_suspended(moved, 0, s.err);  // the stages that V passed through are free
      auto free_stage = [&](uint64_t* bar, int use) {
        return ok = ok && !*abort_flag && wait_suspended(bar, (uint32_t)(use + 1) & 1u, s.err);
      };
      for (int i = 0; ok && i <= n; ++i) {
        if (i == nq && i < n) {
          if (!free_stage(&qempty[i % QS], i / QS)) break;
          copy_q(i);
          ++nq;
        }
        if (i - 1 == nd) {
          if (!free_stage(&dempty[nd % DS], nd / DS)) break;
          copy_d(nd);
          ++nd;
        }
        if (i - 1 == nt) {
          // block nt - 2's statistics were last read for its dS, before dK(nt-2), which freed its stage of Q
          if (!free_stage(&qempty[(nt - 2) % QS], (nt - 2) / QS + 1)) break;
          copy_stats(nt);
          ++nt;
        }
      }
      if (!ok) *abort_flag = 1;
      // every copy has landed before the CTA may end
      unsigned long long end = 0;  // for all of them
      wait_suspended(stayfull, 0, s.err, end);
      for (int e = max(0, nq - QS); e < nq; ++e) wait_suspended(&qfull[e % QS], (uint32_t)(e / QS) & 1u, s.err, end);
      for (int e = max(0, nd - DS); e < nd; ++e) wait_suspended(&dfull[e % DS], (uint32_t)(e / DS) & 1u, s.err, end);
      for (int e = max(0, nt - 2); e < nt; ++e) wait_suspended(&tfull[e & 1], (uint32_t)(e >> 1) & 1u, s.err, end);
    }
    if (warp == 1 && n > 0 && jxd::elect_one()) {
      // ---- MMA
      const uint32_t qbase = jxd::smem_u32(ring), dbase = qbase + QS * STAGE;
      bool ok = wait_suspended(stayfull, 0, s.err) && (L::APART || wait_suspended(moved, 0, s.err));
      auto ready = [&](uint64_t* bar, int i) {
        ok = ok && wait_polling(bar, (uint32_t)i & 1u, s.err);
        jxd::tc_fence_after();
        return ok;
      };
      auto q_scores = [&](int u) {
        if (u >= n || !ready(&qfull[u % QS], u / QS)) return;
        mma_scores<DP, BLK, false>(tmem + L::X + (u & 1) * L::X_STEP, jxd::smem_u32(smem), qbase + (u % QS) * STAGE,
                                   HPANEL, PART);
        jxd::mma_commit(&sfull[u & 1]);
      };
      auto d_scores = [&](int u) {
        if (u >= n || !ready(&dfull[u % DS], u / DS)) return;
        mma_scores<DP, BLK, !L::APART>(tmem + L::Y + (u & 1) * L::Y_STEP,
                                       L::APART ? jxd::smem_u32(at_v) : tmem + L::V, dbase + (u % DS) * STAGE, HPANEL,
                                       PART);
        jxd::mma_commit(&dpfull[u & 1]);
      };
      auto v_sums = [&](int u) {
        mma_sums<DP, BLK>(tmem + L::Z, tmem + L::X + (u & 1) * L::X_STEP, dbase + (u % DS) * STAGE, HPANEL, PART);
        jxd::mma_commit(zfull);
        jxd::mma_commit(&dempty[u % DS]);
      };
      auto k_sums = [&](int u) {
        mma_sums<DP, BLK>(tmem + L::W, tmem + L::Y + (u & 1) * L::Y_STEP, qbase + (u % QS) * STAGE, HPANEL, PART);
        jxd::mma_commit(wfull);
        jxd::mma_commit(&qempty[u % QS]);
      };
      q_scores(0);
      d_scores(0);
      if (!L::APART) q_scores(1);
      for (int u = 0; ok && u < n; ++u) {
        if constexpr (L::APART) {
          q_scores(u + 1);  // over P of u-1, which dV(u-1) has read
          if (!ready(pfull, u) || !ready(zfree, u + 1)) break;
          v_sums(u);
          if (!ready(dsfull, u) || !ready(wfree, u + 1)) break;
          k_sums(u);
          d_scores(u + 1);
        } else {
          if (!ready(pfull, u) || !ready(wfree, u + 1)) break;
          v_sums(u);
          d_scores(u + 1);
          if (!ready(dsfull, u) || !ready(zfree, u)) break;
          k_sums(u);
          q_scores(u + 2);
        }
      }
      if (!ok) *abort_flag = 1;
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(BW_HIGH_REGS));
    const int quarter = warp & 3, half = (warp - BW_FIRST) >> 2, row = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    bool ok = true;
    auto ready = [&](uint64_t* bar, int i) {
      warp_wait(bar, (uint32_t)i & 1u, ok, abort_flag, s.err);
      jxd::tc_fence_after();
    };
    auto done = [&](uint64_t* bar) {
      jxd::tc_fence_before();
      __syncwarp();
      if (lane == 0) jxd::mbar_arrive(bar);
    };
    if (!L::APART && n > 0) {
      ready(stayfull, 0);
      if constexpr (!L::APART) tile_to_tmem<DP>(at_v, row, half, tmem + lanes + L::V);
      tmem_st_wait();
      done(moved);
    }
    const float4 num_k = bt.num_k[kslot];
    const float f_tile = num_k.x * (s.scale * LOG2E), inv_v = num_k.y, norm_v = num_k.z;
    const int first = row < rows ? sq.first_row(j0 + row, s.causal) : 0x7fffffff;  // first query row that sees this key
    const int first_all = sq.first_row(j0 + rows - 1, s.causal);

    float ak[DP / 2], av[DP / 2];
#pragma unroll
    for (int c = 0; c < DP / 2; ++c) ak[c] = av[c] = 0.0f;
    float g_prev = 0.0f;
    constexpr int C = BLK / 2;  // columns of the scores that this thread has
    int i0 = (blk0 + (n > 0 ? it0 % nblk : 0) - 1) * BLK;  // the block's first row
    const float2* later = bt.later + (qslot0 + (n > 0 ? it0 / nblk : 0)) * TILE;  // of the head's first tile
    for (int u = 0; u < n; ++u) {
      i0 += BLK;  // the next block, or the next head's first
      if (i0 >= sq.lq) {
        i0 = blk0 * BLK;
        later += TILE;
      }
      // the block's rows from the first that sees this key on
      const float2 tops = later[(long long)(i0 / TILE) * s.heads * TILE + i0 % TILE + min(max(first - i0, 0), BLK - 1)];
      const float* lse2 = stats + (u & 1) * L::STATS + half * C;
      const float* delta = lse2 + BLK;
      const uint32_t xa = tmem + lanes + L::X + (u & 1) * L::X_STEP + half * C;
      const uint32_t ya = tmem + lanes + L::Y + (u & 1) * L::Y_STEP + half * C;
      const bool edge = i0 < first_all || rows < TILE;  // some key is not seen by all of the block's rows
      float2 p[C / 2];
      warp_wait(&tfull[u & 1], (uint32_t)(u >> 1) & 1u, ok, abort_flag, s.err);
      const float4 num = *reinterpret_cast<const float4*>(stats + (u & 1) * L::STATS + 2 * BLK);
      const float inv_q = num.x, inv_d = num.y, norm_d = fmaxf(tops.x, num.z * LEAST_NORM), f = f_tile * inv_q;
      const float2 f2 = make_float2(f, f);
      ready(&sfull[u & 1], u >> 1);
#pragma unroll
      for (int c = 0; c < C; c += 32) {
        uint32_t r[32];
        jxd::tmem_ld32(xa + c, r);
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
#pragma unroll
        for (int i = 0; i < C / 2; ++i) {
          if (i0 + half * C + 2 * i < first) p[i].x = 0.0f;
          if (i0 + half * C + 2 * i + 1 < first) p[i].y = 0.0f;
        }
      }
#pragma unroll
      for (int c = 0; c < C; c += 32) {
        uint32_t hi[16], lo[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) split_half(p[c / 2 + i].x, p[c / 2 + i].y, hi[i], lo[i]);
        tmem_st16(xa + c, hi);
        tmem_st16(xa + c + 16, lo);
      }
      tmem_st_wait();
      done(pfull);
      if (u > 0) {
        ready(wfull, u - 1);
        drain<DP>(ak, tmem + lanes + L::W + half * (DP / 2), g_prev);
        done(wfree);
      }
      // P is at most 2^14
      const float fd = inv_v * inv_d, sc = bound_scale(16384.0f * (norm_v * norm_d + tops.y));
      const float pf = scale_ratio(sc, fd), nf = -inverse_pow2(fd);
      const float2 pf2 = make_float2(pf, pf), nf2 = make_float2(nf, nf);
      ready(&dpfull[u & 1], u >> 1);
#pragma unroll
      for (int c = 0; c < C; c += 32) {
        uint32_t r[32], hi[16], lo[16];
        jxd::tmem_ld32(ya + c, r);
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
        tmem_st16(ya + c, hi);
        tmem_st16(ya + c + 16, lo);
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
    // every MMA has retired: the tiles' and the stages' memory is free
    const int tid = threadIdx.x - 32 * BW_FIRST;
    uint8_t* area_v = smem + area_bytes(DP);
    half_to_area<DP>(smem, ak, s.scale, row, half);
    half_to_area<DP>(area_v, av, 1.0f, row, half);
    movers_sync();
    rows_store<DP>(out_k + (sq.k0 + j0) * ld_k + kd, ld_k, smem, rows, s.dim, aligned16(out_k, s.dim, ld_k), tid);
    rows_store<DP>(out_v + (sq.k0 + j0) * ld_v + kd, ld_v, area_v, rows, s.dim, aligned16(out_v, s.dim, ld_v), tid);
  }
  jxd::tc_fence_before();
  __syncthreads();
  jxd::tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    jxd::tmem_dealloc(tmem, 512);
  }
}

// Both in one launch, so that one kind's CTAs start as the other's last ones run.
// Neither reads what the other writes.  dk's and dv's come first, being the longer
// ones: 8 heads, 32 rows 15.6 us in a graph against 17.5 the other way round, 4096 packed tokens 184 against 186.
// (As launches of their own, where dk's has to wait for dq's end before it may read
// the tiles, these take 23.3 and 180: dq's steps are 450 cycles shorter in a kernel of its own.)
template <int DP>
__global__ void __launch_bounds__(BW_THREADS, 1)
    attn_bwd_kernel(const __grid_constant__ Shape s, const __grid_constant__ BwdTiles bt, const float* __restrict__ q,
                    const float* __restrict__ k, const float* __restrict__ v, const float* __restrict__ o,
                    const float* __restrict__ lse, const float* __restrict__ dout, float* dq, float* dk, float* dv) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const unsigned dkv_blocks = (unsigned)bt.k_tiles * (unsigned)s.kv_heads * (unsigned)bt.parts;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the tiles are complete behind it
  if (blockIdx.x < dkv_blocks) dkv_tile<DP>(s, bt, smem_raw, blockIdx.x, q, k, v, o, lse, dout, dk, dv);
  else dq_tile<DP>(s, bt, smem_raw, blockIdx.x - dkv_blocks, q, k, v, o, lse, dout, dq);
}

// The parts' sums in order, 16 key rows of one key head per block.
constexpr int JOIN_ROWS = 16;
template <bool VEC>
__global__ void __launch_bounds__(256) attn_dkv_join_kernel(const __grid_constant__ Shape s,
                                                           const __grid_constant__ BwdTiles bt, float* dk, float* dv) {
  int jt;
  const int b = seq_of_tile(s.cu_k, s.batch, s.total_k, blockIdx.x / (TILE / JOIN_ROWS), &jt);
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
  constexpr size_t smem = std::max(DqLayout<DP>::SMEM, KvLayout<DP>::SMEM);
  if (int rc = prepare_kernel((const void*)attn_bwd_kernel<DP>, DP == 128 ? 2 : 3, smem, BW_LAUNCH_REGS)) return rc;
  const long long blocks = (long long)bt.q_tiles * s.heads + (long long)bt.k_tiles * s.kv_heads * bt.parts;
  JX_CUDA(launch_overlapped(attn_bwd_kernel<DP>, blocks, BW_THREADS, smem, st, s, bt, q, k, v, o, lse, dout, dq, dk, dv));
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

static int bwd_heads(const Shape& s, const float* q, const float* k, const float* v, const float* o, const float* lse,
              const float* dout, float* dq, float* dk, float* dv, long long max_q, cudaStream_t st) {
  const int DP = s.dim <= 64 ? 64 : 128;
  const long long kt = tile_count(s.total_k, s.batch), qt = tile_count(s.total_q, s.batch);
  // key tiles are few where heads are shared: enough parts of the query rows for four CTAs per SM, of four blocks at least
  const long long ctas = kt * s.kv_heads, blocks = s.group * ((max_q + 63) / 64);
  const int parts =
      (int)std::max<long long>(1, std::min(std::min<long long>(8, blocks / 4), 4LL * jx::num_sms() / std::max(1LL, ctas)));
  JX_REQUIRE(qt * s.heads + kt * s.kv_heads * parts < (1LL << 31) && kt < (1LL << 27),
             "attention_bwd: too many rows");
  const size_t ks = (size_t)kt * s.kv_heads, qs = (size_t)qt * s.heads, tb = tile_bytes(DP);
  const size_t part_floats = parts > 1 ? (size_t)parts * s.total_k * s.kv_heads * s.dim : 0;
  // tiles first, then arrays whose pieces the copies read 16-byte aligned, then the rest
  const size_t bytes = (2 * ks + 2 * qs) * tb + 5 * qs * TILE * 4 + (6 * ks + 6 * qs) * 4 + (qt + kt) * sizeof(TileRef) +
                       2 * part_floats * 4;
  void* p = nullptr;
  if (int rc = jx::scratch_get(bytes + 64, &p, st)) return rc;
  uint8_t* at = static_cast<uint8_t*>(p);
  auto take = [&](size_t n) {
    uint8_t* r = at;
    at += n;
    return r;
  };
  uint8_t *tk = take(ks * tb), *tv = take(ks * tb), *tq = take(qs * tb), *td = take(qs * tb);
  TileRef *order_q = (TileRef*)take(qt * sizeof(TileRef)), *order_k = (TileRef*)take(kt * sizeof(TileRef));
  float* lse2 = (float*)take(qs * TILE * 4);
  float* delta = (float*)take(qs * TILE * 4);
  float* row_norm = (float*)take(qs * TILE * 4);
  float2* later = (float2*)take(qs * TILE * 8);
  float *num_q = (float*)take(qs * 16), *num_k = (float*)take(ks * 16);
  float* part_k = (float*)take(part_floats * 4);
  float* part_v = (float*)take(part_floats * 4);
  int *bad_k = (int*)take(ks * 4), *bad_v = (int*)take(ks * 4), *bad_q = (int*)take(qs * 4), *bad_d = (int*)take(qs * 4);
  TileSources src = {};
  src.keys = src.queries = 2;
  src.order_q = order_q;
  src.order_k = order_k;
  src.t[0] = {k, s.ldk, tk, num_k, bad_k, 4};
  src.t[1] = {v, s.ldv, tv, num_k + 1, bad_v, 4, num_k + 2};
  src.t[2] = {q, s.ldq, tq, num_q, bad_q, 4};
  src.t[3] = {dout, s.ldo, td, num_q + 1, bad_d, 4, num_q + 2, o, lse, lse2, delta, row_norm, later};
  const BwdTiles bt = {tq,    tk,    tv,    td,    (const float4*)num_q, (const float4*)num_k, bad_q, bad_k,
                       bad_v, bad_d, lse2,  delta, row_norm, later, (int)qt, (int)kt, parts, order_q, order_k, part_k, part_v};
  int rc = split_tiles(s, src, DP, st);
  if (!rc)
    rc = DP == 128 ? launch<128>(s, bt, q, k, v, o, lse, dout, dq, dk, dv, st)
                   : launch<64>(s, bt, q, k, v, o, lse, dout, dq, dk, dv, st);
  jx::scratch_release(p, st);
  return rc;
}

int attention_bwd_tiles(const Shape& s, const float* q, const float* k, const float* v, const float* o,
                        const float* lse, const float* dout, float* dq, float* dk, float* dv, long long max_q,
                        cudaStream_t st) {
  const int DP = s.dim <= 64 ? 64 : 128;
  const long long tiles = 2 * tile_count(s.total_k, s.batch) + 2 * s.group * tile_count(s.total_q, s.batch);
  const int each = group_of_heads(s.kv_heads, (size_t)tiles * tile_bytes(DP));
  for (int hk = 0; hk < s.kv_heads; hk += each) {
    const long long h = (long long)hk * s.group, hd = h * s.dim, kd = (long long)hk * s.dim;
    if (int rc = bwd_heads(heads_of(s, std::min(each, s.kv_heads - hk)), q + hd, k + kd, v + kd, o + hd,
                           lse + h * s.total_q, dout + hd, dq + hd, dk + kd, dv + kd, max_q, st))
      return rc;
  }
  return JX_OK;
}

}  // namespace jxa
