// attn_fwd.cu -- attention's forward pass on the tensor cores, and the split of
// its streamed operands into f16 tiles (attn_tc.cuh).
//
// One CTA per (128 query rows, head).  Q's parts lie in tensor memory; the parts of K
// and V tiles of 128 keys stream through shared memory.  Per key tile j, at dim 128:
//   S = Q K^T          24 MMAs of 128 x 128 x 16 (3 products x 8 steps), 64 cycles each
//   P = exp2(S f - m)  eight warps, two threads per row, 64 columns each; P's
//                      parts go back over S's columns
//   part = P V         24 MMAs, A from tensor memory
//   O = O alpha + part in registers, 64 columns per thread
// The MMA warp issues S(j+1) before part(j), so the softmax of tile j+1 has the
// time of part(j) and S(j+2).  Tensor memory: S twice 128 columns, Q 128, part 128.
//
// A step takes 3090 cycles (the mean of 64), 99% of the MMAs' rate.  8192 tokens, 32
// heads on 8, dim 128, causal: 1.31 to 1.33 ms, 1240 to 1260 TFLOP/s of f16 products, under
// the power limit (1372 MHz).  Short sequences pay about 5 us per CTA besides: its
// start, Q on its way through shared memory, the first tiles' latency, O's store.
// (Persistent CTAs, tried with the gradients, made the loops slower by what they saved.)
#include <algorithm>
#include <atomic>

#include "attn_tc.cuh"

namespace {

using namespace jxa;
using jxg::wait_bounded;

// ---- splitting -----------------------------------------------------------------
// One block per (tile, head, tensor): eight columns of four rows per thread.  (Of 64
// columns with 512 threads, two rows each, the packed gradient's call takes 6 us
// longer: the fewer blocks of an SM load and store in step.)
__host__ __device__ constexpr int sp_threads(int DP) { return 4 * DP; }

__device__ __forceinline__ void load_part(float (&x)[8], const float* p, int left, bool vec) {
#pragma unroll
  for (int e = 0; e < 8; e += 4) {
    float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
    if (vec && e + 4 <= left) {
      f = *reinterpret_cast<const float4*>(p + e);
    } else {
      if (e < left) f.x = p[e];
      if (e + 1 < left) f.y = p[e + 1];
      if (e + 2 < left) f.z = p[e + 2];
      if (e + 3 < left) f.w = p[e + 3];
    }
    x[e] = f.x;
    x[e + 1] = f.y;
    x[e + 2] = f.z;
    x[e + 3] = f.w;
  }
}

// Tiles that the tile's CTA works through: key tiles that a query tile's last row
// sees, or query tiles that see a key tile's first key.
__device__ __forceinline__ int tile_work(const Shape& s, bool over_q, int id, TileRef* ref) {
  const int32_t* cu = over_q ? s.cu_q : s.cu_k;
  const long long total = over_q ? s.total_q : s.total_k;
  int lo = 0, hi = s.batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first_tile_of(cu, mid, total) <= id) lo = mid;
    else hi = mid;
  }
  const int j = id - first_tile_of(cu, lo, total);
  const Seq sq = seq_bounds(s, lo);
  const bool in = j >= 0 && (long long)j * TILE < (over_q ? sq.lq : sq.lk);
  *ref = {sq.q0, sq.k0, sq.lq, sq.lk, lo, in ? j : -1};
  if (!in) return 0;
  if (over_q) return (sq.visible(min(j * TILE + TILE, sq.lq) - 1, s.causal) + TILE - 1) / TILE + 1;
  return max(0, (sq.lq - sq.first_row(j * TILE, s.causal) + TILE - 1) / TILE) + 1;
}
// One block: a counting sort by falling work.  Ids of equal work come in any order,
// which changes when they are computed and nothing else.
template <int THREADS>
__device__ void order_tiles(const Shape& s, bool over_q, int tiles, int shift, TileRef* order) {
  constexpr int EACH = ORDER_KEYS / THREADS;  // keys of a thread
  __shared__ int count[ORDER_KEYS], sums[THREADS / 32];
  const int tid = threadIdx.x;
  for (int i = tid; i < ORDER_KEYS; i += THREADS) count[i] = 0;
  __syncthreads();
  TileRef ref;
  auto key = [&](int id) { return ORDER_KEYS - 1 - min(tile_work(s, over_q, id, &ref) >> shift, ORDER_KEYS - 1); };
  for (int id = tid; id < tiles; id += THREADS) atomicAdd(&count[key(id)], 1);
  __syncthreads();
  // exclusive prefix sums
  int own[EACH], x = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) x += own[i] = count[EACH * tid + i];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if ((tid & 31) >= o) x += y;
  }
  if ((tid & 31) == 31) sums[tid >> 5] = x;
  __syncthreads();
  for (int w = 0; w < (tid >> 5); ++w) x += sums[w];
#pragma unroll
  for (int i = EACH - 1; i >= 0; --i) count[EACH * tid + i] = x -= own[i];
  __syncthreads();
  for (int id = tid; id < tiles; id += THREADS) {
    const int at = atomicAdd(&count[key(id)], 1);
    order[at] = ref;
  }
}

template <int DP>
__global__ void __launch_bounds__(sp_threads(DP), 1024 / sp_threads(DP))
    split_tiles_kernel(const __grid_constant__ Shape s, const __grid_constant__ TileSources src) {
  constexpr int SP_THREADS = sp_threads(DP);
  constexpr int PER_ROW = DP / 8, STEP = SP_THREADS / PER_ROW, ROWS = TILE / STEP;  // threads; rows at a time; rows each
  __shared__ uint32_t sm_top[SP_THREADS / 32], sm_low[SP_THREADS / 32];
  asm volatile("griddepcontrol.launch_dependents;");
  if (blockIdx.x < 2) {  // the orders
    if (blockIdx.x == 0 && src.order_q) order_tiles<SP_THREADS>(s, true, src.q_tiles, src.shift, src.order_q);
    if (blockIdx.x == 1 && src.order_k) order_tiles<SP_THREADS>(s, false, src.k_tiles, src.shift, src.order_k);
    return;
  }
  // the tensor, tile and head
  long long at_block = blockIdx.x - 2;
  const long long per_k = (long long)src.k_tiles * s.kv_heads, per_q = (long long)src.q_tiles * s.heads;
  const bool over_q = at_block >= src.keys * per_k;
  if (over_q) at_block -= src.keys * per_k;
  const int which = (int)(at_block / (over_q ? per_q : per_k)) + (over_q ? src.keys : 0);
  at_block %= over_q ? per_q : per_k;
  const int heads = over_q ? s.heads : s.kv_heads;
  const TileSource& t = src.t[which];
  const int id = (int)(at_block / heads), h = (int)(at_block - (long long)id * heads);
  int j;
  const int b = seq_of_tile(over_q ? s.cu_q : s.cu_k, s.batch, over_q ? s.total_q : s.total_k, id, &j);
  const Seq sq = seq_bounds(s, b);
  const int len = over_q ? sq.lq : sq.lk;
  if (j < 0 || (long long)j * TILE >= len) return;
  const long long row0 = (over_q ? sq.q0 : sq.k0) + (long long)j * TILE;
  const int rows = min(TILE, len - j * TILE);
  const int c = threadIdx.x % PER_ROW, r0 = threadIdx.x / PER_ROW;
  const int col = c * 8, left = s.dim - col;
  const long long hd = (long long)h * s.dim + col;
  const bool vec = (s.dim & 3) == 0 && (t.ld & 3) == 0 && (reinterpret_cast<uintptr_t>(t.x) & 15) == 0;
  float x[ROWS][8];
  {
    const float* p = t.x + (row0 + r0) * t.ld + hd;
#pragma unroll
    for (int i = 0; i < ROWS; ++i, p += STEP * t.ld) load_part(x[i], p, r0 + STEP * i < rows ? left : 0, vec);
  }
  uint32_t top = 0, low = 0x7fffffffu;  // the tile's largest row maximum, and the smallest one that is not zero
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(x[i][e]) & 0x7fffffffu);
#pragma unroll
    for (int o = PER_ROW / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    top = max(top, m);
    if (m) low = min(low, m);
  }
#pragma unroll
  for (int o = PER_ROW; o < 32; o <<= 1) {
    top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    low = min(low, __shfl_xor_sync(0xffffffffu, low, o));
  }
  if ((threadIdx.x & 31) == 0) {
    sm_top[threadIdx.x >> 5] = top;
    sm_low[threadIdx.x >> 5] = low;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < SP_THREADS / 32; ++w) {
    top = max(top, sm_top[w]);
    low = min(low, sm_low[w]);
  }
  const int e_top = (int)(top >> 23), e_low = (int)(low >> 23);
  const long long slot = (long long)id * heads + h;
  if (threadIdx.x == 0) {
    t.inverse[slot * t.step] = inverse_of(e_top);
    t.bad[slot] = unscaled(top) || (top && e_top - e_low > WIDE_BITS);
  }
  const float factor = scale_of(e_top);
  const int at = col * 2;  // byte of the row; r0 + STEP * i has the same low three bits for every i
  uint8_t* out = t.tiles + slot * tile_bytes(DP) + (at >> 7) * PANEL + r0 * 128 + ((((at & 127) >> 4) ^ (r0 & 7)) << 4);
  static_assert(STEP % 8 == 0, "rows of a thread share their swizzle");
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) split_half(x[i][2 * e] * factor, x[i][2 * e + 1] * factor, hi[e], lo[e]);
    *reinterpret_cast<uint4*>(out + i * STEP * 128) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    *reinterpret_cast<uint4*>(out + i * STEP * 128 + tile_part(DP)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  }
  if (t.norm) {
    __shared__ float sm_norm[TILE], sm_delta[TILE];  // of the rows: the scaled norm's square, |rowsum(dout o)|
    const bool vec_o = (s.dim & 3) == 0 && (s.ldo & 3) == 0 && (reinterpret_cast<uintptr_t>(t.o) & 15) == 0;
    float most = 0.0f;
    bool odd = false;
    const float* p = t.o + (row0 + r0) * s.ldo + hd;
#pragma unroll
    for (int i = 0; i < ROWS; ++i, p += STEP * s.ldo) {
      const int r = r0 + STEP * i;
      float n = 0.0f, d = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) n = fmaf(x[i][e] * factor, x[i][e] * factor, n);
      if (t.o) {
        float y[8];
        load_part(y, p, r < rows ? left : 0, vec_o);
#pragma unroll
        for (int e = 0; e < 8; ++e) d = fmaf(x[i][e], y[e], d);
      }
#pragma unroll
      for (int o = PER_ROW / 2; o > 0; o >>= 1) {
        n += __shfl_xor_sync(0xffffffffu, n, o);
        d += __shfl_xor_sync(0xffffffffu, d, o);
      }
      most = fmaxf(most, n);
      if (t.o && c == 0) {
        const float z = r < rows ? t.lse[(long long)h * s.total_q + row0 + r] : -INFINITY;
        odd = odd || !isfinite(d) || isnan(z) || z == INFINITY;
        t.lse2[slot * TILE + r] = z == -INFINITY ? INFINITY : z * LOG2E - P_SHIFT;
        t.delta[slot * TILE + r] = d;
        t.row_norm[slot * TILE + r] = sqrtf(n) * inverse_of(e_top);
        sm_norm[r] = n;
        sm_delta[r] = fabsf(d);
      }
    }
    odd = __syncthreads_or(odd);
    if (t.o && threadIdx.x < TILE) {  // from the back, over the rows of each block
      const int r = threadIdx.x, end = (r | (kv_block(DP) - 1)) + 1;
      float n = sm_norm[r], d = sm_delta[r];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        n = fmaxf(n, __shfl_down_sync(0xffffffffu, n, o));
        d = fmaxf(d, __shfl_down_sync(0xffffffffu, d, o));
      }
      for (int w = (r | 31) + 1; w < end; w += 32) {  // the block's later warps
        float n1 = sm_norm[w + (r & 31)], d1 = sm_delta[w + (r & 31)];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, o));
          d1 = fmaxf(d1, __shfl_xor_sync(0xffffffffu, d1, o));
        }
        n = fmaxf(n, n1);
        d = fmaxf(d, d1);
      }
      t.later[slot * TILE + r] = make_float2(sqrtf(n) * inverse_of(e_top), d);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    if ((threadIdx.x & 31) == 0) sm_low[threadIdx.x >> 5] = __float_as_uint(most);
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < SP_THREADS / 32; ++w) most = fmaxf(most, __uint_as_float(sm_low[w]));
      t.norm[slot * t.step] = sqrtf(most) * inverse_of(e_top);
      if (t.o && odd) t.bad[slot] = 1;
    }
  }
}

// ---- forward -------------------------------------------------------------------
constexpr int FW_THREADS = 384;  // warp 0 copies, warp 1 MMA, warps 4..11 softmax
constexpr int FW_FIRST = 4;
constexpr int FW_LAUNCH_REGS = 168;
constexpr int FW_LOW_REGS = 56;
constexpr int FW_HIGH_REGS = 216;
static_assert(128 * FW_LOW_REGS + 256 * FW_HIGH_REGS <= FW_THREADS * FW_LAUNCH_REGS,
              "register split exceeds the launch allocation");
constexpr uint32_t T_Q = 256, T_O = 384;  // columns of tensor memory; S0 at 0, S1 at 128

// A stage is one part of a tile: the lo part is used, and its stage free again,
// before the hi part is.
__host__ __device__ constexpr int fw_stages(int DP) { return DP == 128 ? 6 : 12; }
__host__ __device__ constexpr size_t fw_smem(int DP) {
  return (size_t)fw_stages(DP) * tile_part(DP) + 1024 /*align*/ + 4 * 128 * 4 /*exchange*/ + 512 /*barriers*/;
}

struct FwdTiles {
  const uint8_t* k;
  const uint8_t* v;
  const float* inv_k;
  const float* inv_v;
  const int* bad_k;
  const int* bad_v;
  const TileRef* order;  // of the query tiles
};

template <int DP>
__global__ void __launch_bounds__(FW_THREADS, 1)
    attn_fwd_kernel(const __grid_constant__ Shape s, const __grid_constant__ FwdTiles ft, const float* __restrict__ q,
                    const float* __restrict__ k, const float* __restrict__ v, float* o, float* lse) {
  constexpr int STAGES = fw_stages(DP), STAGE = tile_part(DP), PART = tile_part(DP);
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = jxd::smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
  float* xch = reinterpret_cast<float*>(smem + STAGES * STAGE);  // [2][2][128]
  uint64_t* full = reinterpret_cast<uint64_t*>(xch + 4 * 128);   // [STAGES]
  uint64_t* empty = full + STAGES;                               // [STAGES]
  uint64_t* sfull = empty + STAGES;                              // [2]
  uint64_t* pfull = sfull + 2;                                   // [2]
  uint64_t* ofull = pfull + 2;
  uint64_t* ofree = ofull + 1;
  uint64_t* qfull = ofree + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(qfull + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the split is complete behind it
  // the tiles that see the most keys start first
  const TileRef ref = load_ref(ft.order + blockIdx.x / (unsigned)s.heads);
  const int h = (int)(blockIdx.x % (unsigned)s.heads), b = ref.b, jt = ref.jt;
  const Seq sq = seq_of(ref);
  if (jt < 0) return;
  const int i0 = jt * TILE, rows = min(TILE, sq.lq - i0);
  const int hk = h / s.group;
  const int nk = sq.visible(i0 + rows - 1, s.causal);  // keys that the tile's last row sees
  const int nb = (nk + TILE - 1) / TILE;
  const long long slot0 = (long long)first_tile(sq.k0, b) * s.kv_heads + hk;

  const int quarter = warp & 3, half = (warp - FW_FIRST) >> 2, tid = threadIdx.x - 32 * FW_FIRST;
  const int row = quarter * 32 + lane;
  const bool soft = warp >= FW_FIRST;
  // Q passes through the last two stages; the copies for the others start at once
  uint8_t* area = smem + (STAGES - 2) * STAGE;
  const long long hd = (long long)h * s.dim;
  // copies, in the order of use: K0 K1 V0 K2 V1 ... K(n-1) V(n-2) V(n-1), of each its lo part, then hi
  auto copy = [&](int u, int stage) {
    const int w = u >> 1;
    const bool is_v = w == 2 * nb - 1 || (w >= 2 && (w & 1) == 0);
    const int j = w == 0 ? 0 : w == 2 * nb - 1 ? nb - 1 : is_v ? w / 2 - 1 : (w + 1) / 2;
    jxd::mbar_arrive_expect_tx(&full[stage], STAGE);
    bulk_load(jxd::smem_u32(smem + stage * STAGE),
              (is_v ? ft.v : ft.k) + (slot0 + (long long)j * s.kv_heads) * tile_bytes(DP) + (u & 1 ? 0 : STAGE), STAGE,
              &full[stage]);
  };
  const int first = min(4 * nb, STAGES - 2);
  bool bad = false;
  if (warp == 0 && lane == 0) {
    for (int i = 0; i < STAGES; ++i) {
      jxd::mbar_init(&full[i], 1);
      jxd::mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      jxd::mbar_init(&sfull[i], 1);
      jxd::mbar_init(&pfull[i], 8);
    }
    jxd::mbar_init(ofull, 1);
    jxd::mbar_init(ofree, 8);
    jxd::mbar_init(qfull, 8);
    *abort_flag = 0;
    jxd::fence_mbar_init();
    jxd::fence_proxy_async_smem();
    for (int u = 0; u < first; ++u) copy(u, u);
  } else if (warp == 1) {
    jxd::tmem_alloc(tmem_slot, 512);
    jxd::tmem_relinquish();
  } else if (soft) {
    float4 f[DP / 8];
    rows_load<DP>(f, q + (sq.q0 + i0) * s.ldq + hd, s.ldq, rows, s.dim, aligned16(q, s.dim, s.ldq), tid);
    rows_to_area<DP>(area, f, tid);
  } else if (warp >= 2) {
    for (int j = (int)threadIdx.x - 64; j < nb; j += 64)
      bad = bad || ft.bad_k[slot0 + (long long)j * s.kv_heads] || ft.bad_v[slot0 + (long long)j * s.kv_heads];
  }
  jxd::tc_fence_before();
  __syncthreads();
  jxd::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  float x[DP / 2];
  uint32_t top = 0;
  if (soft) {
    top = half_from_area<DP>(x, area, row, half);
    reinterpret_cast<uint32_t*>(xch)[half * 128 + row] = top;
    pair_sync(1 + quarter);
    top = max(top, reinterpret_cast<uint32_t*>(xch)[(half ^ 1) * 128 + row]);
    bad = unscaled(top);
  }
  if (__syncthreads_or(bad)) {
    // row by row, in plain f32
    for (int r = warp; r < rows; r += FW_THREADS / 32) {
      const long long t = sq.q0 + i0 + r;
      row_fwd(q + t * s.ldq + hd, k + sq.k0 * s.ldk + (long long)hk * s.dim, v + sq.k0 * s.ldv + (long long)hk * s.dim,
              o + t * s.ldo + hd, lse ? lse + (long long)h * s.total_q + t : nullptr, sq.visible(i0 + r, s.causal),
              s.dim, s.ldk, s.ldv, s.scale);
    }
    if (warp == 0 && lane == 0) {  // every copy has landed before the CTA may end
      unsigned long long end = 0;  // for all of them
      for (int u = 0; u < first; ++u) wait_suspended(&full[u], 0, s.err, end);
    }
    if (warp == 1) {
      __syncwarp();
      jxd::tmem_dealloc(tmem, 512);
    }
    return;
  }

  if (!soft) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(FW_LOW_REGS));
    if (warp == 0 && jxd::elect_one()) {
      // ---- the remaining copies
      int stage = first % STAGES, issued = first;
      uint32_t phase = 0;
      if (4 * nb > first && !wait_bounded(qfull, 0, s.err)) *abort_flag = 1;  // the last stages are free of Q
      for (int u = first; u < 4 * nb && !*abort_flag; ++u) {
        if (!wait_bounded(&empty[stage], phase ^ 1u, s.err)) { *abort_flag = 1; break; }
        copy(u, stage);
        ++issued;
        if (++stage == STAGES) { stage = 0; phase ^= 1u; }
      }
      // every copy has landed before the CTA may end
      unsigned long long end = 0;  // for all of them
      for (int u = max(0, issued - STAGES); u < issued; ++u)
        wait_suspended(&full[u % STAGES], (uint32_t)(u / STAGES) & 1u, s.err, end);
    }
    if (warp == 1 && nb > 0 && jxd::elect_one()) {
      // ---- MMA
      constexpr uint32_t id_s = idesc_f16(128, false), id_o = idesc_f16(DP, true);
      constexpr uint32_t SHRINK = 2;  // acc: 0 from zero, 1 onto the sum, SHRINK onto the sum times 2^-LO_BITS
      const uint32_t sbase = jxd::smem_u32(smem);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = wait_bounded(qfull, 0, s.err);
      // the next stage's shared-memory address once its copy has landed
      auto next = [&]() {
        ok = ok && wait_polling(&full[stage], phase, s.err);
        jxd::tc_fence_after();
        return sbase + stage * STAGE;
      };
      auto release = [&]() {
        jxd::mma_commit(&empty[stage]);
        if (++stage == STAGES) { stage = 0; phase ^= 1u; }
      };
      auto scores = [&](int j) {
        const uint32_t d = tmem + (j & 1) * 128u;
        auto step = [&](uint32_t kt, int ks, uint32_t a, uint32_t acc) {
          const uint64_t bd = jxd::smem_desc_k_sw128(kt + (ks >> 2) * PANEL + (ks & 3) * 32);
          if (acc == SHRINK) mma_f16_ts_shrink(d, tmem + T_Q + a + ks * 8, bd, id_s);
          else mma_f16_ts(d, tmem + T_Q + a + ks * 8, bd, id_s, acc);
        };
        uint32_t kt = next();
        if (!ok) return;
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) step(kt, ks, 0, ks > 0);  // hi.lo
        release();
        kt = next();
        if (!ok) return;
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) step(kt, ks, DP / 2, 1);  // lo.hi
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) step(kt, ks, 0, ks > 0 ? 1 : SHRINK);
        jxd::mma_commit(&sfull[j & 1]);
        release();
      };
      scores(0);
      for (int j = 0; j < nb && ok; ++j) {
        if (j + 1 < nb) scores(j + 1);
        if (!ok || !(ok = wait_polling(&pfull[j & 1], (uint32_t)(j >> 1) & 1u, s.err) &&
                          wait_polling(ofree, (uint32_t)(j + 1) & 1u, s.err)))
          break;
        const uint32_t p = tmem + (j & 1) * 128u, d = tmem + T_O;
        // P's keys 0..63: hi at column 0, lo at 32; keys 64..127: hi at 64, lo at 96
        auto step = [&](uint32_t vt, int ks, uint32_t a, uint32_t acc) {
          const uint32_t at = p + a + (ks >> 2) * 64 + (ks & 3) * 8;
          const uint64_t bd = smem_desc_mn_sw128(vt + ks * 2048, PANEL);
          if (acc == SHRINK) mma_f16_ts_shrink(d, at, bd, id_o);
          else mma_f16_ts(d, at, bd, id_o, acc);
        };
        uint32_t vt = next();
        if (!ok) break;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) step(vt, ks, 0, ks > 0);
        release();
        vt = next();
        if (!ok) break;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) step(vt, ks, 32, 1);
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) step(vt, ks, 0, ks > 0 ? 1 : SHRINK);
        jxd::mma_commit(ofull);
        release();
      }
      if (!ok) *abort_flag = 1;
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(FW_HIGH_REGS));
    // ---- softmax and output
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const int e_row = (int)(top >> 23);
    row_half_store<DP>(x, s.scale < 0.0f ? -scale_of(e_row) : scale_of(e_row), tmem + lanes + T_Q, half);
    tmem_st_wait();
    jxd::fence_proxy_async_smem();  // the area becomes a copy's destination
    jxd::tc_fence_before();
    __syncwarp();
    if (lane == 0) jxd::mbar_arrive(qfull);
    const float f_row = inverse_of(e_row) * (fabsf(s.scale) * LOG2E);
    const int vis = row < rows ? sq.visible(i0 + row, s.causal) : 0;
    const int vis_all = sq.visible(i0, s.causal);  // keys that every row of the tile sees

    float acc[DP / 2];
#pragma unroll
    for (int c = 0; c < DP / 2; ++c) acc[c] = 0.0f;
    float m = -INFINITY, shift = INFINITY, sum = 0.0f, alpha_prev = 0.0f, inv_v_prev = 0.0f;
    bool ok = true;

    auto add_part = [&](int j, float alpha, float inv_v) {
      warp_wait(ofull, (uint32_t)j & 1u, ok, abort_flag, s.err);
      jxd::tc_fence_after();
#pragma unroll
      for (int c = 0; c < DP / 2; c += 32) {
        uint32_t r[32];
        jxd::tmem_ld32(tmem + lanes + T_O + half * (DP / 2) + c, r);
        jxd::tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          const float2 part = make_float2(__uint_as_float(r[i]) * inv_v, __uint_as_float(r[i + 1]) * inv_v);
          const float2 v2 = fma2(make_float2(acc[c + i], acc[c + i + 1]), make_float2(alpha, alpha), part);
          acc[c + i] = v2.x;
          acc[c + i + 1] = v2.y;
        }
      }
      jxd::tc_fence_before();
      __syncwarp();
      if (lane == 0) jxd::mbar_arrive(ofree);
    };

    for (int j = 0; j < nb; ++j) {
      const float inv_k = ft.inv_k[slot0 + (long long)j * s.kv_heads];
      const float inv_v = ft.inv_v[slot0 + (long long)j * s.kv_heads];
      const float f = fmaxf(f_row * inv_k, 1.17549435e-38f);  // above zero, so that a masked score stays -inf
      warp_wait(&sfull[j & 1], (uint32_t)(j >> 1) & 1u, ok, abort_flag, s.err);
      jxd::tc_fence_after();
      const uint32_t s_addr = tmem + lanes + (j & 1) * 128u + half * 64u;
      float sc[64];
      {
        uint32_t r[32];
        jxd::tmem_ld32(s_addr, r);
        jxd::tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i) sc[i] = __uint_as_float(r[i]);
        jxd::tmem_ld32(s_addr + 32, r);
        jxd::tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i) sc[32 + i] = __uint_as_float(r[i]);
      }
      const int key0 = j * TILE + half * 64;
      if (j * TILE + TILE > vis_all) {  // some row does not see all of the tile's keys
#pragma unroll
        for (int i = 0; i < 64; ++i)
          if (key0 + i >= vis) sc[i] = -INFINITY;
      }
      float mx = sc[0];
#pragma unroll
      for (int i = 1; i < 64; ++i) mx = fmaxf(mx, sc[i]);
      // the row's other half (two turns: who writes a place again has seen the other at the turn between)
      float* turn = xch + (j & 1) * 256;
      turn[half * 128 + row] = mx;
      pair_sync(1 + quarter);
      mx = fmaxf(mx, turn[(half ^ 1) * 128 + row]);
      const float m_new = mx == -INFINITY ? m : fmaxf(m, mx * f);
      // the shift as it is rounded: everything else is computed with it, so that its error cancels
      const float up = m_new == -INFINITY ? P_SHIFT : P_SHIFT - m_new;
      const float alpha = exp2_fast(up - shift);
      m = m_new;
      if (m_new != -INFINITY) shift = up;
      const float2 f2 = make_float2(f, f), b2 = make_float2(up, up);
      float2 add = make_float2(0.0f, 0.0f);
      uint32_t hi[32], lo[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const float2 z = fma2(make_float2(sc[2 * i], sc[2 * i + 1]), f2, b2);
        const float2 p = make_float2(exp2_fast(z.x), exp2_fast(z.y));
        add.x += p.x;
        add.y += p.y;
        split_half(p.x, p.y, hi[i], lo[i]);
      }
      sum = sum * alpha + (add.x + add.y);
      tmem_st32(s_addr, hi);
      tmem_st32(s_addr + 32, lo);
      tmem_st_wait();
      jxd::tc_fence_before();
      __syncwarp();
      if (lane == 0) jxd::mbar_arrive(&pfull[j & 1]);
      if (j > 0) add_part(j - 1, alpha_prev, inv_v_prev);
      alpha_prev = alpha;
      inv_v_prev = inv_v;
    }
    if (nb > 0) add_part(nb - 1, alpha_prev, inv_v_prev);

    xch += (nb & 1) * 256;
    xch[half * 128 + row] = sum;
    pair_sync(1 + quarter);
    sum += xch[(half ^ 1) * 128 + row];
    // every MMA has retired: the stages are free
    half_to_area<DP>(smem, acc, sum == 0.0f ? 0.0f : 1.0f / sum, row, half);
    if (lse && half == 0 && row < rows)
      lse[(long long)h * s.total_q + sq.q0 + i0 + row] =
          sum == 0.0f ? -INFINITY : fmaf(P_SHIFT - shift, LN2, log2f(sum * 6.103515625e-05f) * LN2);  // 2^-14
    movers_sync();
    rows_store<DP>(o + (sq.q0 + i0) * s.ldo + hd, s.ldo, smem, rows, s.dim, aligned16(o, s.dim, s.ldo), tid);
  }
  jxd::tc_fence_before();
  __syncthreads();
  jxd::tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    jxd::tmem_dealloc(tmem, 512);
  }
}

}  // namespace

namespace jxa {

int split_tiles(const Shape& s, const TileSources& src, int DP, cudaStream_t st) {
  TileSources ts = src;
  ts.q_tiles = (int)tile_count(s.total_q, s.batch);
  ts.k_tiles = (int)tile_count(s.total_k, s.batch);
  for (ts.shift = 0; (std::max(ts.q_tiles, ts.k_tiles) >> ts.shift) >= ORDER_KEYS - 1; ++ts.shift) {}
  const long long blocks =
      2 + (long long)src.keys * ts.k_tiles * s.kv_heads + (long long)src.queries * ts.q_tiles * s.heads;
  JX_REQUIRE(blocks < (1LL << 31), "attention: too many rows");
  if (DP == 128) split_tiles_kernel<128><<<(unsigned)blocks, sp_threads(DP), 0, st>>>(s, ts);
  else split_tiles_kernel<64><<<(unsigned)blocks, sp_threads(DP), 0, st>>>(s, ts);
  JX_LAUNCH_CHECK("split_tiles_kernel");
  return JX_OK;
}

// Per device and variant, once: the shared-memory limit, and (launch_regs not 0) a
// check of the registers that the kernel was built with.
int prepare_kernel(const void* kernel, int variant, size_t smem, int launch_regs) {
  static std::atomic<int> done[64][32];
  int dev = 0;
  JX_CUDA(cudaGetDevice(&dev));
  std::atomic<int>& d = done[dev & 63][variant];
  if (d.load(std::memory_order_acquire)) return JX_OK;
  if (launch_regs) {
    cudaFuncAttributes fa;
    JX_CUDA(cudaFuncGetAttributes(&fa, kernel));
    if (fa.numRegs != launch_regs)  // setmaxnreg.inc would wait for registers that never come
      return jx::fail(JX_EUNSUPPORTED, "attention kernel built with %d registers per thread, expected %d", fa.numRegs,
                      launch_regs);
  }
  JX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  d.store(1, std::memory_order_release);
  return JX_OK;
}

static int fwd_heads(const Shape& s, const float* q, const float* k, const float* v, float* o, float* lse, cudaStream_t st) {
  const int DP = s.dim <= 64 ? 64 : 128;
  const long long kt = tile_count(s.total_k, s.batch), qt = tile_count(s.total_q, s.batch);
  JX_REQUIRE(qt * s.heads < (1LL << 31) && kt < (1LL << 31), "attention: too many rows");
  const size_t slots = (size_t)kt * s.kv_heads, bytes = slots * tile_bytes(DP);
  void* p = nullptr;
  if (int rc = jx::scratch_get(2 * bytes + qt * sizeof(TileRef) + 4 * slots * sizeof(float), &p, st)) return rc;
  uint8_t* base = static_cast<uint8_t*>(p);
  TileRef* order = reinterpret_cast<TileRef*>(base + 2 * bytes);
  float* inv = reinterpret_cast<float*>(order + qt);
  int* bad = reinterpret_cast<int*>(inv + 2 * slots);
  TileSources src = {};
  src.t[0] = {k, s.ldk, base, inv, bad, 1};
  src.t[1] = {v, s.ldv, base + bytes, inv + slots, bad + slots, 1};
  src.keys = 2;
  src.order_q = order;
  FwdTiles ft = {base, base + bytes, inv, inv + slots, bad, bad + slots, order};
  int rc = split_tiles(s, src, DP, st);
  if (!rc) {
    const unsigned grid = (unsigned)(qt * s.heads);
    if (DP == 128) {
      if (!(rc = prepare_kernel((const void*)attn_fwd_kernel<128>, 0, fw_smem(128), FW_LAUNCH_REGS)))
        rc = jx::check_cuda(launch_overlapped(attn_fwd_kernel<128>, grid, FW_THREADS, fw_smem(128), st, s, ft, q, k, v, o, lse),
                            "attn_fwd_kernel");
    } else {
      if (!(rc = prepare_kernel((const void*)attn_fwd_kernel<64>, 1, fw_smem(64), FW_LAUNCH_REGS)))
        rc = jx::check_cuda(launch_overlapped(attn_fwd_kernel<64>, grid, FW_THREADS, fw_smem(64), st, s, ft, q, k, v, o, lse),
                            "attn_fwd_kernel");
    }
  }
  jx::scratch_release(p, st);
  return rc;
}

int attention_fwd_tiles(const Shape& s, const float* q, const float* k, const float* v, float* o, float* lse,
                        cudaStream_t st) {
  const int DP = s.dim <= 64 ? 64 : 128;
  const int each = group_of_heads(s.kv_heads, 2 * (size_t)tile_count(s.total_k, s.batch) * tile_bytes(DP));
  for (int hk = 0; hk < s.kv_heads; hk += each) {
    const long long h = (long long)hk * s.group;
    if (int rc = fwd_heads(heads_of(s, std::min(each, s.kv_heads - hk)), q + h * s.dim, k + (long long)hk * s.dim,
                           v + (long long)hk * s.dim, o + h * s.dim, lse ? lse + h * s.total_q : nullptr, st))
      return rc;
  }
  return JX_OK;
}

}  // namespace jxa
