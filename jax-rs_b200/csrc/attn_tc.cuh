// attn_tc.cuh -- the tensor-core attention kernels' shared pieces: operand
// tiles split into two f16 parts, their layout in scratch and shared memory,
// and the tcgen05 wrappers for operands in tensor memory.
//
// Numbers.  An f32 operand x is held as hi + 2^-11 lo, hi = f16(x s), lo =
// f16((x s - hi) 2^11), with s a power of two that brings the largest magnitude of
// its scaling group (a row of forward's Q, 128 rows of one head otherwise) into
// [2^14, 2^15).  hi + 2^-11 lo keeps 22 bits of every value within 2^-28 of the
// largest and an absolute 2^-50 of the largest below that (without the 2^11, lo
// would run out of f16's exponents at 2^-17).  A product is 2^-11 (lo.hi + hi.lo) +
// hi.hi, three f16 products with f32 sums: twice the rate of the same with tf32
// parts, whose 22 bits are the same; the first hi.hi product shrinks the sum so far
// by 2^-11 as it adds.  A tile that holds a non-finite value, or rows whose largest
// values differ by more than 2^20, is marked; the tiles of output that need it are
// computed row by row in plain f32.
//
// Sums.  The tensor core truncates as it accumulates, so a sum in tensor memory
// spans at most 128 terms, small parts first; spans are added in f32 registers.
//
// Layout.  Tile (id, head): 128 rows of DP = 64 or 128 columns (zero behind the
// head's dim), [hi][lo], each part as panels of 64 columns: row r of a panel is
// 128 bytes, its 16-byte chunk c at r * 128 + ((c ^ (r & 7)) * 16), the 128-byte
// swizzle.  The same bytes serve as a K-major operand (rows x columns summed
// over columns) and as an MN-major one (summed over rows).
//
// Tiles of a packed sequence.  Sequence b's tile j has id (start / 128) + b + j:
// ids of different sequences never meet, whatever the lengths, and
// total / 128 + batch of them are enough, so neither a table nor the lengths on
// the host are needed.
#pragma once

#include <cuda_fp16.h>

#include <algorithm>

#include "attn_common.cuh"
#include "tc_gemm.cuh"

namespace jxa {

constexpr int TILE = 128;
constexpr int PANEL = TILE * 128;  // bytes of 128 rows x 64 f16 columns
constexpr int WIDE_BITS = 20;
__host__ __device__ constexpr int kv_block(int DP) { return DP == 64 ? 128 : 64; }  // query rows of a step of dk and dv
constexpr int LO_BITS = 11;  // lo parts are held times 2^LO_BITS
constexpr float P_SHIFT = 14.0f;  // softmax weights are scaled by 2^14 for their f16 parts

__host__ __device__ constexpr int tile_part(int DP) { return DP / 64 * PANEL; }      // one part of a tile
__host__ __device__ constexpr int tile_bytes(int DP) { return 2 * tile_part(DP); }   // hi and lo

inline long long tile_count(long long total, int batch) { return total / TILE + batch; }

// Tiles are whole, so that sequences far shorter than 128 rows take scratch by
// their number, not by their rows.  Beyond SCRATCH of it the key heads are taken in
// groups, one group's launches behind the other's (SCRATCH is some ten thousand
// CTAs' work, so that a group fills the GPU as all of them would).
constexpr size_t SCRATCH = size_t{2} << 30;
// Key heads of a group, for `bytes` of scratch a key head.
inline int group_of_heads(int kv_heads, size_t bytes) {
  const int most = (int)std::max<size_t>(1, std::min<size_t>(kv_heads, SCRATCH / std::max<size_t>(1, bytes)));
  const int groups = (kv_heads + most - 1) / most;
  return (kv_heads + groups - 1) / groups;
}
// Whether even one key head's tiles are beyond SCRATCH, and four times what its rows alone would fill.
inline bool tiles_mostly_empty(const Shape& s, bool gradients) {
  const long long per_q = gradients ? 2 * s.group : 0;
  const long long tiles = 2 * tile_count(s.total_k, s.batch) + per_q * tile_count(s.total_q, s.batch);
  const long long filled = 2 * tile_count(s.total_k, 1) + per_q * tile_count(s.total_q, 1);
  return tiles > 4 * filled && (size_t)tiles * tile_bytes(s.dim <= 64 ? 64 : 128) > SCRATCH;
}
// The call's shape for `n` of its key heads.
inline Shape heads_of(const Shape& s, int n) {
  Shape r = s;
  r.kv_heads = n;
  r.heads = n * s.group;
  return r;
}

__device__ __forceinline__ int first_tile(long long start, int b) { return (int)(start >> 7) + b; }
// The first tile of sequence b from its offset, taken into the tensor as seq_bounds takes it.
__device__ __forceinline__ int first_tile_of(const int32_t* cu, int b, long long total) {
  return first_tile(max(0LL, min((long long)cu[b], total)), b);
}
// Sequence and index within it of tile `id` (warp-uniform); the index may lie behind the sequence's end.
__device__ __forceinline__ int seq_of_tile(const int32_t* cu, int batch, long long total, int id, int* j) {
  const int b = last_at_most(batch, id, [&](int i) { return (long long)first_tile_of(cu, i, total); });
  *j = id - first_tile_of(cu, b, total);
  return b;
}

// Power of two that brings a magnitude with biased exponent e into [2^14, 2^15), and its inverse.
// e below LEAST_E (zeros among them) takes LEAST_E's scale.
constexpr int LEAST_E = 79;
__device__ __forceinline__ float scale_of(int e) {
  return __uint_as_float((uint32_t)(268 - min(max(e, LEAST_E), 254)) << 23);
}
__device__ __forceinline__ float inverse_of(int e) {
  return __uint_as_float((uint32_t)(min(max(e, LEAST_E), 254) - 14) << 23);
}
// Magnitude bits that the scales do not serve: not finite, or tiny but not zero.
__device__ __forceinline__ bool unscaled(uint32_t top) {
  return top >= 0x7f800000u || (top != 0 && (int)(top >> 23) < LEAST_E - 17);
}

__device__ __forceinline__ uint32_t pack_half(float a, float b) {  // a in the low half
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\t"
      "mov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmov.b64 rc, {%6, %7};\n\t"
      "fma.rn.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\t"
      "mov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
      "mul.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
// hi and lo parts of two scaled values; both steps of the remainder are exact.
__device__ __forceinline__ void split_half(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = pack_half(a, b);
  const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  constexpr float UP = 1 << LO_BITS;
  const float2 r = mul2(fma2(h, make_float2(-1.0f, -1.0f), make_float2(a, b)), make_float2(UP, UP));
  lo = pack_half(r.x, r.y);
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// ---- tcgen05 ------------------------------------------------------------------
// D f32, A and B f16; N columns, M = 128 rows; B_MN: B is MN-major.
__host__ __device__ constexpr uint32_t idesc_f16(int N, bool B_MN) {
  return (1u << 4) | (B_MN ? (1u << 16) : 0u) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
// D[tmem] = A[tmem] * B[smem] + D * 2^-LO_BITS: the step from the sum of the small products to hi.hi
__device__ __forceinline__ void mma_f16_ts_shrink(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, 1, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p, %4;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "n"(LO_BITS)
      : "memory");
}
// D[tmem] = A[smem] * B[smem] + D * 2^-LO_BITS
__device__ __forceinline__ void mma_f16_ss_shrink(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, 1, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p, %4;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "n"(LO_BITS)
      : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem]
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// D[tmem] (+)= A[smem] * B[smem]
__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// MN-major f16 operand with 128-byte swizzle: groups of eight k-rows 1024 B apart
// (SBO), panels of 64 columns `panel` bytes apart (LBO).
__device__ __forceinline__ uint64_t smem_desc_mn_sw128(uint32_t addr, uint32_t panel) {
  uint64_t d = 0;
  d |= (uint64_t)((addr >> 4) & 0x3FFFu);
  d |= (uint64_t)((panel >> 4) & 0x3FFFu) << 16;
  d |= (uint64_t)((1024u >> 4) & 0x3FFFu) << 32;
  d |= (uint64_t)1u << 46;
  d |= (uint64_t)2u << 61;
  return d;
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Untiled bulk copy, global -> shared, both 16-byte aligned.
__device__ __forceinline__ void bulk_load(uint32_t smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_dst),
      "l"(src), "r"(bytes), "r"(jxd::smem_u32(bar))
      : "memory");
}
// Whether a phase is complete.
__device__ __forceinline__ bool poll(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(jxd::smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// Bounded waits in a few instructions.  With jxg::wait_bounded and its clock at every
// wait the gradient of packed sequences took 7% longer.  Polling takes some 20 to 50
// cycles a time, so that 2^26 polls are one to two seconds.  The copies' thread may be
// suspended, for as long as the hardware likes at each try, so that its limit is a
// time: the clock is read from the 64th try on.
__device__ __forceinline__ bool wait_polling(uint64_t* bar, uint32_t parity, unsigned int* err) {
  for (uint32_t i = 0; !poll(bar, parity); ++i) {
    if (i == 1u << 26) {
      atomicOr(err, JX_DEVERR_TIMEOUT);
      return false;
    }
  }
  return true;
}
constexpr unsigned long long WAIT_NS = 4000000000ull;
// `end` (0 before the first late try) is the time at which waits that share it give up.
__device__ __forceinline__ bool wait_suspended(uint64_t* bar, uint32_t parity, unsigned int* err,
                                               unsigned long long& end, unsigned long long limit_ns = WAIT_NS) {
  for (uint32_t i = 0; !jxd::mbar_try_wait(bar, parity); ++i) {
    if (i < 64) continue;
    const unsigned long long now = jxg::global_ns();
    if (end == 0) end = now + limit_ns;
    if (now >= end) {
      atomicOr(err, JX_DEVERR_TIMEOUT);
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ bool wait_suspended(uint64_t* bar, uint32_t parity, unsigned int* err) {
  unsigned long long end = 0;
  return wait_suspended(bar, parity, err, end);
}
// A warp waits, every lane for itself: polling by one lane and telling the others
// cost 100 cycles more at each of the three to five waits of a step.
__device__ __forceinline__ void warp_wait(uint64_t* bar, uint32_t parity, bool& ok, volatile int* abort_flag,
                                          unsigned int* err) {
  uint32_t i = ok ? 0 : 1u << 26;
  while (!poll(bar, parity)) {
    if (i++ >= 1u << 26) {
      if (ok) atomicOr(err, JX_DEVERR_TIMEOUT);
      ok = false;
      *abort_flag = 1;
      break;
    }
  }
  __syncwarp();
}
__device__ __forceinline__ void pair_sync(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }

// ---- rows of a [rows, heads, dim] tensor through shared memory ----
// 256 threads move a tile of 128 rows between global memory, whole rows at a time,
// and a thread-per-row layout: an area of 128 x DP floats, the 16-byte chunk c
// of row r at r * 4 DP + ((c ^ (r & 7)) << 4), without conflicts either way.
// (Thread-per-row accesses to global memory took 5500 cycles a tile, this 1500.)
constexpr int MOVERS = 256;
__host__ __device__ constexpr int area_bytes(int DP) { return TILE * DP * 4; }  // a tile's hi and lo parts' size, too

__device__ __forceinline__ void movers_sync() { asm volatile("bar.sync 5, 256;" ::: "memory"); }
__device__ __forceinline__ bool aligned16(const void* p, int dim, long long ld) {
  return (dim & 3) == 0 && (ld & 3) == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0;
}
template <int DP>
__device__ __forceinline__ uint32_t area_at(uint32_t row, uint32_t chunk) {
  return row * (DP * 4) + ((chunk ^ (row & 7)) << 4);
}
// `src`: the tile's first row; zeros behind `rows` and `dim`.
template <int DP>
__device__ __forceinline__ void rows_load(float4 (&x)[DP / 8], const float* src, long long ld, int rows, int dim,
                                          bool vec, int tid) {
#pragma unroll
  for (int i = 0; i < DP / 8; ++i) {
    const int f = i * MOVERS + tid, r = f / (DP / 4), c = f % (DP / 4) * 4;
    x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r < rows) {
      const float* p = src + r * ld + c;
      if (vec) {
        if (c < dim) x[i] = *reinterpret_cast<const float4*>(p);
      } else {
        if (c < dim) x[i].x = p[0];
        if (c + 1 < dim) x[i].y = p[1];
        if (c + 2 < dim) x[i].z = p[2];
        if (c + 3 < dim) x[i].w = p[3];
      }
    }
  }
}
template <int DP>
__device__ __forceinline__ void rows_to_area(uint8_t* area, const float4 (&x)[DP / 8], int tid) {
#pragma unroll
  for (int i = 0; i < DP / 8; ++i) {
    const int f = i * MOVERS + tid;
    *reinterpret_cast<float4*>(area + area_at<DP>(f / (DP / 4), f % (DP / 4))) = x[i];
  }
}
// This thread's half of row `row`; returns the largest magnitude's bits.
template <int DP>
__device__ __forceinline__ uint32_t half_from_area(float (&x)[DP / 2], const uint8_t* area, int row, int half) {
  uint32_t top = 0;
#pragma unroll
  for (int c = 0; c < DP / 8; ++c) {
    const float4 f = *reinterpret_cast<const float4*>(area + area_at<DP>(row, half * (DP / 8) + c));
    x[4 * c] = f.x;
    x[4 * c + 1] = f.y;
    x[4 * c + 2] = f.z;
    x[4 * c + 3] = f.w;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = max(top, __float_as_uint(x[4 * c + i]) & 0x7fffffffu);
  }
  return top;
}
// The halves, times `factor`, and out again: dst is the tile's first row.
template <int DP>
__device__ __forceinline__ void half_to_area(uint8_t* area, const float (&x)[DP / 2], float factor, int row, int half) {
#pragma unroll
  for (int c = 0; c < DP / 8; ++c)
    *reinterpret_cast<float4*>(area + area_at<DP>(row, half * (DP / 8) + c)) =
        make_float4(x[4 * c] * factor, x[4 * c + 1] * factor, x[4 * c + 2] * factor, x[4 * c + 3] * factor);
}
template <int DP>
__device__ __forceinline__ void rows_store(float* dst, long long ld, const uint8_t* area, int rows, int dim, bool vec,
                                           int tid) {
#pragma unroll
  for (int i = 0; i < DP / 8; ++i) {
    const int f = i * MOVERS + tid, r = f / (DP / 4), c = f % (DP / 4) * 4;
    if (r < rows) {
      const float4 x = *reinterpret_cast<const float4*>(area + area_at<DP>(r, c / 4));
      float* p = dst + r * ld + c;
      if (vec) {
        if (c < dim) *reinterpret_cast<float4*>(p) = x;
      } else {
        if (c < dim) p[0] = x.x;
        if (c + 1 < dim) p[1] = x.y;
        if (c + 2 < dim) p[2] = x.z;
        if (c + 3 < dim) p[3] = x.w;
      }
    }
  }
}

// ---- the operand that stays: rows into tensor memory ----
// Two warps share 32 rows (TMEM lanes), each thread half a row.
// Stores the scaled halves' parts: hi at column `col` of tensor memory, lo DP/2 columns behind it.
template <int DP>
__device__ __forceinline__ void row_half_store(const float (&x)[DP / 2], float factor, uint32_t taddr, int half) {
  constexpr int N = DP / 4;  // packed columns of this half: 32 or 16
  uint32_t hi[N], lo[N];
#pragma unroll
  for (int c = 0; c < N; ++c) split_half(x[2 * c] * factor, x[2 * c + 1] * factor, hi[c], lo[c]);
  if constexpr (N == 32) {
    tmem_st32(taddr + half * N, hi);
    tmem_st32(taddr + DP / 2 + half * N, lo);
  } else {
    tmem_st16(taddr + half * N, hi);
    tmem_st16(taddr + DP / 2 + half * N, lo);
  }
}

// A tensor that is split into tiles.
struct TileSource {
  const float* x;
  long long ld;
  uint8_t* tiles;
  float* inverse;  // of the tile's scale, [id][head], `step` floats apart, as are norm and delta_top
  int* bad;        // the tile is marked, [id][head]
  int step;
  float* norm;     // largest Euclidean norm of the tile's rows; may be NULL
  // for dout alone (NULL otherwise): o and lse; the rows' lse in base 2 less
  // P_SHIFT (+inf for rows without keys or behind the end), rowsum(dout o), the rows'
  // norms, and over each row and the later ones of its block the largest norm and
  // the largest |rowsum(dout o)|: [id][head][TILE]
  const float* o;
  const float* lse;
  float* lse2;
  float* delta;
  float* row_norm;
  float2* later;
};
// A tile of a packed sequence, as a CTA finds it with one load: everything that the
// offsets say about it.
struct __align__(16) TileRef {
  long long q0, k0;  // of its sequence
  int lq, lk, b, jt;  // jt: the tile's index within it, or -1: no tile
};
__device__ __forceinline__ TileRef load_ref(const TileRef* p) {
  const int4 a = reinterpret_cast<const int4*>(p)[0], b = reinterpret_cast<const int4*>(p)[1];
  TileRef r;
  r.q0 = (long long)(uint32_t)a.x | ((long long)a.y << 32);
  r.k0 = (long long)(uint32_t)a.z | ((long long)a.w << 32);
  r.lq = b.x;
  r.lk = b.y;
  r.b = b.z;
  r.jt = b.w;
  return r;
}
__device__ __forceinline__ Seq seq_of(const TileRef& r) {
  Seq s;
  s.q0 = r.q0;
  s.k0 = r.k0;
  s.lq = r.lq;
  s.lk = r.lk;
  return s;
}

// One launch of split_tiles_kernel: tensors over the keys' tiles, then over the
// query rows'.
struct TileSources {
  TileSource t[4];
  int keys, queries;  // tensors of each kind
  // Order of work: tiles by falling work (query tiles by their key tiles, key tiles
  // by their query rows), the ids behind a sequence's end last.  May be NULL.  work
  // >> shift is below ORDER_KEYS.
  TileRef *order_q, *order_k;
  int shift, q_tiles, k_tiles;
};
constexpr int ORDER_KEYS = 1024;

// A launch whose CTAs may start while the last ones of the launch before it run.
template <typename... Params, typename... Args>
cudaError_t launch_overlapped(void (*kernel)(Params...), long long grid, int threads, size_t smem, cudaStream_t st,
                              const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}

// Implemented in attn_fwd.cu: one launch that splits all tensors of `src`.
int split_tiles(const Shape& s, const TileSources& src, int DP, cudaStream_t st);
int prepare_kernel(const void* kernel, int variant, size_t smem, int launch_regs);
int attention_fwd_tiles(const Shape& s, const float* q, const float* k, const float* v, float* o, float* lse,
                        cudaStream_t st);
int attention_decode(const Shape& s, const float* q, const float* k, const float* v, float* o, float* lse,
                     long long rows, cudaStream_t st);
int attention_bwd_tiles(const Shape& s, const float* q, const float* k, const float* v, const float* o,
                        const float* lse, const float* dout, float* dq, float* dk, float* dv, long long max_q,
                        cudaStream_t st);

}  // namespace jxa
