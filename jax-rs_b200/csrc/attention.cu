// attention.cu -- scaled dot-product attention over packed sequences with
// grouped heads, forward and backward.
//
//   nn::scaled_dot_product_attention / multi_head_attention src/nn.rs:1460,1556
//   (CPU loops over one sequence, untraced)
//
//   forward   x = scale q k^T, o = softmax(x) v, lse = log(sum exp(x))
//   backward  p = exp(x - lse), dv = p^T do, ds = p (do v^T - rowsum(do o)),
//             dq = scale ds k, dk = scale ds^T q
#include <algorithm>

#include "attn_tc.cuh"

namespace {

using namespace jxa;

constexpr int ROW_WARPS = 8;

// One warp per (query row, head).
__global__ void __launch_bounds__(32 * ROW_WARPS) attn_rows_dq_kernel(const __grid_constant__ Shape s,
                                                                     const float* __restrict__ q,
                                                                     const float* __restrict__ k,
                                                                     const float* __restrict__ v,
                                                                     const float* __restrict__ o,
                                                                     const float* __restrict__ lse,
                                                                     const float* __restrict__ dout, float* dq) {
  const long long w = (long long)blockIdx.x * ROW_WARPS + (threadIdx.x >> 5);
  const long long t = w / s.heads;
  const int h = (int)(w - t * s.heads);
  if (t >= s.total_q) return;
  const int b = seq_of_row(s.cu_q, s.batch, t);
  const Seq sq = seq_bounds(s, b);
  if (t < sq.q0 || t >= sq.q0 + sq.lq) return;
  const long long hk = h / s.group, hd = (long long)h * s.dim;
  row_dq(q + t * s.ldq + hd, k + sq.k0 * s.ldk + hk * s.dim, v + sq.k0 * s.ldv + hk * s.dim, o + t * s.ldo + hd,
         dout + t * s.ldo + hd, lse[(long long)h * s.total_q + t], dq + t * s.ldq + hd,
         sq.visible((int)(t - sq.q0), s.causal), s.dim, s.ldk, s.ldv, s.scale);
}

// One warp per (key row, key head).
__global__ void __launch_bounds__(32 * ROW_WARPS) attn_rows_dkv_kernel(const __grid_constant__ Shape s,
                                                                      const float* __restrict__ q,
                                                                      const float* __restrict__ k,
                                                                      const float* __restrict__ v,
                                                                      const float* __restrict__ o,
                                                                      const float* __restrict__ lse,
                                                                      const float* __restrict__ dout, float* dk,
                                                                      float* dv) {
  const long long w = (long long)blockIdx.x * ROW_WARPS + (threadIdx.x >> 5);
  const long long t = w / s.kv_heads;
  const int hk = (int)(w - t * s.kv_heads);
  if (t >= s.total_k) return;
  const int b = seq_of_row(s.cu_k, s.batch, t);
  const Seq sq = seq_bounds(s, b);
  if (t < sq.k0 || t >= sq.k0 + sq.lk) return;
  const long long hd = (long long)hk * s.dim, h0 = (long long)hk * s.group;
  row_dkv(q + sq.q0 * s.ldq + h0 * s.dim, o + sq.q0 * s.ldo + h0 * s.dim, dout + sq.q0 * s.ldo + h0 * s.dim,
          lse + h0 * s.total_q + sq.q0, k + t * s.ldk + hd, v + t * s.ldv + hd, dk + t * s.ldk + hd,
          dv + t * s.ldv + hd, sq.first_row((int)(t - sq.k0), s.causal), sq.lq, s.group, s.dim, s.ldq, s.ldo,
          s.total_q, s.scale);
}

// Whether the tensor-core kernels or the plain-f32 rings take a forward call, from
// the hints, in microseconds as measured at dim 128: the rings read K and V once
// for every 32 query rows of a key head, 18 us and about 1 ns a key and head each
// time (0.25 ns at 4 rows: HBM's rate); the tiles cost 2.3 us per 128 keys for each wave of
// (query tile, head) CTAs, and the split of K and V 0.4 ns a key and head.
// (4 sequences of 8192 keys, 64 heads on 1: rings 83, tiles 248; 1000 keys x 8, 20
// rows, 16 heads: 140 and 101; 2048 keys x 4, 64 rows a head: 91 and 68.  The figures
// rest on few shapes; at dim 64 the first takes 73 and 181, and 700 and 1500 keys, 8 rows, 16
// heads on 4 of dim 40 19 and 26.)
bool tiles_are_faster(const Shape& s, int64_t max_q, int64_t max_k) {
  const double rows = (double)max_q * s.group;
  if (rows <= 16 || tiles_mostly_empty(s, false)) return false;
  if (rows > 128) return true;
  const double keys = (double)s.total_k * s.kv_heads;
  const double ctas = (double)s.batch * s.heads * ((max_q + 127) / 128);
  const double waves = ceil(ctas / jx::num_sms());
  const double rings = ceil(rows / 32) * (18 + keys * 1e-3);
  const double tiles = 20 + 2.3 * waves * (double)((max_k + 127) / 128) + keys * 0.4e-3;
  return tiles < rings;
}

// Whether the gradients are computed row by row (two launches, a warp per row and head)
// or by tiles (two, or three where key tiles are few), from the hints, in
// microseconds as measured: a row's warp takes 0.3 us a key, a key's 0.72 us a row of its
// heads, each besides what all of them together cost; the tiles' cost is their
// launches and 0.14 us a CTA.  (8 heads, 8 rows and keys: 12 and 16; 16 of
// each: 19 and 16; 16 sequences, 32 heads on 8, 8 of each: 39 and 94; 1 row behind
// 128 keys: 173 and 99.)
// Tiles that would be mostly empty, and more than the scratch can hold, leave the call to the rows.
bool rows_are_faster(const Shape& s, int64_t max_q, int64_t max_k) {
  if (tiles_mostly_empty(s, true)) return true;
  const double rows = (double)max_q * s.group, keys = (double)max_k, heads = (double)s.batch * s.heads;
  const double by_row =
      6 + 0.72 * rows + 0.3 * keys + 0.3e-3 * heads * (double)max_q * keys + 6e-3 * (double)s.total_k * s.kv_heads;
  return by_row < 15 + (s.group > 1 ? 8 : 0) + 0.14 * heads;
}

// Waits for a barrier that nothing completes, `waits` times with one time to give up.
__global__ void wait_selftest_kernel(int waits, unsigned long long limit_ns, unsigned int* err, int* given_up,
                                     unsigned long long* ns) {
  __shared__ uint64_t bar;
  jxd::mbar_init(&bar, 1);
  const unsigned long long start = jxg::global_ns();
  unsigned long long end = 0;
  for (int i = 0; i < waits; ++i) *given_up += !wait_suspended(&bar, 0, err, end, limit_ns);
  *ns = jxg::global_ns() - start;
}

int check_shape(const char* what, Shape& s, const int32_t* cu_q, const int32_t* cu_k, int64_t batch, int64_t total_q,
                int64_t total_k, int64_t max_q, int64_t max_k, int64_t heads, int64_t kv_heads, int64_t head_dim,
                int64_t ldq, int64_t ldk, int64_t ldv, int64_t ldo, float scale, int causal) {
  JX_REQUIRE(batch >= 0 && batch < (1 << 24), "%s: batch must be in [0, 2^24)", what);
  JX_REQUIRE(total_q >= 0 && total_q < (1LL << 31) && total_k >= 0 && total_k < (1LL << 31),
             "%s: total_q and total_k must be in [0, 2^31)", what);
  JX_REQUIRE(max_q >= 0 && max_k >= 0, "%s: max_q and max_k must not be negative", what);
  JX_REQUIRE(heads >= 1 && kv_heads >= 1 && heads <= 65535 && heads % kv_heads == 0,
             "%s: heads must be a multiple of kv_heads (and at most 65535)", what);
  JX_REQUIRE(head_dim >= 1 && head_dim <= MAX_DIM, "%s: head_dim must be in [1, %d]", what, MAX_DIM);
  JX_REQUIRE(ldq >= heads * head_dim && ldo >= heads * head_dim && ldk >= kv_heads * head_dim &&
                 ldv >= kv_heads * head_dim,
             "%s: row stride smaller than the row", what);
  JX_REQUIRE(isfinite(scale), "%s: scale must be finite", what);
  s.cu_q = cu_q;
  s.cu_k = cu_k;
  s.batch = (int)batch;
  s.heads = (int)heads;
  s.kv_heads = (int)kv_heads;
  s.group = (int)(heads / kv_heads);
  s.dim = (int)head_dim;
  s.total_q = total_q;
  s.total_k = total_k;
  s.ldq = ldq;
  s.ldk = ldk;
  s.ldv = ldv;
  s.ldo = ldo;
  s.scale = scale;
  s.causal = causal != 0;
  return JX_OK;
}

}  // namespace

extern "C" {

int jx_attention_f32(const float* q, const float* k, const float* v, float* o, float* lse, const int32_t* cu_q,
                     const int32_t* cu_k, int64_t batch, int64_t total_q, int64_t total_k, int64_t max_q,
                     int64_t max_k, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t ldq, int64_t ldk,
                     int64_t ldv, int64_t ldo, float scale, int causal, jx_stream_t stream) {
  JX_TRACE("jx_attention_f32");
  Shape s;
  if (int rc = check_shape("attention", s, cu_q, cu_k, batch, total_q, total_k, max_q, max_k, heads, kv_heads,
                           head_dim, ldq, ldk, ldv, ldo, scale, causal))
    return rc;
  if (batch == 0 || total_q == 0) return JX_OK;
  JX_REQUIRE(q && o && cu_q && cu_k && (total_k == 0 || (k && v)), "attention: NULL pointer");
  JX_REQUIRE(o != q && o != k && o != v, "attention: o must not be an input");
  cudaStream_t st = jx::as_stream(stream);
  if (!(s.err = jx::device_error_word())) return jx::fail(JX_ENOMEM, "device error word unavailable");
  JX_REQUIRE(total_q * heads < (1LL << 31), "attention: too many rows");
  max_q = std::min(max_q, total_q);
  max_k = std::min(max_k, total_k);
  if (total_k == 0) return attention_decode(s, q, k, v, o, lse, 1, st);  // its last launch writes rows without keys
  if (tiles_are_faster(s, max_q, max_k)) return attention_fwd_tiles(s, q, k, v, o, lse, st);
  return attention_decode(s, q, k, v, o, lse, max_q * s.group, st);
}

int jx_attention_bwd_f32(const float* q, const float* k, const float* v, const float* o, const float* lse,
                         const float* dout, float* dq, float* dk, float* dv, const int32_t* cu_q, const int32_t* cu_k,
                         int64_t batch, int64_t total_q, int64_t total_k, int64_t max_q, int64_t max_k, int64_t heads,
                         int64_t kv_heads, int64_t head_dim, int64_t ldq, int64_t ldk, int64_t ldv, int64_t ldo,
                         float scale, int causal, jx_stream_t stream) {
  JX_TRACE("jx_attention_bwd_f32");
  Shape s;
  if (int rc = check_shape("attention_bwd", s, cu_q, cu_k, batch, total_q, total_k, max_q, max_k, heads, kv_heads,
                           head_dim, ldq, ldk, ldv, ldo, scale, causal))
    return rc;
  if (batch == 0 || (total_q == 0 && total_k == 0)) return JX_OK;
  JX_REQUIRE(cu_q && cu_k, "attention_bwd: NULL pointer");
  JX_REQUIRE(total_q == 0 || (q && o && lse && dout && dq), "attention_bwd: NULL pointer");
  JX_REQUIRE(total_k == 0 || (k && v && dk && dv), "attention_bwd: NULL pointer");
  {  // dk and dv are computed while dq is written, and the other way round
    const float *in[] = {q, k, v, o, dout, lse}, *out[] = {dq, dk, dv};
    for (int i = 0; i < 3; ++i) {
      for (const float* x : in) JX_REQUIRE(!out[i] || out[i] != x, "attention_bwd: a gradient must not be an input");
      JX_REQUIRE(!out[i] || out[i] != out[(i + 1) % 3], "attention_bwd: the gradients must be different tensors");
    }
  }
  cudaStream_t st = jx::as_stream(stream);
  if (!(s.err = jx::device_error_word())) return jx::fail(JX_ENOMEM, "device error word unavailable");
  max_q = std::min(max_q, total_q);
  max_k = std::min(max_k, total_k);
  if (total_q > 0 && total_k > 0 && !rows_are_faster(s, max_q, max_k))
    return attention_bwd_tiles(s, q, k, v, o, lse, dout, dq, dk, dv, max_q, st);
  const long long bq = (total_q * heads + ROW_WARPS - 1) / ROW_WARPS;
  const long long bk = (total_k * kv_heads + ROW_WARPS - 1) / ROW_WARPS;
  JX_REQUIRE(bq < (1LL << 31) && bk < (1LL << 31), "attention_bwd: too many rows");
  if (bq) attn_rows_dq_kernel<<<(unsigned)bq, 32 * ROW_WARPS, 0, st>>>(s, q, k, v, o, lse, dout, dq);
  if (bk) attn_rows_dkv_kernel<<<(unsigned)bk, 32 * ROW_WARPS, 0, st>>>(s, q, k, v, o, lse, dout, dk, dv);
  JX_LAUNCH_CHECK("attention_bwd kernels");
  return JX_OK;
}

int jx_selftest_wait_timeout(int timeout_ms, int waits, int* timed_out, float* waited_ms) {
  JX_TRACE("jx_selftest_wait_timeout");
  JX_REQUIRE(timed_out && waited_ms && timeout_ms >= 1 && timeout_ms <= 1000 && waits >= 1 && waits <= 64,
             "jx_selftest_wait_timeout: 1..1000 ms, 1..64 waits");
  unsigned int* err = jx::device_error_word();
  if (!err) return jx::fail(JX_ENOMEM, "device error word unavailable");
  void* buf = nullptr;
  JX_CUDA(cudaMalloc(&buf, 16));
  cudaError_t e = cudaMemset(buf, 0, 16);
  if (e == cudaSuccess) {
    wait_selftest_kernel<<<1, 1>>>(waits, timeout_ms * 1000000ull, err, reinterpret_cast<int*>(buf) + 2,
                                   static_cast<unsigned long long*>(buf));
    e = cudaGetLastError();
  }
  if (e == cudaSuccess) e = cudaDeviceSynchronize();
  struct {
    unsigned long long ns;
    int given_up;
  } h = {};
  if (e == cudaSuccess) e = cudaMemcpy(&h, buf, 12, cudaMemcpyDeviceToHost);
  cudaFree(buf);
  if (e != cudaSuccess) return jx::check_cuda(e, "wait self-test");
  *timed_out = h.given_up;
  *waited_ms = (float)(h.ns * 1e-6);
  return JX_OK;
}

}  // extern "C"
