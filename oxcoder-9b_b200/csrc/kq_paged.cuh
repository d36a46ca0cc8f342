// kq_paged.cuh -- a paged K/V cache: appending rotated keys and values (k_page_append) and the
// attention of one new token per sequence over it (k_page_attend). include/kq.h has the formulas.
//
// Page layout: element (page, kv head, row, dim) at page * p + head * h + row * r + dim, dims dense,
// rows on 16-byte boundaries. Element offsets are 64-bit: a cache of many pages passes 2^31 elements.
#pragma once
#include "kq_common.cuh"
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cfloat>

namespace kq {

enum : int { PG_F32 = 0, PG_F16 = 1, PG_BF16 = 2, PG_E4M3 = 3 };   // KQ_F32 .. KQ_E4M3

// x[0] of a row of elements of `type`, as fp32.
__device__ __forceinline__ float pg_load(const void* row, int type, long long i) {
  if (type == PG_F32) return reinterpret_cast<const float*>(row)[i];
  if (type == PG_F16) return __half2float(reinterpret_cast<const __half*>(row)[i]);
  if (type == PG_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(row)[i]);
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(reinterpret_cast<const __nv_fp8_storage_t*>(row)[i], __NV_E4M3)));
}
// One rounding of an fp32 value to `type` (8-bit floats saturate at 448; NaN stays NaN).
__device__ __forceinline__ void pg_store(void* row, int type, long long i, float x) {
  if (type == PG_F32) reinterpret_cast<float*>(row)[i] = x;
  else if (type == PG_F16) reinterpret_cast<__half*>(row)[i] = __float2half_rn(x);
  else if (type == PG_BF16) reinterpret_cast<__nv_bfloat16*>(row)[i] = __float2bfloat16_rn(x);
  else reinterpret_cast<__nv_fp8_storage_t*>(row)[i] = __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
}

struct PageTable {
  const int* table;          // [n_seq][max_pages]
  const int* seq;            // [n] or null
  long long ld;
  int n_seq, max_pages, n_pages, page_shift;
};

// ------------------------------------------------------------------------------ append
struct AppendParams {
  const void *k, *v, *q;
  void *q_out, *kc, *vc;
  long long k_tok, k_head, v_tok, v_head, q_tok, q_head, o_tok, o_head;
  long long kp, kh, kr, vp, vh, vr;      // cache strides
  const float *ks, *vs;
  PageTable T;
  const int* pos;
  const float *cos_t, *sin_t;
  long long rope_ld;
  int n_heads, n_kv, hd, src_type, cache_type, rot, n_pos;
  int* err;
};

// Grid (token, head row): one CTA turns one head row; thread j its pairs (j, j + rot / 2) and dims.
__global__ void __launch_bounds__(128) k_page_append(const __grid_constant__ AppendParams P) {
  const int i = blockIdx.x, r = blockIdx.y, half = P.rot / 2;
  const int pos = P.pos[i];
  if (pos < 0) return;
  if (P.rot && pos >= P.n_pos) {
    if (threadIdx.x == 0) atomicOr(P.err, KQ_DEV_ERR_BAD_POS);
    return;
  }
  const bool is_q = r < P.n_heads, is_v = r >= P.n_heads + P.n_kv;
  const int h = is_q ? r : is_v ? r - P.n_heads - P.n_kv : r - P.n_heads;
  const void* src = is_q ? P.q : is_v ? P.v : P.k;
  const long long so = is_q ? i * P.q_tok + h * P.q_head : is_v ? i * P.v_tok + h * P.v_head : i * P.k_tok + h * P.k_head;
  void* dst = P.q_out;
  long long d0 = i * P.o_tok + h * P.o_head;
  int type = P.src_type;
  float scale = 1.f;
  if (!is_q) {
    const int s = P.T.seq ? P.T.seq[i] : i, pi = pos >> P.T.page_shift;
    if (s < 0 || s >= P.T.n_seq || pi >= P.T.max_pages) {
      if (threadIdx.x == 0) atomicOr(P.err, s < 0 || s >= P.T.n_seq ? KQ_DEV_ERR_BAD_ROW : KQ_DEV_ERR_BAD_POS);
      return;
    }
    const int page = P.T.table[s * P.T.ld + pi];
    if (page < 0 || page >= P.T.n_pages) {
      if (threadIdx.x == 0) atomicOr(P.err, KQ_DEV_ERR_BAD_PAGE);
      return;
    }
    const int row = pos & ((1 << P.T.page_shift) - 1);
    dst = is_v ? P.vc : P.kc;
    d0 = is_v ? page * P.vp + h * P.vh + row * P.vr : page * P.kp + h * P.kh + row * P.kr;
    type = P.cache_type;
    const float* sc = is_v ? P.vs : P.ks;
    if (sc) scale = sc[h];
  }
  const int rot = is_v ? 0 : half;
  for (int j = threadIdx.x; j < rot; j += blockDim.x) {
    const float a = pg_load(src, P.src_type, so + j), b = pg_load(src, P.src_type, so + j + half);
    const float c = P.cos_t[pos * P.rope_ld + j], s = P.sin_t[pos * P.rope_ld + j];
    pg_store(dst, type, d0 + j, __fdiv_rn(__fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s)), scale));
    pg_store(dst, type, d0 + j + half, __fdiv_rn(__fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s)), scale));
  }
  for (int j = 2 * rot + threadIdx.x; j < P.hd; j += blockDim.x)
    pg_store(dst, type, d0 + j, __fdiv_rn(pg_load(src, P.src_type, so + j), scale));
}

// ------------------------------------------------------------------------------ attention
struct AttendParams {
  const void* q;
  void* out;
  long long q_tok, q_head, o_tok, o_head;
  const void *kc, *vc;
  long long kp, kh, kr, vp, vh, vr;
  const float *ks, *vs;
  PageTable T;
  const int* len;
  int n, n_heads, n_kv, type, cache_type, window;
  float scale;
  int* err;
};

// The keys of token i: [first, last) of table row `row` (row < 0: none).
struct KeyRange { int row, first, last; };
__device__ __forceinline__ KeyRange pg_keys(const AttendParams& P, int i, bool report) {
  KeyRange R = {P.T.seq ? P.T.seq[i] : i, 0, 0};
  if (R.row < 0 || R.row >= P.T.n_seq) {
    if (report) atomicOr(P.err, KQ_DEV_ERR_BAD_ROW);
    R.row = -1;
    return R;
  }
  const long long cap = (long long)P.T.max_pages << P.T.page_shift;
  int n = max(P.len[i], 0);
  if (n > cap) {
    if (report) atomicOr(P.err, KQ_DEV_ERR_BAD_LEN);
    n = (int)cap;
  }
  R.first = P.window > 0 ? max(0, n - P.window) : 0;
  R.last = n;
  return R;
}

// Grid (token, query head), 4 warps: a warp takes every fourth key, a lane HD / 32 dims; online
// softmax per warp, the warps joined in order.
template <int HD>
__global__ void __launch_bounds__(128) k_page_attend(const __grid_constant__ AttendParams P) {
  constexpr int D = HD / 32;
  const int i = blockIdx.x, h = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = h / (P.n_heads / P.n_kv);
  __shared__ float s_m[4], s_l[4], s_o[4][HD];
  const KeyRange R = pg_keys(P, i, threadIdx.x == 0);
  float q[D], o[D], m = -INFINITY, l = 0.f;
  const float scale = P.scale * (P.ks ? P.ks[g] : 1.f);
#pragma unroll
  for (int d = 0; d < D; ++d) {
    q[d] = pg_load(P.q, P.type, i * P.q_tok + h * P.q_head + D * lane + d);
    o[d] = 0.f;
  }
  for (int t = R.first + warp; t < R.last; t += 4) {
    const int page = P.T.table[R.row * P.T.ld + (t >> P.T.page_shift)], row = t & ((1 << P.T.page_shift) - 1);
    if (page < 0 || page >= P.T.n_pages) {
      if (lane == 0) atomicOr(P.err, KQ_DEV_ERR_BAD_PAGE);
      continue;
    }
    const long long k0 = page * P.kp + g * P.kh + row * P.kr, v0 = page * P.vp + g * P.vh + row * P.vr;
    float s = 0.f;
#pragma unroll
    for (int d = 0; d < D; ++d) s = __fmaf_rn(q[d], pg_load(P.kc, P.cache_type, k0 + D * lane + d), s);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    s *= scale;
    const float mn = fmaxf(m, s), u = mn == -INFINITY ? 0.f : mn, f = expf(m - u), p = expf(s - u);
    m = mn;
    l = __fmaf_rn(l, f, p);
#pragma unroll
    for (int d = 0; d < D; ++d) o[d] = __fmaf_rn(o[d], f, p * pg_load(P.vc, P.cache_type, v0 + D * lane + d));
  }
  if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
#pragma unroll
  for (int d = 0; d < D; ++d) s_o[warp][D * lane + d] = o[d];
  __syncthreads();
  float M = -INFINITY, L = 0.f, w[4];
  for (int x = 0; x < 4; ++x) M = fmaxf(M, s_m[x]);
  for (int x = 0; x < 4; ++x) {
    w[x] = s_m[x] == -INFINITY && !(s_l[x] != 0.f) ? 0.f : expf(s_m[x] - (M == -INFINITY ? 0.f : M));
    L = __fmaf_rn(w[x], s_l[x], L);
  }
  const float vs = P.vs ? P.vs[g] : 1.f;
  for (int d = threadIdx.x; d < HD; d += blockDim.x) {
    float v = 0.f;
    for (int x = 0; x < 4; ++x)
      if (w[x] != 0.f) v = __fmaf_rn(w[x], s_o[x][d], v);
    pg_store(P.out, P.type, i * P.o_tok + h * P.o_head + d, L == 0.f ? 0.f : __fdiv_rn(v, L) * vs);
  }
}

}  // namespace kq
