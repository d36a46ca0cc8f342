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

// Elements i, i + 1 (i even, the row 4-byte aligned at least) of a row of fp32 or 16-bit elements.
__device__ __forceinline__ float2 pg_load2(const void* row, int type, long long i) {
  if (type == PG_F32) return *reinterpret_cast<const float2*>(reinterpret_cast<const float*>(row) + i);
  if (type == PG_F16) return __half22float2(*reinterpret_cast<const __half2*>(reinterpret_cast<const __half*>(row) + i));
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(reinterpret_cast<const __nv_bfloat16*>(row) + i));
}
// One rounding of an fp32 value to `type` (fp32 or 16 bits).
__device__ __forceinline__ void pg_store(void* row, int type, long long i, float x) {
  if (type == PG_F32) reinterpret_cast<float*>(row)[i] = x;
  else if (type == PG_F16) reinterpret_cast<__half*>(row)[i] = __float2half_rn(x);
  else reinterpret_cast<__nv_bfloat16*>(row)[i] = __float2bfloat16_rn(x);
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
  int n_heads, n_kv, hd, rot, n_pos;
  int* err;
};

// 16 bytes of elements of type T as V values.
template <int T, int V>
__device__ __forceinline__ void ap_widen(const uint4& a, float (&x)[V]) {
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (T == PG_F32) {
      x[i] = __uint_as_float(w[i]);
    } else {
      const float2 f = T == PG_F16 ? __half22float2(*reinterpret_cast<const __half2*>(&w[i]))
                                   : __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
      x[(2 * i) % V] = f.x;
      x[(2 * i + 1) % V] = f.y;
    }
  }
}
// V values rounded to type T (8-bit floats saturate at 448; NaN stays NaN); p aligned to the V elements.
template <int T, int V>
__device__ __forceinline__ void ap_store(void* p, const float (&x)[V]) {
  if (T == PG_F32) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  } else if (T == PG_E4M3) {
    uint32_t w[V / 4];
#pragma unroll
    for (int i = 0; i < V / 4; ++i)
      w[i] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(x[4 * i], x[4 * i + 1]), __NV_SATFINITE, __NV_E4M3) |
             (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(x[4 * i + 2], x[4 * i + 3]), __NV_SATFINITE, __NV_E4M3) << 16;
    if (V == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[V / 4 - 1]);
    else *reinterpret_cast<uint32_t*>(p) = w[0];
  } else {
    uint32_t w[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      if (T == PG_F16) {
        const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    if (V == 8) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[V / 2 - 2], w[V / 2 - 1]);
    else *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  }
}

// Bound by memory: each source row is read and each stored row written once, in 16-byte loads. Grid
// (token, slice of its head rows); a thread owns V pairs (j, j + rot / 2), V = 16 bytes of the source type, or 2 V
// dims that do not turn, of U head rows: the rows' loads are all requested before the position is known,
// and one look at the table and the angles serves them all. 8192 tokens of 32 + 2 x 8 bf16 heads of 128: 40.2 us, 5.1
// TB/s, 0.78 of the copy rate (a row per thread 44.5); one token about 2.5 us, all of it latency.
constexpr int AP_THREADS = 128;
constexpr int AP_DEEP = 3;   // head rows per thread of a large append
template <int ST, int CT, int U>
__global__ void __launch_bounds__(AP_THREADS) k_page_append(const __grid_constant__ AppendParams P) {
  constexpr int V = ST == PG_F32 ? 4 : 8, ES = ST == PG_F32 ? 4 : 2, CS = CT == PG_E4M3 ? 1 : 2;
  pdl_wait();
  pdl_trigger();
  const int i = blockIdx.x, units = P.hd / (2 * V), u = threadIdx.x % units;   // units divides AP_THREADS
  const int r0 = (blockIdx.y * U * AP_THREADS + threadIdx.x) / units, rstep = AP_THREADS / units;
  const int rows = P.n_heads + 2 * P.n_kv, half = P.rot / 2;
  const int jt = u < half / V ? u * V : 2 * V * u, jt2 = u < half / V ? jt + half : jt + V;   // rows that turn
  const int pos = P.pos[i];
  uint4 ra[U], rb[U];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const int r = r0 + k * rstep;
    if (r < rows) {
      const bool is_q = r < P.n_heads, is_v = r >= P.n_heads + P.n_kv;
      const int h = is_q ? r : is_v ? r - P.n_heads - P.n_kv : r - P.n_heads;
      const char* src = reinterpret_cast<const char*>(is_q ? P.q : is_v ? P.v : P.k) +
                        (is_q ? i * P.q_tok + h * P.q_head : is_v ? i * P.v_tok + h * P.v_head : i * P.k_tok + h * P.k_head) * ES;
      ra[k] = *reinterpret_cast<const uint4*>(src + (is_v ? 2 * V * u : jt) * ES);
      rb[k] = *reinterpret_cast<const uint4*>(src + (is_v ? 2 * V * u + V : jt2) * ES);
    }
  }
  if (pos < 0) return;
  if (P.rot && pos >= P.n_pos) {
    atomicOr(P.err, KQ_DEV_ERR_BAD_POS);
    return;
  }
  // the page; a bad one keeps the keys and values out, the queries are still turned
  const int s = P.T.seq ? P.T.seq[i] : i, pi = pos >> P.T.page_shift;
  long long page = -1;
  if (s >= 0 && s < P.T.n_seq && pi < P.T.max_pages) page = P.T.table[s * P.T.ld + pi];
  float c[V], sn[V];
  if (u < half / V) {
#pragma unroll
    for (int x = 0; x < V; x += 4) {
      const float4 cc = *reinterpret_cast<const float4*>(P.cos_t + pos * P.rope_ld + jt + x);
      const float4 ss = *reinterpret_cast<const float4*>(P.sin_t + pos * P.rope_ld + jt + x);
      c[x] = cc.x; c[x + 1] = cc.y; c[x + 2] = cc.z; c[x + 3] = cc.w;
      sn[x] = ss.x; sn[x + 1] = ss.y; sn[x + 2] = ss.z; sn[x + 3] = ss.w;
    }
  }
  if (page < 0 || page >= P.T.n_pages) {
    if (r0 + (U - 1) * rstep >= P.n_heads)
      atomicOr(P.err, s < 0 || s >= P.T.n_seq ? KQ_DEV_ERR_BAD_ROW
                      : pi >= P.T.max_pages   ? KQ_DEV_ERR_BAD_POS
                                              : KQ_DEV_ERR_BAD_PAGE);
    page = -1;
  }
  const int row = pos & ((1 << P.T.page_shift) - 1);
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const int r = r0 + k * rstep;
    if (r >= rows) break;
    const bool is_q = r < P.n_heads, is_v = r >= P.n_heads + P.n_kv;
    const int h = is_q ? r : is_v ? r - P.n_heads - P.n_kv : r - P.n_heads;
    const int j = is_v ? 2 * V * u : jt, j2 = is_v ? j + V : jt2;
    float a[V], b[V];
    ap_widen<ST, V>(ra[k], a);
    ap_widen<ST, V>(rb[k], b);
    if (!is_v && u < half / V) {
#pragma unroll
      for (int x = 0; x < V; ++x) {
        const float p = a[x], q = b[x];
        a[x] = __fsub_rn(__fmul_rn(p, c[x]), __fmul_rn(q, sn[x]));
        b[x] = __fadd_rn(__fmul_rn(q, c[x]), __fmul_rn(p, sn[x]));
      }
    }
    if (is_q) {
      char* dst = reinterpret_cast<char*>(P.q_out) + (i * P.o_tok + h * P.o_head) * ES;
      ap_store<ST, V>(dst + j * ES, a);
      ap_store<ST, V>(dst + j2 * ES, b);
    } else if (page >= 0) {
      if (CT == PG_E4M3) {
        const float* sc = is_v ? P.vs : P.ks;
        const float scale = sc ? sc[h] : 1.f;
#pragma unroll
        for (int x = 0; x < V; ++x) {
          a[x] = __fdiv_rn(a[x], scale);
          b[x] = __fdiv_rn(b[x], scale);
        }
      }
      char* dst = reinterpret_cast<char*>(is_v ? P.vc : P.kc) +
                  (is_v ? page * P.vp + h * P.vh + row * P.vr : page * P.kp + h * P.kh + row * P.kr) * CS;
      ap_store<CT, V>(dst + j * CS, a);
      ap_store<CT, V>(dst + j2 * CS, b);
    }
  }
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
  int n, n_heads, n_kv, type, window;
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

// ---- matrix-instruction fragments. S^T = K Q^T and O^T = V^T P^T on m16n8k16 (fp16 or bf16 operands,
// fp32 accumulation): the keys (then the dims) are the 16 rows and 8 query heads of one K/V head the
// columns, so a group of up to 8 heads wastes no rows, and a thread keeps the two heads 2 t4,
// 2 t4 + 1 in every accumulator (grp = lane / 4, t4 = lane % 4).
template <bool BF>
__device__ __forceinline__ void pa_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void pa_ldsm(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void pa_ldsm_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t pa_trans(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ void pa_cp16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// 2^x to 2 ulp (the instruction's documented error); results below 2^-126 are 0.
__device__ __forceinline__ float pa_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two e4m3 bytes (the low half of x) as fp16; exact.
__device__ __forceinline__ uint32_t pa_e4m3x2(uint32_t x) {
  uint32_t d;
  asm volatile("{\n .reg .b16 t;\n cvt.u16.u32 t, %1;\n cvt.rn.f16x2.e4m3x2 %0, t;\n}\n" : "=r"(d) : "r"(x));
  return d;
}
// N 16-bit terms whose sum is (a, b) to N * 11 (fp16) or N * 8 (bf16) bits, largest first.
template <bool BF, int N>
__device__ __forceinline__ void pa_split(float a, float b, uint32_t (&t)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float x, y;
    if (BF) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
      t[i] = *reinterpret_cast<const uint32_t*>(&h);
      x = __bfloat162float(h.x);
      y = __bfloat162float(h.y);
    } else {
      const __half2 h = __floats2half2_rn(a, b);
      t[i] = *reinterpret_cast<const uint32_t*>(&h);
      x = __half2float(h.x);
      y = __half2float(h.y);
    }
    if (i + 1 < N) {
      a = __fsub_rn(a, x);
      b = __fsub_rn(b, y);
    }
  }
}

constexpr int PA_WARPS = 4;
constexpr int PA_SUB = 16;                     // keys of one warp's step: within one page, whose size is a multiple of 16
constexpr int PA_TILE = PA_WARPS * PA_SUB;     // the unit the work is divided in
constexpr int PA_MAX_CTAS = 148 * 2;           // CTAs of one launch, and partial slots (two each) of the scratch
constexpr int PA_MAX_HEADS = 16;               // query heads of one K/V head a CTA takes at once

template <int CT, int HD, int NT, bool PREC>
struct PaShape {
  static constexpr bool BF = CT == PG_BF16;
  static constexpr int ES = CT == PG_E4M3 ? 1 : 2;
  static constexpr int HEADS = 8 * NT;
  static constexpr int ROW = HD * ES, LD = ROW + 16;           // odd multiples of 16 bytes: conflict-free ldmatrix rows
  static constexpr int KV = 2 * PA_SUB * LD;                   // K and V rows of one step of a warp
  static constexpr int QX = HEADS * (HD + 8) * 4;              // a segment's query rows, or a warp's (o, m, l) rows
  static constexpr int STAGE = KV > QX ? KV : QX;              // a ring slot holds any of the three
  static constexpr int KS = HD / 16;
  static constexpr int NQ = PREC ? (BF ? 3 : 2) : 1;           // terms of a query element
  static constexpr int NP = PREC ? (BF ? 3 : 2) : 2;           // terms of a softmax weight
  static constexpr bool QREG = KS * NQ * NT * 2 <= 64;         // query fragments in registers, else in shared memory
  static constexpr int QBYTES = QREG ? 0 : KS * NQ * NT * 256;
  static constexpr int MLD = HD + 4;                           // row of the warps' exchange: o, m, l
  // CTAs per SM: three of shallower rings measured slower (one 4K sequence 15.4 against 13.5 us, 64 x 32K 845 against 809)
  static constexpr int PER_SM = STAGE > 12000 ? 1 : 2;
  static constexpr int FIT = (226 * 1024 / PER_SM - 4608 - QBYTES) / (PA_WARPS * STAGE);
  static constexpr int STAGES = FIT > 8 ? 8 : FIT;
  static_assert(STAGES >= 2, "a ring of two slots at least");
  static constexpr int SMEM = PA_WARPS * STAGES * STAGE + QBYTES;
};
constexpr int PA_JOIN = 16;                    // partials of a chain read at once (24, 32: more code, not faster)
constexpr int PA_COST = 3;                     // what a (sequence, head) costs beside its tiles, in tiles (128 ragged
                                               // sequences at 1 / 2 / 3 / 5: 90 / 72 / 68 / 71 us)
constexpr int PA_PLD = 256 + 4;                // floats of a scratch row (the widest head_dim)

struct AttendScratch {
  float* part;      // [2 * PA_MAX_CTAS][PA_MAX_HEADS][PA_PLD]: o, m, l of a CTA's first (0) and last (1) segment
  int* ticket;      // [PA_MAX_CTAS], zero between launches
};

// a / b of non-negative numbers, in 32 bits where both fit (the common case; a 64-bit division is slow).
__device__ __forceinline__ long long pa_div(long long a, long long b) {
  return ((a | b) >> 32) == 0 ? (long long)((uint32_t)a / (uint32_t)b) : a / b;
}

// A cursor over a CTA's run: the units of (sequence, virtual head) are PA_COST empty ones and its tiles.
struct PaCursor {
  int seq, head, at, tiles, t0, t1;   // at: unit in the segment; [t0, t1): the run's tiles of this segment
  long long seg, left;                // first unit of the segment, units left of the run
  KeyRange R;
};

// Bound by memory where runs are long: 64 sequences of 8K to 32K keys (fp16, 32/8 heads of 128) 785 to 839 us,
// 5.9 to 6.3 TB/s of K/V, 0.90 to 0.96 of the copy rate; 128 sequences of 9 to 4096 keys 65 to 69 us (floor 49); by
// latency where they are short: one sequence of 4096 keys 13.2 us (lengths, table, keys, two steps and the
// join follow one another; a step costs about 1.1 us of a warp's dependent instructions).
// The work is cut into equal runs of units, one per CTA, in the order sequence, head, 64-key tile,
// wherever sequences end: CTAs finish together whatever the lengths are (cut by tiles alone, the CTAs
// with many short sequences were 4 times behind the others). A CTA walks its run segment by segment
// (one sequence and head at a time). Each warp owns a ring of slots and fills it STAGES - 1 steps
// ahead, across segment borders: a segment's query rows first, then its steps of 16 keys, so nothing
// but the last slots of a run is waited for in full. A segment that is a whole (sequence, head) is
// written out; otherwise its (o, m, l) goes to the scratch and the last CTA of the chain to arrive
// joins the chain's partials in CTA order, so the sums' order is fixed.
template <int CT, int HD, int NT, bool PREC>
__global__ void __launch_bounds__(PA_WARPS * 32, PaShape<CT, HD, NT, PREC>::PER_SM)
k_page_attend(const __grid_constant__ AttendParams P, const AttendScratch W) {
  using S = PaShape<CT, HD, NT, PREC>;
  constexpr bool BF = S::BF, E8 = CT == PG_E4M3;
  constexpr int KS = S::KS, NQ = S::NQ, NP = S::NP;
  constexpr float PSCALE = BF ? 1.f : 16384.f;   // fp16 weights use 2^14 .. 2^-24: 38 bits below the largest
  extern __shared__ __align__(128) uint8_t pa_smem[];
  __shared__ __align__(16) float4 s_sum[PA_WARPS * 32];
  __shared__ float2 s_ml[PA_WARPS * 32];
  __shared__ long long s_start;
  __shared__ KeyRange s_keys;
  __shared__ int s_tiles;
  __shared__ long long s_scan[PA_WARPS];
  __shared__ int s_seq, s_last;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, grp = lane >> 2, t4 = lane & 3;
  const int G = P.n_heads / P.n_kv, HT = (G + S::HEADS - 1) / S::HEADS, H = P.n_kv * HT;

  pdl_wait();      // everything below may read what the kernels before this one wrote
  pdl_trigger();   // the next kernel may be scheduled as CTAs leave (it waits for this grid's end itself)
  auto tiles_of = [&](int i, KeyRange& R) {
    R = pg_keys(P, i, false);
    return R.last > R.first ? (R.last - (R.first & ~(PA_SUB - 1)) + PA_TILE - 1) / PA_TILE : 0;
  };
  auto units_of = [&](int i) {
    KeyRange R;
    const int t = tiles_of(i, R);
    return t ? t + PA_COST : 0;
  };
  // ---- where this CTA's run begins: a scan of the sequences' units, consecutive ones per thread
  const int per = (P.n + PA_WARPS * 32 - 1) / (PA_WARPS * 32), i0 = min(P.n, tid * per), i1 = min(P.n, i0 + per);
  long long mine = 0;
  for (int i = i0; i < i1; ++i) {
    if (blockIdx.x == 0) pg_keys(P, i, true);
    mine += units_of(i);
  }
  long long incl = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += v;
  }
  if (lane == 31) s_scan[warp] = incl;
  __syncthreads();
  long long before = incl - mine, total = 0;
#pragma unroll
  for (int w = 0; w < PA_WARPS; ++w) {
    if (w < warp) before += s_scan[w];
    total += s_scan[w];
  }
  total *= H;
  const long long run = pa_div(total + gridDim.x - 1, gridDim.x);
  const long long begin = min(total, blockIdx.x * run), end = min(total, begin + run);
  if (begin < end && before * H <= begin && begin < (before + mine) * H) {
    long long b = before;
    for (int i = i0; i < i1; ++i) {
      KeyRange R;
      const int t = tiles_of(i, R), u = t ? t + PA_COST : 0;
      if (begin < (b + u) * H) {
        s_seq = i;
        s_start = b * H;
        s_keys = R;
        s_tiles = t;
        break;
      }
      b += u;
    }
  }
  // rows without a key: zeros
  for (int i = blockIdx.x; i < P.n; i += gridDim.x) {
    if (units_of(i)) continue;
    for (int e = tid; e < P.n_heads * HD; e += PA_WARPS * 32)
      pg_store(P.out, P.type, i * P.o_tok + (e / HD) * P.o_head + e % HD, 0.f);
  }
  __syncthreads();
  if (begin >= end) return;

  // the run's tiles of the segment under the cursor; none if the run ends before its first
  auto settle = [&](PaCursor& c) {
    c.t0 = max(0, c.at - PA_COST);
    c.t1 = (int)min((long long)(c.tiles + PA_COST), c.at + c.left) - PA_COST;
    if (c.t1 <= c.t0) c.left = 0;
  };
  auto next_segment = [&](PaCursor& c) {
    c.left -= c.t1 + PA_COST - c.at;
    c.at = 0;
    c.seg += c.tiles + PA_COST;
    if (c.left > 0 && ++c.head == H) {
      c.head = 0;
      do c.tiles = tiles_of(++c.seq, c.R);
      while (c.tiles == 0);
    }
    settle(c);
  };
  PaCursor cur;
  cur.seq = s_seq;
  cur.tiles = s_tiles;
  cur.R = s_keys;
  cur.head = (int)pa_div(begin - s_start, cur.tiles + PA_COST);
  cur.seg = s_start + (long long)cur.head * (cur.tiles + PA_COST);
  cur.at = (int)(begin - cur.seg);
  cur.left = end - begin;
  settle(cur);

  // ---- the ring's loader
  const uint32_t ring = smem_u32(pa_smem) + warp * S::STAGES * S::STAGE;
  constexpr int CH = S::ROW / 16, NCP = S::ROW / 32;   // 16-byte chunks of a row; a lane's chunks of 16 rows
  constexpr int RSTEP = 32 / CH;                       // rows between a lane's chunks
  const int lr = lane / CH, lc = lane % CH;
  const int q_es = P.type == PG_F32 ? 4 : 2, q_ld = HD * q_es + 32;
  PaCursor ld = cur;
  int ld_tile = ld.t0 - 1;                             // t0 - 1: the query rows
  uint32_t pages_ok = 0;                               // one bit per slot: its page exists
  int slot = 0, fill = 0;
  // of the loader's segment: this lane's place in row 0 of its head, the table row; and of the next step
  // its first key; and the page ids of 32 steps, a lane each, requested together when the segment begins:
  // no copy waits for the table on its own
  const char *kseg = nullptr, *vseg = nullptr;
  const int* tseg = nullptr;
  int ld_key = 0, ld_pages = -1;
  auto request_pages = [&]() {   // of the steps from the current one on
    const int t = max(ld_tile, ld.t0) + lane, key = (ld.R.first & ~(PA_SUB - 1)) + t * PA_TILE + warp * PA_SUB;
    ld_pages = t < ld.t1 && key < ld.R.last ? tseg[key >> P.T.page_shift] : -1;
  };
  auto begin_segment = [&]() {
    const int kv = ld.head / HT;
    kseg = reinterpret_cast<const char*>(P.kc) + (kv * P.kh + lr * P.kr) * S::ES + lc * 16;
    vseg = reinterpret_cast<const char*>(P.vc) + (kv * P.vh + lr * P.vr) * S::ES + lc * 16;
    tseg = P.T.table + ld.R.row * P.T.ld;
    ld_key = (ld.R.first & ~(PA_SUB - 1)) + ld.t0 * PA_TILE + warp * PA_SUB;
    ld_tile = ld.t0 - 1;
    request_pages();
  };
  if (ld.left > 0) begin_segment();
  auto load = [&]() {
    const uint32_t dst = ring + fill * S::STAGE;
    if (ld.left > 0) {
      if (ld_tile < ld.t0) {
        const int kv = ld.head / HT;
        const int h0 = kv * G + (ld.head % HT) * S::HEADS, nh = min(S::HEADS, (kv + 1) * G - h0), qc = HD * q_es / 16;
        const char* q = reinterpret_cast<const char*>(P.q) + (ld.seq * P.q_tok + h0 * P.q_head) * q_es;
        for (int e = lane; e < nh * qc; e += 32) {
          const int h = e / qc, c = e % qc;
          pa_cp16(dst + h * q_ld + c * 16, q + h * P.q_head * q_es + c * 16, 16u);
        }
      } else {
        const int step_of = ld_tile - ld.t0;
        if (step_of > 0 && (step_of & 31) == 0) request_pages();
        const int ld_page = __shfl_sync(0xffffffffu, ld_pages, step_of & 31);
        if (ld_key < ld.R.last) {
          const bool ok = ld_page >= 0 && ld_page < P.T.n_pages;
          pages_ok = (pages_ok & ~(1u << fill)) | ((uint32_t)ok << fill);
          if (!ok && lane == 0) atomicOr(P.err, KQ_DEV_ERR_BAD_PAGE);
          const int row = ld_key & ((1 << P.T.page_shift) - 1);
          const char* ks = kseg + (ok ? (ld_page * P.kp + row * P.kr) * S::ES : 0);
          const char* vs = vseg + (ok ? (ld_page * P.vp + row * P.vr) * S::ES : 0);
          const uint32_t d = dst + lr * S::LD + lc * 16;
          if (ok && ld_key >= ld.R.first && ld_key + PA_SUB <= ld.R.last) {
#pragma unroll
            for (int c = 0; c < NCP; ++c) {
              pa_cp16(d + c * RSTEP * S::LD, ks + c * RSTEP * P.kr * S::ES, 16u);
              pa_cp16(d + c * RSTEP * S::LD + PA_SUB * S::LD, vs + c * RSTEP * P.vr * S::ES, 16u);
            }
          } else {
#pragma unroll
            for (int c = 0; c < NCP; ++c) {
              const int t = ld_key + lr + c * RSTEP;
              const bool in = ok && t >= ld.R.first && t < ld.R.last;   // rows outside are not read: they may hold anything
              pa_cp16(d + c * RSTEP * S::LD, in ? ks + c * RSTEP * P.kr * S::ES : (const char*)P.kc, in ? 16u : 0u);
              pa_cp16(d + c * RSTEP * S::LD + PA_SUB * S::LD, in ? vs + c * RSTEP * P.vr * S::ES : (const char*)P.vc, in ? 16u : 0u);
            }
          }
        }
        ld_key += PA_TILE;
      }
      if (++ld_tile == ld.t1) {
        next_segment(ld);
        if (ld.left > 0) begin_segment();
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    fill = fill + 1 == S::STAGES ? 0 : fill + 1;
  };
#pragma unroll 1
  for (int s = 0; s < S::STAGES - 1; ++s) load();
  // waits for the next slot, keeps the ring filled, and returns the slot
  auto step = [&]() {
    asm volatile("cp.async.wait_group %0;" ::"n"(S::STAGES - 2) : "memory");
    __syncwarp();   // every lane's copies are here, and every lane has left the slot that load() fills
    const int now = slot;
    slot = slot + 1 == S::STAGES ? 0 : slot + 1;
    load();
    return now;
  };

  uint2* qs = reinterpret_cast<uint2*>(pa_smem + (S::SMEM - S::QBYTES));
  const int mi = lane >> 3, ml = lane & 7;
  const uint32_t k_off = (uint32_t)(((mi & 1) * 8 + ml) * S::LD + (mi >> 1) * 16);
  const uint32_t v_off = (uint32_t)(E8 ? ((mi & 1) * 8 + ml) * S::LD + (mi >> 1) * 16 : ((mi >> 1) * 8 + ml) * S::LD + (mi & 1) * 16) +
                         PA_SUB * S::LD;
  while (cur.left > 0) {
    const int kv = cur.head / HT, h0 = kv * G + (cur.head % HT) * S::HEADS, nh = min(S::HEADS, (kv + 1) * G - h0);
    // ---- query fragments (column grp of each 8 heads), scaled to [2^9, 2^10) by a power of two
    const uint8_t* qrow = pa_smem + warp * S::STAGES * S::STAGE + step() * S::STAGE;
    uint32_t qf[S::QREG ? NQ : 1][S::QREG ? NT : 1][S::QREG ? KS : 1][2];
    float sc[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int hh = nt * 8 + grp;
      const void* q = qrow + min(hh, nh - 1) * q_ld;
      float mx = 0.f;
#pragma unroll
      for (int d = 2 * t4; d < HD; d += 8) {
        const float2 a = pg_load2(q, P.type, d);
        mx = fmaxf(mx, fmaxf(fabsf(a.x), fabsf(a.y)));
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      int e = 0;
      if (mx > 0.f && mx < INFINITY) e = max(-100, (int)((__float_as_uint(mx) >> 23) & 255u) - 127);
      const float up = __uint_as_float((uint32_t)(127 + 9 - e) << 23);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        if (!S::QREG && (ks & 3) != warp) continue;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          // the dims of k indices 2 t4, 2 t4 + 1 (+ 8): 8-bit K fragments hold dims 4 t4 .. 4 t4 + 3
          const int d = 16 * ks + (E8 ? 4 * t4 + 2 * half : 2 * t4 + 8 * half);
          uint32_t t[NQ];
          const float2 a = hh < nh ? pg_load2(q, P.type, d) : make_float2(0.f, 0.f);
          pa_split<BF, NQ>(a.x * up, a.y * up, t);
#pragma unroll
          for (int j = 0; j < NQ; ++j) {
            if (S::QREG) qf[j][nt][ks][half] = t[j];
            else reinterpret_cast<uint32_t*>(qs + ((j * NT + nt) * KS + ks) * 32 + lane)[half] = t[j];
          }
        }
      }
      const float f = P.scale * 1.4426950408889634f * (P.ks ? P.ks[kv] : 1.f);
      const int ea = __shfl_sync(0xffffffffu, e, 8 * t4), eb = __shfl_sync(0xffffffffu, e, 8 * t4 + 4);
      sc[nt][0] = f * __uint_as_float((uint32_t)(127 - 9 + ea) << 23);
      sc[nt][1] = f * __uint_as_float((uint32_t)(127 - 9 + eb) << 23);
    }
    if (!S::QREG) __syncthreads();

    float o[KS][NT][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int d = 0; d < KS; ++d) o[d][nt][0] = o[d][nt][1] = o[d][nt][2] = o[d][nt][3] = 0.f;
    }
    int key = (cur.R.first & ~(PA_SUB - 1)) + cur.t0 * PA_TILE + warp * PA_SUB, now = 0;
    for (int tile = cur.t0; tile < cur.t1; ++tile, key += PA_TILE) {
      const bool ok_now = (pages_ok >> slot) & 1u;
      now = step();
      if (key >= cur.R.last) continue;
      const uint32_t kb = ring + now * S::STAGE + k_off, vb = ring + now * S::STAGE + v_off;
      // ---- scores: the terms of the queries in accumulators of their own, smallest added first
      float s[NQ][NT][4];
#pragma unroll
      for (int j = 0; j < NQ; ++j)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[j][nt][0] = s[j][nt][1] = s[j][nt][2] = s[j][nt][3] = 0.f;
      auto score = [&](int ks, const uint32_t (&a)[4]) {
#pragma unroll
        for (int j = 0; j < NQ; ++j)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            if (S::QREG) pa_mma<BF>(s[j][nt], a, qf[j][nt][ks][0], qf[j][nt][ks][1]);
            else {
              const uint2 b = qs[((j * NT + nt) * KS + ks) * 32 + lane];
              pa_mma<BF>(s[j][nt], a, b.x, b.y);
            }
          }
      };
      if (E8) {
#pragma unroll
        for (int ks = 0; ks < KS; ks += 2) {
          uint32_t r[4];
          pa_ldsm(kb + ks * 16, r);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t a[4] = {pa_e4m3x2(r[2 * j]), pa_e4m3x2(r[2 * j + 1]), pa_e4m3x2(r[2 * j] >> 16),
                                   pa_e4m3x2(r[2 * j + 1] >> 16)};
            score(ks + j, a);
          }
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          uint32_t a[4];
          pa_ldsm(kb + ks * 32, a);
          score(ks, a);
        }
      }
      // ---- online softmax, in powers of two: rows (keys) grp and grp + 8, heads 2 t4 and 2 t4 + 1
      const bool va = ok_now && key + grp >= cur.R.first && key + grp < cur.R.last;
      const bool vb8 = ok_now && key + grp + 8 >= cur.R.first && key + grp + 8 < cur.R.last;
      uint32_t pf[NP][NT][2];
      float f[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          // an infinite key makes the leading term's sum infinite and a zero lower term's sum NaN
          float a = s[NQ - 1][nt][e];
#pragma unroll
          for (int j = NQ - 2; j >= 0; --j)
            a = j > 0 || fabsf(s[0][nt][e]) < INFINITY ? __fadd_rn(a, s[j][nt][e]) : s[0][nt][e];
          x[e] = (e < 2 ? va : vb8) ? __fmul_rn(a, sc[nt][e & 1]) : -INFINITY;
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float mx = fmaxf(x[c], x[c + 2]);
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          const float mn = fmaxf(m[nt][c], mx), u = mn == -INFINITY ? 0.f : mn;
          f[nt][c] = pa_exp2(m[nt][c] - u);
          m[nt][c] = mn;
          x[c] = pa_exp2(x[c] - u) * PSCALE;
          x[c + 2] = pa_exp2(x[c + 2] - u) * PSCALE;
          l[nt][c] = __fmaf_rn(l[nt][c], f[nt][c], x[c] + x[c + 2]);
        }
        uint32_t ta[NP], tb[NP];
        pa_split<BF, NP>(x[0], x[1], ta);
        pa_split<BF, NP>(x[2], x[3], tb);
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          pf[j][nt][0] = pa_trans(ta[j]);
          pf[j][nt][1] = pa_trans(tb[j]);
        }
      }
      // ---- O^T += V^T P^T: a step's product is summed apart and added in fp32 (the matrix units cut
      // off low bits when they add to a large accumulator; over thousands of steps that would show)
      auto accumulate = [&](int d, const uint32_t (&a)[4]) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = NP - 1; j >= 0; --j) pa_mma<BF>(t, a, pf[j][nt][0], pf[j][nt][1]);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[d][nt][e] = __fmaf_rn(o[d][nt][e], f[nt][e & 1], t[e]);
        }
      };
      if (E8) {
        // a 32-bit word of the transposed fragment: dims 2 grp, 2 grp + 1 of keys 2 t4 (low half) and 2 t4 + 1
#pragma unroll
        for (int d = 0; d < KS; d += 2) {
          uint32_t r[4];
          pa_ldsm_t(vb + d * 16, r);   // keys 0-7, 8-15 of 16 dims, then of the next 16
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t lo = r[2 * j], hi = r[2 * j + 1];
            const uint32_t a[4] = {pa_e4m3x2(__byte_perm(lo, 0, 0x4420)), pa_e4m3x2(__byte_perm(lo, 0, 0x4431)),
                                   pa_e4m3x2(__byte_perm(hi, 0, 0x4420)), pa_e4m3x2(__byte_perm(hi, 0, 0x4431))};
            accumulate(d + j, a);
          }
        }
      } else {
#pragma unroll
        for (int d = 0; d < KS; ++d) {
          uint32_t a[4];
          pa_ldsm_t(vb + d * 32, a);
          accumulate(d, a);
        }
      }
    }
    // ---- join the warps: (o, m, l) rows through the slots just read
    __syncwarp();
    auto xrow = [&](int w, int h) {
      return reinterpret_cast<float*>(pa_smem + (w * S::STAGES + now) * S::STAGE) + h * S::MLD;
    };
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float ls = l[nt][c];
        ls += __shfl_xor_sync(0xffffffffu, ls, 4);
        ls += __shfl_xor_sync(0xffffffffu, ls, 8);
        ls += __shfl_xor_sync(0xffffffffu, ls, 16);
        float* row = xrow(warp, nt * 8 + 2 * t4 + c);
        if (grp == 0) {
          row[HD] = m[nt][c];
          row[HD + 1] = ls;
        }
#pragma unroll
        for (int d = 0; d < KS; ++d) {
          row[16 * d + (E8 ? 2 * grp : grp)] = o[d][nt][c];
          row[16 * d + (E8 ? 2 * grp + 1 : grp + 8)] = o[d][nt][c + 2];
        }
      }
    }
    __syncthreads();
    const bool whole = cur.t0 == 0 && cur.t1 == cur.tiles;
    float* part = W.part + (size_t)(2 * blockIdx.x + (cur.t0 == 0 ? 1 : 0)) * PA_MAX_HEADS * PA_PLD;
    const float vscale = P.vs ? P.vs[kv] : 1.f;
    for (int e = tid; e < nh * HD; e += PA_WARPS * 32) {
      const int h = e / HD, d = e % HD;
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < PA_WARPS; ++w) M = fmaxf(M, xrow(w, h)[HD]);
      const float u = M == -INFINITY ? 0.f : M;
      float L = 0.f, O = 0.f;
#pragma unroll
      for (int w = 0; w < PA_WARPS; ++w) {
        const float* row = xrow(w, h);
        const float wt = pa_exp2(row[HD] - u);
        L = __fmaf_rn(wt, row[HD + 1], L);
        O = __fmaf_rn(wt, row[d], O);
      }
      if (whole) {
        pg_store(P.out, P.type, cur.seq * P.o_tok + (h0 + h) * P.o_head + d, L == 0.f ? 0.f : __fdiv_rn(O, L) * vscale);
      } else {
        __stcg(part + h * PA_PLD + d, O);
        if (d == 0) {
          __stcg(part + h * PA_PLD + HD, M);
          __stcg(part + h * PA_PLD + HD + 1, L);
        }
      }
    }
    if (!whole) {
      const int c0 = (int)pa_div(cur.seg + PA_COST, run), c1 = (int)pa_div(cur.seg + PA_COST + cur.tiles - 1, run);
      __threadfence();
      __syncthreads();
      if (tid == 0) s_last = atomicAdd(&W.ticket[c0], 1) == c1 - c0;
      __syncthreads();
      if (s_last) {
        __threadfence();
        // float4 columns of the output, PA_JOIN partials of a column requested at a time (a round trip to
        // the L2 each, which is what a join costs); the chain's rows split over the thread groups that a
        // narrow segment leaves idle
        const int nc = c1 - c0 + 1, cols = nh * (HD / 4);
        const int groups = cols < PA_WARPS * 32 ? PA_WARPS * 32 / cols : 1, per_group = (nc + groups - 1) / groups;
        float M, L;
        float4 O;
        auto column = [&](int e, int ca, int cb) {
          const float* base = W.part + (size_t)(e / (HD / 4)) * PA_PLD;
          const int d4 = e % (HD / 4);
          M = -INFINITY;
          L = 0.f;
          O = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int c = ca; c < cb; c += PA_JOIN) {
            float4 v[PA_JOIN];
            float2 s2[PA_JOIN];
            float mx = M;
#pragma unroll
            for (int j = 0; j < PA_JOIN; ++j) {
              const float* row = base + (size_t)(2 * (c0 + c + j) + (c + j == 0)) * PA_MAX_HEADS * PA_PLD;
              const bool in = c + j < cb;
              v[j] = in ? __ldcg(reinterpret_cast<const float4*>(row) + d4) : make_float4(0.f, 0.f, 0.f, 0.f);
              s2[j] = in ? __ldcg(reinterpret_cast<const float2*>(row + HD)) : make_float2(-INFINITY, 0.f);
            }
#pragma unroll
            for (int j = 0; j < PA_JOIN; ++j) mx = fmaxf(mx, s2[j].x);
            const float u = mx == -INFINITY ? 0.f : mx, f = pa_exp2(M - u);
            M = mx;
            L *= f;
            O.x *= f; O.y *= f; O.z *= f; O.w *= f;
#pragma unroll
            for (int j = 0; j < PA_JOIN; ++j) {
              const float wt = pa_exp2(s2[j].x - u);
              L = __fmaf_rn(wt, s2[j].y, L);
              O.x = __fmaf_rn(wt, v[j].x, O.x); O.y = __fmaf_rn(wt, v[j].y, O.y);
              O.z = __fmaf_rn(wt, v[j].z, O.z); O.w = __fmaf_rn(wt, v[j].w, O.w);
            }
          }
        };
        auto write = [&](int e) {
          const float r[4] = {O.x, O.y, O.z, O.w};
          const long long at = cur.seq * P.o_tok + (h0 + e / (HD / 4)) * P.o_head + 4 * (e % (HD / 4));
#pragma unroll
          for (int x = 0; x < 4; ++x) pg_store(P.out, P.type, at + x, L == 0.f ? 0.f : __fdiv_rn(r[x], L) * vscale);
        };
        if (groups == 1) {
          for (int e = tid; e < cols; e += PA_WARPS * 32) {
            column(e, 0, nc);
            write(e);
          }
        } else {
          const int e = tid % cols, gi = tid / cols;
          if (gi < groups) column(e, min(nc, gi * per_group), min(nc, (gi + 1) * per_group));
          if (gi > 0 && gi < groups) {
            s_sum[tid] = O;
            s_ml[tid] = make_float2(M, L);
          }
          __syncthreads();
          if (gi == 0) {
            for (int x = 1; x < groups; ++x) {
              const float4 v = s_sum[x * cols + e];
              const float2 s2 = s_ml[x * cols + e];
              const float mx = fmaxf(M, s2.x), u = mx == -INFINITY ? 0.f : mx, f = pa_exp2(M - u), wt = pa_exp2(s2.x - u);
              M = mx;
              L = __fmaf_rn(wt, s2.y, L * f);
              O.x = __fmaf_rn(wt, v.x, O.x * f); O.y = __fmaf_rn(wt, v.y, O.y * f);
              O.z = __fmaf_rn(wt, v.z, O.z * f); O.w = __fmaf_rn(wt, v.w, O.w * f);
            }
            write(e);
          }
        }
        if (tid == 0) W.ticket[c0] = 0;
      }
    }
    __syncthreads();   // the exchange slots are free again
    next_segment(cur);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

}  // namespace kq
