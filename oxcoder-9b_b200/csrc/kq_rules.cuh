// kq_rules.cuh -- rules on logits: penalties for repeated tokens, biases, grammar masks, and the
// greedy id of each row. include/kq.h has the formulas.
#pragma once
#include "kq_common.cuh"
#include <cuda_bf16.h>

namespace kq {

struct RuleParams {
  const void* in;
  void* out;
  long long in_ld, out_ld;
  int* best;
  const int* hist;
  const int *hist_len, *prompt_len;
  long long hist_ld;
  const float *rep, *freq, *pres;
  const int* bias_id;
  const float* bias;
  long long bias_ld;
  const uint32_t* mask;
  const int* mask_row;
  long long mask_ld;
  int n, vocab, max_hist, n_bias, n_masks;
  int span;                  // ids of a row that one CTA of its cluster owns, a multiple of 16
  int* err;
};

template <typename T> __device__ __forceinline__ float rl_get(T x);
template <> __device__ __forceinline__ float rl_get<float>(float x) { return x; }
template <> __device__ __forceinline__ float rl_get<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float rl_get<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T rl_put(float x);
template <> __device__ __forceinline__ float rl_put<float>(float x) { return x; }
template <> __device__ __forceinline__ __half rl_put<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 rl_put<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// The penalties in the definition's order, every operation rounded on its own; `seen`: bit 31 the id is
// in the prompt, below it its count after the prompt. An id that is not in the history keeps its bits.
__device__ __forceinline__ float rl_penalise(float z, uint32_t seen, float rep, float freq, float pres) {
  if (!seen) return z;
  z = z > 0.f ? __fdiv_rn(z, rep) : __fmul_rn(z, rep);
  const uint32_t c = seen & 0x7fffffffu;
  return __fsub_rn(z, __fadd_rn(__fmul_rn(freq, (float)c), __fmul_rn(pres, c ? 1.f : 0.f)));
}

__device__ __forceinline__ uint32_t rl_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t rl_ranks() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void rl_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address of this CTA's shared variable p in the CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t rl_at(const void* p, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ void rl_add(uint32_t a, uint32_t v) {
  asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}
__device__ __forceinline__ void rl_or(uint32_t a, uint32_t v) {
  asm volatile("red.relaxed.cluster.shared::cluster.or.b32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}
__device__ __forceinline__ void rl_max(uint32_t a, uint32_t v) {
  asm volatile("red.relaxed.cluster.shared::cluster.max.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}

constexpr int RL_THREADS = 512, RL_PRE = 5, RL_CLUSTER = 16;

// Bound by memory: a row is read and written once. A cluster of CTAs owns a row, a CTA `span`
// consecutive ids of it, with a count and the last bias entry of each id in its shared memory. The
// history and the bias list are scanned once per row, each CTA a part, the hits sent to the owner's
// shared memory (integer adds and maxima: their order does not matter). The CTA's logits and mask
// words are requested into registers before that, RL_PRE 16-byte groups a thread, so the scan runs
// under their latency. Positions count from the 16-byte boundary at or below the row's start
// (u = id + shift), so rows of any alignment take 16-byte groups; only a row's ends are handled singly.
template <typename T>
__global__ void __launch_bounds__(RL_THREADS, 2) k_logit_rules(const __grid_constant__ RuleParams P) {
  constexpr int VEC = 16 / (int)sizeof(T);
  extern __shared__ __align__(16) uint32_t rl_smem[];
  __shared__ float s_v[RL_THREADS / 32], s_cv[RL_CLUSTER];
  __shared__ int s_i[RL_THREADS / 32], s_ci[RL_CLUSTER];
  const int tid = threadIdx.x, rank = (int)rl_rank(), ranks = (int)rl_ranks(), i = blockIdx.x / ranks, span = P.span;
  uint32_t* cnt = rl_smem;
  uint32_t* last = rl_smem + (P.hist ? span : 0);
  pdl_wait();
  pdl_trigger();
  const T* in = reinterpret_cast<const T*>(P.in) + i * P.in_ld;
  T* out = reinterpret_cast<T*>(P.out) + i * P.out_ld;
  const int shift = (int)((reinterpret_cast<uintptr_t>(in) / sizeof(T)) % VEC);
  const bool vec = (int)((reinterpret_cast<uintptr_t>(out) / sizeof(T)) % VEC) == shift;
  const int u_begin = rank * span, u_end = min(u_begin + span, P.vocab + shift);
  int mrow = P.mask ? (P.mask_row ? P.mask_row[i] : i) : -1;
  const bool none = P.mask && (mrow < -1 || mrow >= P.n_masks);
  if (none) {
    if (tid == 0) atomicOr(P.err, KQ_DEV_ERR_BAD_ROW);
    mrow = -1;
  }
  const uint32_t* mask = mrow >= 0 ? P.mask + mrow * P.mask_ld : nullptr;
  const int words = (P.vocab + 31) >> 5;
  // group k of this thread: positions [u, u + VEC); whole: it lies inside the row and both rows are aligned alike
  auto group = [&](int k) { return u_begin + (k * RL_THREADS + tid) * VEC; };
  auto whole = [&](int u) { return vec && u >= shift && u + VEC <= u_end; };
  auto request = [&](int u, uint4& x, uint32_t& m0, uint32_t& m1) {
    if (whole(u)) x = *reinterpret_cast<const uint4*>(in + (u - shift));
    m0 = m1 = 0xffffffffu;
    if (mask && u < u_end) {
      const int w = max(u - shift, 0) >> 5;
      m0 = mask[w];
      m1 = w + 1 < words ? mask[w + 1] : 0u;
    }
  };
  uint4 x[RL_PRE];
  uint32_t m0[RL_PRE], m1[RL_PRE];
#pragma unroll
  for (int k = 0; k < RL_PRE; ++k) request(group(k), x[k], m0[k], m1[k]);

  const int nh = P.hist ? min(max(P.hist_len[i], 0), P.max_hist) : 0;
  const int np = P.prompt_len ? P.prompt_len[i] : 0;
  const bool scan = nh > 0 || P.n_bias > 0;   // the same in all CTAs of the row
  if (scan) {
    const int fields = (P.hist ? span : 0) + (P.n_bias ? span : 0);   // span is a multiple of 4
    for (int j = tid; j < fields / 4; j += RL_THREADS) reinterpret_cast<uint4*>(rl_smem)[j] = make_uint4(0, 0, 0, 0);
    rl_cluster_sync();                        // every CTA's fields are zero
    const int* hist = P.hist + i * P.hist_ld;
    for (int j = rank * RL_THREADS + tid; j < nh; j += ranks * RL_THREADS) {
      const int id = hist[j];
      if (id < 0 || id >= P.vocab) continue;
      const uint32_t u = (uint32_t)(id + shift), r = u / (uint32_t)span, a = rl_at(cnt + (u - r * span), r);
      if (j < np) rl_or(a, 0x80000000u);
      else rl_add(a, 1u);
    }
    for (int j = rank * RL_THREADS + tid; j < P.n_bias; j += ranks * RL_THREADS) {
      const int id = P.bias_id[i * P.bias_ld + j];
      if (id < 0 || id >= P.vocab) continue;
      const uint32_t u = (uint32_t)(id + shift), r = u / (uint32_t)span;
      rl_max(rl_at(last + (u - r * span), r), (uint32_t)j + 1u);
    }
    rl_cluster_sync();                        // every hit has arrived
  }

  const float rep = P.rep ? P.rep[i] : 1.f, freq = P.freq ? P.freq[i] : 0.f, pres = P.pres ? P.pres[i] : 0.f;
  float bv = -INFINITY;
  int bi = 0x7fffffff;
  auto value = [&](float z, int u, bool allowed) {
    if (scan) {
      if (P.hist) z = rl_penalise(z, cnt[u - u_begin], rep, freq, pres);
      if (P.n_bias) {
        const uint32_t e = last[u - u_begin];
        if (e) z = __fadd_rn(z, P.bias[i * P.bias_ld + e - 1]);
      }
    }
    return allowed && !none ? z : -INFINITY;
  };
  auto offer = [&](T r, int u) {
    const float f = rl_get<T>(r);
    if (f > bv) { bv = f; bi = u - shift; }
  };
  auto process = [&](int u, const uint4& v, uint32_t w0, uint32_t w1) {
    if (u >= u_end) return;
    const int id0 = u - shift;                // below 0 only in a row's first group
    if (whole(u)) {
      const uint32_t ok = (id0 & 31) ? __funnelshift_r(w0, w1, id0 & 31) : w0;
      union { uint4 q; T t[VEC]; } y;
      y.q = v;
      uint32_t any = 0;                       // does a count or a bias touch the group?
      if (scan) {
#pragma unroll
        for (int j = 0; j < VEC; j += 4) {
          if (P.hist) {
            const uint4 c = *reinterpret_cast<const uint4*>(cnt + (u - u_begin) + j);
            any |= c.x | c.y | c.z | c.w;
          }
          if (P.n_bias) {
            const uint4 c = *reinterpret_cast<const uint4*>(last + (u - u_begin) + j);
            any |= c.x | c.y | c.z | c.w;
          }
        }
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const bool allowed = (ok >> j) & 1u;
        if (any) y.t[j] = rl_put<T>(value(rl_get<T>(y.t[j]), u + j, allowed));
        else if (!allowed || none) y.t[j] = rl_put<T>(-INFINITY);
        offer(y.t[j], u + j);
      }
      *reinterpret_cast<uint4*>(out + id0) = y.q;
      return;
    }
    for (int p = max(u, shift); p < min(u + VEC, u_end); ++p) {
      const int id = p - shift;
      const T r = rl_put<T>(value(rl_get<T>(in[id]), p, !mask || ((mask[id >> 5] >> (id & 31)) & 1u)));
      out[id] = r;
      offer(r, p);
    }
  };
#pragma unroll
  for (int k = 0; k < RL_PRE; ++k) process(group(k), x[k], m0[k], m1[k]);
  for (int k = RL_PRE; group(k) < u_end; ++k) {
    request(group(k), x[0], m0[0], m1[0]);
    process(group(k), x[0], m0[0], m1[0]);
  }
  if (!P.best) return;
  // ---- the greedy id: warp, CTA, cluster; equal values: the lowest id
  auto better = [&](float v, int j) {
    if (v > bv || (v == bv && j < bi)) { bv = v; bi = j; }
  };
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) better(__shfl_xor_sync(0xffffffffu, bv, off), __shfl_xor_sync(0xffffffffu, bi, off));
  if ((tid & 31) == 0) { s_v[tid >> 5] = bv; s_i[tid >> 5] = bi; }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < RL_THREADS / 32; ++w) better(s_v[w], s_i[w]);
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(rl_at(&s_cv[rank], 0)), "f"(bv) : "memory");
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(rl_at(&s_ci[rank], 0)), "r"(bi) : "memory");
  }
  rl_cluster_sync();
  if (rank == 0 && tid == 0) {
    bv = -INFINITY;
    bi = 0x7fffffff;
    for (int r = 0; r < ranks; ++r) better(s_cv[r], s_ci[r]);
    P.best[i] = bi == 0x7fffffff ? -1 : bi;
  }
}

}  // namespace kq
