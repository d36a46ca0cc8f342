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

// The penalties in the definition's order, every operation rounded on its own.
__device__ __forceinline__ float rl_penalise(float z, uint32_t seen, float rep, float freq, float pres) {
  if (seen) z = z > 0.f ? __fdiv_rn(z, rep) : __fmul_rn(z, rep);
  const uint32_t c = seen & 0x7fffffffu;
  return __fsub_rn(z, __fadd_rn(__fmul_rn(freq, (float)c), __fmul_rn(pres, c ? 1.f : 0.f)));
}

constexpr int RL_THREADS = 512, RL_SLICE = 4096;

// One CTA per row: slices of RL_SLICE ids in turn, each with its counts (bit 31: seen in the prompt)
// and its last bias entry built in shared memory from the whole history and list.
template <typename T>
__global__ void __launch_bounds__(RL_THREADS) k_logit_rules(const __grid_constant__ RuleParams P) {
  __shared__ uint32_t s_cnt[RL_SLICE], s_own[RL_SLICE];
  __shared__ float s_v[RL_THREADS / 32];
  __shared__ int s_i[RL_THREADS / 32];
  const int i = blockIdx.x, tid = threadIdx.x;
  pdl_wait();
  pdl_trigger();
  const T* in = reinterpret_cast<const T*>(P.in) + i * P.in_ld;
  T* out = reinterpret_cast<T*>(P.out) + i * P.out_ld;
  const int nh = P.hist ? min(max(P.hist_len[i], 0), P.max_hist) : 0;
  const int np = P.prompt_len ? P.prompt_len[i] : 0;
  const float rep = P.rep ? P.rep[i] : 1.f, freq = P.freq ? P.freq[i] : 0.f, pres = P.pres ? P.pres[i] : 0.f;
  int mrow = P.mask ? (P.mask_row ? P.mask_row[i] : i) : -1;
  const bool none = P.mask && (mrow < -1 || mrow >= P.n_masks);
  if (none) {
    if (tid == 0) atomicOr(P.err, KQ_DEV_ERR_BAD_ROW);
    mrow = -1;
  }
  float bv = -INFINITY;
  int bi = 0x7fffffff;
  for (int v0 = 0; v0 < P.vocab; v0 += RL_SLICE) {
    for (int j = tid; j < RL_SLICE; j += RL_THREADS) s_cnt[j] = s_own[j] = 0;
    __syncthreads();
    for (int j = tid; j < nh; j += RL_THREADS) {
      const int id = P.hist[i * P.hist_ld + j];
      if (id < 0 || id >= P.vocab || id < v0 || id - v0 >= RL_SLICE) continue;
      if (j < np) atomicOr(&s_cnt[id - v0], 0x80000000u);
      else atomicAdd(&s_cnt[id - v0], 1u);
    }
    for (int j = tid; j < P.n_bias; j += RL_THREADS) {
      const int id = P.bias_id[i * P.bias_ld + j];
      if (id >= 0 && id < P.vocab && id >= v0 && id - v0 < RL_SLICE) atomicMax(&s_own[id - v0], (uint32_t)j + 1u);
    }
    __syncthreads();
    for (int j = tid; j < RL_SLICE && v0 + j < P.vocab; j += RL_THREADS) {
      const int id = v0 + j;
      float z = rl_penalise(rl_get<T>(in[id]), s_cnt[j], rep, freq, pres);
      if (s_own[j]) z = __fadd_rn(z, P.bias[i * P.bias_ld + s_own[j] - 1]);
      if (none || (mrow >= 0 && !((P.mask[mrow * P.mask_ld + (id >> 5)] >> (id & 31)) & 1u))) z = -INFINITY;
      const T r = rl_put<T>(z);
      out[id] = r;
      const float x = rl_get<T>(r);
      if (x > bv) { bv = x; bi = id; }
    }
    __syncthreads();
  }
  if (!P.best) return;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    const float ov = __shfl_xor_sync(0xffffffffu, bv, off);
    const int oi = __shfl_xor_sync(0xffffffffu, bi, off);
    if (ov > bv || (ov == bv && oi < bi)) { bv = ov; bi = oi; }
  }
  if ((tid & 31) == 0) { s_v[tid >> 5] = bv; s_i[tid >> 5] = bi; }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < RL_THREADS / 32; ++w)
      if (s_v[w] > bv || (s_v[w] == bv && s_i[w] < bi)) { bv = s_v[w]; bi = s_i[w]; }
    P.best[i] = bi == 0x7fffffff ? -1 : bi;
  }
}

}  // namespace kq
