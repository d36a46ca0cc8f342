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
  int span;                  // ids of a row that one CTA of its cluster owns: whole turns
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
// The cluster's first barrier phase, in two halves: arrived at as the kernel starts, waited for before the first
// access to another CTA's shared memory, which may be touched only once that CTA runs.
__device__ __forceinline__ void rl_started() { asm volatile("barrier.cluster.arrive.relaxed.aligned;"); }
__device__ __forceinline__ void rl_all_started() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
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

constexpr int RL_THREADS = 512;
constexpr int RL_CLUSTER = 16;       // CTAs of a row at most
constexpr int RL_BYTES = 76 * 1024;  // of counts a CTA holds at most if it may: two CTAs per SM
constexpr int RL_BATCH = 2;          // 16-byte groups of logits a thread requests ahead (4 or 6: more code, slower)
constexpr int RL_TOUCH = 2048;       // touched ids a CTA lists; where there are more it goes through its counts
constexpr int RL_LIST = 512;         // bias entries of a CTA's ids that it keeps; a longer list is read again, an entry per thread
static_assert(RL_LIST == RL_THREADS, "the kept entries' places serve as a thread's slot each");
constexpr int RL_LOCAL = 16384;      // histories up to here are scanned by every CTA of the row

// Counts of a CTA's ids in shared memory: 16 bits an id, or 32 where histories may be longer. Beside the
// count: the id is in the prompt, has a bias.
template <bool LONG>
struct RlCount {
  using type = uint16_t;
  static constexpr uint32_t PROMPT = 0x8000u, BIASED = 0x4000u, MOST = 0x3fffu;
};
template <>
struct RlCount<true> {
  using type = uint32_t;
  static constexpr uint32_t PROMPT = 0x80000000u, BIASED = 0x40000000u, MOST = 0x3fffffffu;
};

// Bound by memory: a row is read and written once. A small cluster of CTAs owns a row, its ids dealt out
// in turns of RL_THREADS 16-byte groups (the frequent ids of a vocabulary lie together: consecutive
// shares gave one CTA of each row most of the touched ids). First the CTA counts its ids' occurrences
// in shared memory: a short history is scanned by every CTA of the row (16 KB from the L2 each, no
// barrier between CTAs), a long one (over RL_LOCAL) by its parts, with the hits sent to the owner's
// shared memory. The first to count an id lists it. Then the CTA's logits stream through registers,
// RL_BATCH groups of 16 bytes a thread ahead (the first batch flies during the scan): mask, write, pick
// among the untouched; and last the listed ids, a thread each. (Touched ids handled within the stream
// cost every warp their whole latency at almost every step.) Counts are integer adds and the last
// bias entry is a maximum, so nothing depends on the order of arrival.
// Positions count from the 16-byte boundary at or below the row's start (u = id + shift), so a row whose input and
// output lie alike moves in 16-byte groups wherever it starts, the groups over its ends element by
// element; where they lie differently (an odd vocabulary into a padded output) the whole row does.
// Measured: 128 fp32 rows of 151936 with histories of up to 4096 tokens, 300 biases and masks 49.4 us (3.2
// TB/s read and written; the copy rate would take 23.8: two waves of CTAs, each counting before it
// streams); in the stream 124, one CTA per row 240, clusters of 16 with the logits held meanwhile 109
// to 119 (a cluster waits until 16 slots of one GPC are free). One row 6.9 us.
template <typename T, bool LONG>
__global__ void __launch_bounds__(RL_THREADS, 2) k_logit_rules(const __grid_constant__ RuleParams P) {
  using Count = typename RlCount<LONG>::type;
  using K = RlCount<LONG>;
  constexpr int VEC = 16 / (int)sizeof(T);
  extern __shared__ __align__(16) uint8_t rl_smem[];
  __shared__ float s_v[RL_THREADS / 32], s_cv[RL_CLUSTER], s_bias[RL_LIST];
  __shared__ int s_i[RL_THREADS / 32], s_ci[RL_CLUSTER], s_entry[RL_LIST], s_id[RL_LIST], s_touched[RL_TOUCH], s_entries, s_n;
  rl_started();
  const int tid = threadIdx.x, rank = (int)rl_rank(), ranks = (int)rl_ranks(), i = blockIdx.x / ranks, span = P.span;
  Count* cnt = reinterpret_cast<Count*>(rl_smem);                                    // [span]
  const bool counted = P.hist || P.n_bias;
  const T* in = reinterpret_cast<const T*>(P.in) + i * P.in_ld;
  T* out = reinterpret_cast<T*>(P.out) + i * P.out_ld;
  const int shift = (int)((reinterpret_cast<uintptr_t>(in) / sizeof(T)) % VEC);
  const bool vec_out = (int)((reinterpret_cast<uintptr_t>(out) / sizeof(T)) % VEC) == shift;
  // position u is in turn u / STEP, which CTA (turn % ranks) owns as its (turn / ranks)-th; ranks is a power of two
  constexpr int STEP = RL_THREADS * VEC;
  const int lg = 31 - __clz(ranks), u_end = P.vocab + shift;
  auto owner = [&](int u) { return (u / STEP) & (ranks - 1); };
  auto local = [&](int u) { return ((u / STEP) >> lg) * STEP + (u & (STEP - 1)); };
  auto place = [&](int turn) { return (turn * ranks + rank) * STEP; };   // where this CTA's turn begins
  // the CTA's logits on their way from memory to the L2 while it counts (whole groups, a thread per turn; the
  // L2 is where writes of the kernel before this one arrive too, so this need not wait for it)
  if (counted && place(tid) < u_end) {
    const int a = max(place(tid), shift ? VEC : 0), b = min(place(tid) + STEP, u_end / VEC * VEC);
    if (a < b)
      asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(in + (a - shift)), "r"((b - a) * (int)sizeof(T)) : "memory");
  }
  if (counted)
    for (int j = tid; j < span * (int)sizeof(Count) / 16; j += RL_THREADS) reinterpret_cast<uint4*>(cnt)[j] = make_uint4(0, 0, 0, 0);
  if (tid == 0) s_entries = s_n = 0;
  pdl_wait();
  pdl_trigger();
  // turns [t_lo, t_hi) lie inside the row, both rows aligned alike: whole groups, no checks
  const int turns = u_end > rank * STEP ? (u_end - rank * STEP - 1) / (ranks * STEP) + 1 : 0;
  const int t_lo = rank == 0 && shift ? 1 : 0;
  const int inside = (u_end - rank * STEP) / STEP;                       // whole turns of the row from this CTA's first on
  const int t_hi = vec_out && inside > 0 ? max(t_lo, (inside - 1) / ranks + 1) : t_lo;
  const int first = tid * VEC - shift;                                   // id of this thread's group in the turn at 0
  uint4 x[RL_BATCH];
  auto request = [&](int turn) {
#pragma unroll
    for (int k = 0; k < RL_BATCH; ++k)
      if (turn + k < t_hi) x[k] = *reinterpret_cast<const uint4*>(in + (place(turn + k) + first));
  };
  request(t_lo);
  const int nh = P.hist ? min(max(P.hist_len[i], 0), P.max_hist) : 0;
  const int np = P.prompt_len ? P.prompt_len[i] : 0;
  int mrow = P.mask ? (P.mask_row ? P.mask_row[i] : i) : -1;
  const float rep = P.rep ? P.rep[i] : 1.f, freq = P.freq ? P.freq[i] : 0.f, pres = P.pres ? P.pres[i] : 0.f;
  const int* hist = P.hist + i * P.hist_ld;
  const int* bias_id = P.bias_id + i * P.bias_ld;
  const bool none = P.mask && (mrow < -1 || mrow >= P.n_masks);
  if (none) {
    if (tid == 0) atomicOr(P.err, KQ_DEV_ERR_BAD_ROW);
    mrow = -1;
  }
  const uint32_t* mask = mrow >= 0 ? P.mask + mrow * P.mask_ld : nullptr;
  uint32_t m[RL_BATCH];                                   // the mask word of a group's first id
  auto request_mask = [&](int turn) {
#pragma unroll
    for (int k = 0; k < RL_BATCH; ++k)
      if (mask && turn + k < t_hi) m[k] = mask[(place(turn + k) + first) >> 5];
  };
  request_mask(t_lo);
  float bv = -INFINITY;
  int bi = 0x7fffffff;
  auto better = [&](float v, int j) {                     // equal values: the lowest id
    if (v > bv || (v == bv && j < bi)) { bv = v; bi = j; }
  };
  auto mine = [&](int id) { return id >= 0 && id < P.vocab && owner(id + shift) == rank; };
  auto mask_of = [&](int id) { return mask ? mask[id >> 5] : 0xffffffffu; };
  const bool apart = nh > RL_LOCAL;                       // the same for all CTAs of the row
  if (counted) {
    if (apart) {
      rl_all_started();
      rl_cluster_sync();                                  // every CTA's counts are zero
    } else {
      __syncthreads();
    }
    // adds to, or sets bits of, the count of one of this CTA's ids (h < 0: none), and lists it if it was 0; whole warps
    auto mark = [&](int h, uint32_t v, bool bits) {
      bool fresh = false;
      if (h >= 0) {
        const int at = local(h + shift), s = LONG ? 0 : 16 * (at & 1);
        uint32_t* word = reinterpret_cast<uint32_t*>(cnt) + (LONG ? at : at >> 1);
        const uint32_t old = bits ? atomicOr(word, v << s) : atomicAdd(word, v << s);
        fresh = ((old >> s) & (K::PROMPT | K::BIASED | K::MOST)) == 0;
      }
      const uint32_t who = __ballot_sync(0xffffffffu, fresh);
      int base = 0;
      if (who && (tid & 31) == 0) base = atomicAdd(&s_n, __popc(who));
      base = __shfl_sync(0xffffffffu, base, 0) + __popc(who & ((1u << (tid & 31)) - 1u));
      if (fresh && base < RL_TOUCH) s_touched[base] = h;
    };
    if (apart) {
      for (int j = rank * RL_THREADS + tid; j < nh; j += ranks * RL_THREADS) {
        const int h = hist[j];
        if (h < 0 || h >= P.vocab) continue;
        const int at = local(h + shift);
        const uint32_t s = LONG ? 0 : 16 * (at & 1);
        const uint32_t a = rl_at(reinterpret_cast<uint32_t*>(cnt) + (LONG ? at : at >> 1), (uint32_t)owner(h + shift));
        if (j < np) rl_or(a, K::PROMPT << s);
        else rl_add(a, 1u << s);
      }
    } else {
      for (int j0 = 0; j0 < nh; j0 += 4 * RL_THREADS) {
        int h[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) h[k] = j0 + k * RL_THREADS + tid < nh ? hist[j0 + k * RL_THREADS + tid] : -1;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const bool old = j0 + k * RL_THREADS + tid < np;
          if (j0 + k * RL_THREADS < nh) mark(mine(h[k]) ? h[k] : -1, old ? K::PROMPT : 1u, old);
        }
      }
    }
    for (int j0 = 0; j0 < P.n_bias; j0 += RL_THREADS) {
      const int j = j0 + tid, h = j < P.n_bias ? bias_id[j] : -1;
      const bool own_id = mine(h);
      mark(own_id ? h : -1, K::BIASED, true);
      if (own_id) {
        const int e = atomicAdd(&s_entries, 1);
        if (e < RL_LIST) {
          s_entry[e] = j;
          s_id[e] = h;
          s_bias[e] = P.bias[i * P.bias_ld + j];
        }
      }
    }
    if (apart) rl_cluster_sync();                         // every hit has arrived
    else __syncthreads();
  }
  if (!(counted && apart)) rl_all_started();              // by now they do (waited for after the stream: 45 16-bit rows 10.8 us, here 10.4)

  // ---- the stream: masks and writes every id, picks among the untouched. It keeps its largest value and
  // that value's turn; the id is looked up once, at the end.
  float top = -INFINITY;
  int top_turn = -1;
  constexpr int CW = VEC * (int)sizeof(Count) / 4;
  auto fast = [&](int turn, const uint4& v, uint32_t w) {
    union { uint4 q; T t[VEC]; } y;
    y.q = v;
    const int id = place(turn) + first;
    if (mask) {                                           // bit j: id + j is allowed
      uint32_t next = 0;
      if (shift && (id & 31) + VEC > 32 && (id >> 5) + 1 < (P.vocab + 31) >> 5) next = mask[(id >> 5) + 1];
      w = __funnelshift_r(w, next, id & 31);
    }
    if (mask || none) {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (none || !((w >> j) & 1u)) y.t[j] = rl_put<T>(-INFINITY);
    }
    *reinterpret_cast<uint4*>(out + id) = y.q;
    uint32_t c[CW], any = 0;                              // the group's counts
    if (counted) {
#pragma unroll
      for (int j = 0; j < CW; j += 2) {
        const uint2 t = reinterpret_cast<const uint2*>(cnt + turn * STEP + tid * VEC)[j / 2];
        c[j] = t.x;
        c[j + 1] = t.y;
        any |= t.x | t.y;
      }
    }
    float most = -INFINITY;
    if (!any) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) most = fmaxf(most, rl_get<T>(y.t[j]));
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (LONG ? c[j] == 0 : ((c[j / 2] >> (16 * (j & 1))) & 0xffffu) == 0) most = fmaxf(most, rl_get<T>(y.t[j]));
    }
    if (most > top) {
      top = most;
      top_turn = turn;
    }
  };
  auto edge = [&](int turn) {                             // a turn over an end of the row, or unlike alignments
    const int id0 = place(turn) + first;
    if (vec_out && id0 >= 0 && id0 + VEC <= P.vocab) {
      fast(turn, *reinterpret_cast<const uint4*>(in + id0), mask ? mask[id0 >> 5] : 0u);
      return;
    }
#pragma unroll 1
    for (int j = 0; j < VEC; ++j) {
      const int id = id0 + j;
      if (id < 0 || id >= P.vocab) continue;
      const bool allowed = !none && (!mask || ((mask[id >> 5] >> (id & 31)) & 1u));
      const T r = allowed ? in[id] : rl_put<T>(-INFINITY);
      out[id] = r;
      const float f = rl_get<T>(r);
      if (f > -INFINITY && !(counted && cnt[turn * STEP + tid * VEC + j])) better(f, id);
    }
  };
  // turns in their order: of equal values a thread keeps the first
#pragma unroll 1
  for (int turn = 0; turn < min(t_lo, turns); ++turn) edge(turn);
#pragma unroll 1
  for (int turn = t_lo; turn < t_hi; turn += RL_BATCH) {
    uint4 v[RL_BATCH];
    uint32_t w[RL_BATCH];
#pragma unroll
    for (int k = 0; k < RL_BATCH; ++k) {
      v[k] = x[k];
      w[k] = m[k];
    }
    request(turn + RL_BATCH);
    request_mask(turn + RL_BATCH);
#pragma unroll
    for (int k = 0; k < RL_BATCH; ++k)
      if (turn + k < t_hi) fast(turn + k, v[k], w[k]);
  }
#pragma unroll 1
  for (int turn = t_hi; turn < turns; ++turn) edge(turn);
  if (top_turn >= 0) {
    for (int j = VEC - 1; j >= 0; --j) {                  // the lowest of the group's untouched ids with that value
      const int id = place(top_turn) + first + j;
      if (!(counted && cnt[top_turn * STEP + tid * VEC + j]) && rl_get<T>(out[id]) == top) better(top, id);
    }
  }

  if (counted) {
    __syncthreads();                                      // the stream has written the touched ids too
    const int entries = s_entries, kept = entries > RL_LIST ? 0 : entries;
    // v: the id's logit (in place: the value itself, or masked and about to be again), b: its bias
    auto apply = [&](int h, uint32_t c, float v, float b, uint32_t word) {
      if (c & ~K::BIASED) v = rl_penalise(v, (c & K::MOST) | ((c & K::PROMPT) ? 0x80000000u : 0u), rep, freq, pres);
      if (c & K::BIASED) v = __fadd_rn(v, b);
      if (none || !((word >> (h & 31)) & 1u)) v = -INFINITY;
      const T r = rl_put<T>(v);
      out[h] = r;
      const float f = rl_get<T>(r);
      if (f > -INFINITY) better(f, h);
    };
    auto bias_of = [&](int h, uint32_t c) {               // the last entry of the list with this id
      int last = -1;
      float b = 0.f;
      if (c & K::BIASED)
        for (int e = 0; e < kept; ++e)
          if (s_id[e] == h && s_entry[e] > last) {
            last = s_entry[e];
            b = s_bias[e];
          }
      return b;
    };
    if (entries > RL_LIST) {
      // more entries than are kept: the list from its end, a thread an entry. Of the entries whose ids share a slot
      // the last one stands and its id is done; another id of the slot is left for the next turn. (128 rows of 151936
      // with 300 / 2000 / 10000 / 151936 entries 40 / 76 / 168 / 1760 us; a search of the list for each id took 348 us for
      // 2000 and 66 ms for 10000. Short lists pay up to 0.25 us for the larger kernel.)
      for (int j1 = P.n_bias - 1; j1 >= 0; j1 -= RL_THREADS) {
        const int j = j1 - tid, h = j >= 0 ? bias_id[j] : -1, at = mine(h) ? local(h + shift) : -1;
        bool open = at >= 0 && (cnt[at] & K::BIASED);
        while (__syncthreads_or(open)) {
          s_entry[tid] = -1;
          __syncthreads();
          if (open) atomicMax(&s_entry[h & (RL_LIST - 1)], j);
          __syncthreads();
          if (open && s_entry[h & (RL_LIST - 1)] == j) {
            apply(h, cnt[at], rl_get<T>(in[h]), P.bias[i * P.bias_ld + j], mask_of(h));
            cnt[at] = 0;
          }
          __syncthreads();
          open = open && (cnt[at] & K::BIASED);
        }
      }
    }
    if (!apart && s_n <= RL_TOUCH) {
      for (int e = tid; e < s_n; e += RL_THREADS) {
        const int h = s_touched[e];
        const uint32_t c = cnt[local(h + shift)], word = mask_of(h);
        const float v = rl_get<T>(in[h]);                 // on its way while the list is searched
        if (c) apply(h, c, v, bias_of(h, c), word);
      }
    } else {
      for (int at = tid; at < span; at += RL_THREADS) {
        const int h = place(at / STEP) + (at & (STEP - 1)) - shift;
        const uint32_t c = cnt[at];
        if (c) apply(h, c, rl_get<T>(in[h]), bias_of(h, c), mask_of(h));
      }
    }
  }
  if (!P.best) return;
  // ---- the greedy id: warp, CTA, cluster
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) better(__shfl_xor_sync(0xffffffffu, bv, off), __shfl_xor_sync(0xffffffffu, bi, off));
  if ((tid & 31) == 0) { s_v[tid >> 5] = bv; s_i[tid >> 5] = bi; }
  __syncthreads();
  if (tid < 32) {
    bv = tid < RL_THREADS / 32 ? s_v[tid] : -INFINITY;
    bi = tid < RL_THREADS / 32 ? s_i[tid] : 0x7fffffff;
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) better(__shfl_xor_sync(0xffffffffu, bv, off), __shfl_xor_sync(0xffffffffu, bi, off));
    if (tid == 0) {
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(rl_at(&s_cv[rank], 0)), "f"(bv) : "memory");
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(rl_at(&s_ci[rank], 0)), "r"(bi) : "memory");
    }
  }
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  if (rank != 0) return;                      // nothing reads the other CTAs' shared memory any more
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (tid == 0) {
    bv = -INFINITY;
    bi = 0x7fffffff;
    for (int r = 0; r < ranks; ++r) better(s_cv[r], s_ci[r]);
    P.best[i] = bi == 0x7fffffff ? -1 : bi;
  }
}

}  // namespace kq
