// kq_serve.cu -- C ABI (include/kq.h) of the serving operators on device tensors: the paged K/V cache
// (kq_page_append, kq_page_attend) and the rules on logits (kq_logit_rules). Every argument the host
// can see is checked here before anything is launched; the kernels check the rest themselves.
#include "../../include/kq.h"
#include "kq_common.cuh"
#include "kq_host.h"
#include "kq_paged.cuh"
#include "kq_rules.cuh"

#include <cuda_runtime.h>
#include <algorithm>
#include <atomic>
#include <mutex>
#include <new>

using namespace kq;

#define CU(call)                                                                                 \
  do {                                                                                           \
    cudaError_t e_ = (call);                                                                     \
    if (e_ != cudaSuccess) return kqh_error(KQ_ERR_BACKEND, std::string(#call) + ": " + cudaGetErrorString(e_)); \
  } while (0)
#define REQUIRE(cond, text)                              \
  do {                                                   \
    if (!(cond)) return kqh_error(KQ_ERR_ARG, (text));   \
  } while (0)

// The attention's scratch of a handle, or of several whose calls share a stream, and of the graphs that captured
// such calls.
struct ScratchBlock;
struct Scratch {
  AttendScratch s{};
  int device = 0;
  std::atomic<int> users{0};
  ScratchBlock* block = nullptr;
  Scratch* next = nullptr;
};
constexpr int SCRATCH_BLOCK = 4;
struct ScratchBlock {
  void* p = nullptr;
  Scratch s[SCRATCH_BLOCK];
  int idle = 0;
  bool released = false;
  ScratchBlock* next = nullptr;
};

struct kq_pages {
  kq_page_desc d{};
  int device = 0, shift = 0;
  KqhDevice dev{};
  Scratch* scratch = nullptr;
};

// The attention kernel of a cache type, head size, query heads per CTA (8 or 16) and precision.
typedef void (*AttendFn)(AttendParams, AttendScratch);
struct AttendKernel {
  AttendFn fn;
  int smem, per_sm;
};
template <int CT, int HD, int NT, bool PREC>
static AttendKernel attend_entry() {
  return {k_page_attend<CT, HD, NT, PREC>, PaShape<CT, HD, NT, PREC>::SMEM, PaShape<CT, HD, NT, PREC>::PER_SM};
}
template <int CT, int HD>
static AttendKernel attend_of(bool wide, bool prec) {
  if (wide) return prec ? attend_entry<CT, HD, 2, true>() : attend_entry<CT, HD, 2, false>();
  return prec ? attend_entry<CT, HD, 1, true>() : attend_entry<CT, HD, 1, false>();
}
template <int CT>
static AttendKernel attend_of(int hd, bool wide, bool prec) {
  return hd == 64 ? attend_of<CT, 64>(wide, prec) : hd == 128 ? attend_of<CT, 128>(wide, prec) : attend_of<CT, 256>(wide, prec);
}
static AttendKernel attend_kernel(int type, int hd, bool wide, bool prec) {
  return type == KQ_F16 ? attend_of<PG_F16>(hd, wide, prec) : type == KQ_BF16 ? attend_of<PG_BF16>(hd, wide, prec)
                                                                             : attend_of<PG_E4M3>(hd, wide, prec);
}

typedef void (*AppendFn)(AppendParams);
template <int ST, int U>
static AppendFn append_of(int cache) {
  return cache == KQ_F16 ? k_page_append<ST, PG_F16, U> : cache == KQ_BF16 ? k_page_append<ST, PG_BF16, U> : k_page_append<ST, PG_E4M3, U>;
}
template <int U>
static AppendFn append_kernel(int src, int cache) {
  return src == KQ_F32 ? append_of<PG_F32, U>(cache) : src == KQ_F16 ? append_of<PG_F16, U>(cache) : append_of<PG_BF16, U>(cache);
}

// Launch with programmatic stream serialisation: the kernel's CTAs may be scheduled while the previous
// kernel's last ones run; every kernel here begins with the dependency wait, so nothing else changes.
template <typename... A>
static cudaError_t launch(void (*fn)(A...), dim3 grid, int threads, size_t smem, void* stream, int cluster, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)cluster;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, fn, args...);
}

static int type_size(int type) { return type == KQ_F32 ? 4 : type == KQ_E4M3 ? 1 : 2; }
static bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
// A stride of a dimension of one element does not matter.
static long long stride_of(long long stride, long long size) { return size > 1 ? stride : 0; }
// Strides whose rows all start on 16-byte boundaries and do not run backwards.
static bool rows_ok(const void* p, long long a, long long b, int esize) {
  return p && aligned(p, 16) && a >= 0 && b >= 0 && a * esize % 16 == 0 && b * esize % 16 == 0;
}

static int pages_check(const kq_page_desc* d) {
  REQUIRE(d, "kq_pages_create: null description");
  REQUIRE(d->type == KQ_F16 || d->type == KQ_BF16 || d->type == KQ_E4M3, "kq_pages_create: the cache type is f16, bf16 or e4m3");
  REQUIRE(d->head_dim == 64 || d->head_dim == 128 || d->head_dim == 256, "kq_pages_create: head_dim must be 64, 128 or 256");
  REQUIRE(d->page >= 16 && d->page <= 1024 && (d->page & (d->page - 1)) == 0, "kq_pages_create: page must be a power of two from 16 to 1024");
  REQUIRE(d->n_pages >= 1 && d->n_kv_heads >= 1 && d->n_kv_heads <= 1024, "kq_pages_create: bad page or head count");
  const int es = type_size(d->type);
  REQUIRE(rows_ok(d->k, d->k_page, d->k_head, es) && rows_ok(d->k, d->k_row, 0, es) && rows_ok(d->v, d->v_page, d->v_head, es) &&
              rows_ok(d->v, d->v_row, 0, es),
          "kq_pages_create: K and V rows must start on 16-byte boundaries");
  REQUIRE(d->type == KQ_E4M3 || (!d->k_scale && !d->v_scale), "kq_pages_create: only e4m3 caches have scales");
  return KQ_OK;
}

// Scratches are allocated four at a time, and those of freed handles are kept for the next ones: a server makes and
// drops handles while it runs, and an allocation costs some milliseconds. Between launches a scratch's tickets are
// zero, so it can be handed on as it is. Launches may still use a scratch when its last user leaves, and leaving
// makes no CUDA call, for it may happen at any time (a collected Python object, in the middle of a capture). So those
// that were left become idle together: a new handle that finds no idle one, but two of them, waits for the device.
constexpr size_t SCRATCH_PART = (size_t)2 * PA_MAX_CTAS * PA_MAX_HEADS * PA_PLD * sizeof(float);
constexpr size_t SCRATCH_BYTES = SCRATCH_PART + (PA_MAX_CTAS * sizeof(int) + 255) / 256 * 256;
constexpr int SCRATCH_KEEP = 16;     // idle ones per device; blocks of four beyond them are released after that wait
static std::mutex g_scratch_mu;
static struct { Scratch *idle, *left; int n_left; } g_scratch[16];

static Scratch* scratch_pop(int device) {               // an idle one, or null; the lock is held
  Scratch* s = g_scratch[device].idle;
  if (s) {
    g_scratch[device].idle = s->next;
    s->users = 1;
  }
  return s;
}
static cudaError_t scratch_take(int device, Scratch*& out) {
  auto& kept = g_scratch[device];
  Scratch* left = nullptr;
  {
    std::lock_guard<std::mutex> lk(g_scratch_mu);
    if ((out = scratch_pop(device))) return cudaSuccess;
    if (kept.n_left >= 2) {
      left = kept.left;
      kept.left = nullptr;
      kept.n_left = 0;
    }
  }
  if (left) {
    const cudaError_t e = cudaDeviceSynchronize();      // no launch uses these any more
    ScratchBlock* unused = nullptr;
    {
      std::lock_guard<std::mutex> lk(g_scratch_mu);
      int n = 0;
      for (Scratch* s = left; s; s = left) {
        left = s->next;
        Scratch*& list = e == cudaSuccess ? kept.idle : kept.left;
        if (e != cudaSuccess) ++kept.n_left;
        s->next = list;
        list = s;
      }
      if (e != cudaSuccess) return e;
      for (Scratch* s = kept.idle; s; s = s->next, ++n) s->block->idle = 0;
      for (Scratch* s = kept.idle; s; s = s->next) ++s->block->idle;
      for (Scratch** at = &kept.idle; *at;) {           // whole blocks leave the list
        ScratchBlock* b = (*at)->block;
        if (b->idle != SCRATCH_BLOCK || (!b->released && n - SCRATCH_BLOCK < SCRATCH_KEEP)) {
          at = &(*at)->next;
          continue;
        }
        if (!b->released) {
          b->released = true;
          b->next = unused;
          unused = b;
          n -= SCRATCH_BLOCK;
        }
        *at = (*at)->next;
      }
      out = scratch_pop(device);
    }
    while (unused) {
      ScratchBlock* b = unused;
      unused = b->next;
      cudaFree(b->p);
      delete b;
    }
    return cudaSuccess;
  }
  ScratchBlock* b = new (std::nothrow) ScratchBlock;
  if (!b) return cudaErrorMemoryAllocation;
  cudaError_t e = cudaMalloc(&b->p, SCRATCH_BLOCK * SCRATCH_BYTES);
  for (int i = 0; e == cudaSuccess && i < SCRATCH_BLOCK; ++i) {
    char* p = static_cast<char*>(b->p) + i * SCRATCH_BYTES;
    b->s[i].s.part = reinterpret_cast<float*>(p);
    b->s[i].s.ticket = reinterpret_cast<int*>(p + SCRATCH_PART);
    b->s[i].device = device;
    b->s[i].block = b;
    e = cudaMemset(b->s[i].s.ticket, 0, PA_MAX_CTAS * sizeof(int));
  }
  if (e == cudaSuccess) e = cudaStreamSynchronize(0);   // the first call may be on a stream that does not wait for this one
  if (e != cudaSuccess) {
    cudaFree(b->p);
    delete b;
    return e;
  }
  std::lock_guard<std::mutex> lk(g_scratch_mu);
  for (int i = SCRATCH_BLOCK - 1; i >= 0; --i) {
    b->s[i].next = kept.idle;
    kept.idle = &b->s[i];
  }
  out = scratch_pop(device);
  return cudaSuccess;
}
static void scratch_leave(Scratch* s) {
  if (--s->users) return;
  std::lock_guard<std::mutex> lk(g_scratch_mu);
  auto& kept = g_scratch[s->device];
  s->next = kept.left;
  kept.left = s;
  ++kept.n_left;
}
// A graph under capture on `stream` uses the scratch for as long as the graph, or what was instantiated from it, lives.
static cudaError_t scratch_hold(Scratch* s, cudaStream_t stream) {
  cudaStreamCaptureStatus state;
  cudaGraph_t graph = nullptr;
  cudaError_t e = cudaStreamGetCaptureInfo(stream, &state, nullptr, &graph);
  if (e != cudaSuccess || state != cudaStreamCaptureStatusActive) return e;
  cudaUserObject_t held;
  ++s->users;
  e = cudaUserObjectCreate(&held, s, [](void* p) { scratch_leave(static_cast<Scratch*>(p)); }, 1, cudaUserObjectNoDestructorSync);
  if (e != cudaSuccess) {
    --s->users;
    return e;
  }
  e = cudaGraphRetainUserObject(graph, held, 1, cudaGraphUserObjectMove);
  if (e != cudaSuccess) cudaUserObjectRelease(held, 1);
  return e;
}

// The attention kernels' shared memory, allowed once per device (which is current).
static cudaError_t attend_setup(int device, int type, int hd) {
  static std::atomic<unsigned> done[16];
  const int at = (type - KQ_F16) * 3 + (hd == 64 ? 0 : hd == 128 ? 1 : 2);
  if (done[device].load(std::memory_order_acquire) >> at & 1u) return cudaSuccess;
  for (int v = 0; v < 4; ++v) {
    const AttendKernel k = attend_kernel(type, hd, v & 1, v & 2);
    const cudaError_t e = cudaFuncSetAttribute(k.fn, cudaFuncAttributeMaxDynamicSharedMemorySize, k.smem);
    if (e != cudaSuccess) return e;
  }
  done[device].fetch_or(1u << at, std::memory_order_release);
  return cudaSuccess;
}

kq_pages* kqh_pages_create(const void* desc, int device, const kq_pages* with, int* err) {
  const kq_page_desc* given = static_cast<const kq_page_desc*>(desc);
  KqhDevice dev;
  kq_page_desc own{}, *d = nullptr;
  if (given) {
    own = *given;
    own.k_page = stride_of(own.k_page, own.n_pages);
    own.v_page = stride_of(own.v_page, own.n_pages);
    own.k_head = stride_of(own.k_head, own.n_kv_heads);
    own.v_head = stride_of(own.v_head, own.n_kv_heads);
    d = &own;
  }
  if (pages_check(d) || kqh_device(device, &dev)) return nullptr;
  kq_pages* c = new (std::nothrow) kq_pages;
  if (!c) {
    kqh_error(KQ_ERR_MEMORY, "page handle allocation");
    return nullptr;
  }
  c->d = *d;
  c->device = device;
  c->dev = dev;
  if (err) c->dev.err = err;
  while ((1 << c->shift) < d->page) ++c->shift;
  cudaError_t e = attend_setup(device, d->type, d->head_dim);
  if (e == cudaSuccess && with) {
    c->scratch = with->scratch;
    ++c->scratch->users;
  } else if (e == cudaSuccess) {
    e = scratch_take(device, c->scratch);
  }
  if (e != cudaSuccess) {
    kqh_error(e == cudaErrorMemoryAllocation ? KQ_ERR_MEMORY : KQ_ERR_BACKEND,
              std::string("kq_pages_create: scratch allocation or kernel set-up: ") + cudaGetErrorString(e));
    kq_pages_free(c);
    return nullptr;
  }
  return c;
}

extern "C" kq_pages* kq_pages_create(const kq_page_desc* d, int device) { return kqh_pages_create(d, device, nullptr, nullptr); }

extern "C" void kq_pages_free(kq_pages* c) {
  if (!c) return;
  if (c->scratch) scratch_leave(c->scratch);
  delete c;
}

static PageTable table_of(const kq_pages* c, const int32_t* table, const int32_t* seq, long long ld, int n_seq, int max_pages) {
  return PageTable{table, seq, ld, n_seq, max_pages, c->d.n_pages, c->shift};
}
static bool table_ok(const kq_pages* c, const int32_t* table, const int32_t* seq, long long ld, int n_seq, int max_pages, int n) {
  return table && n_seq >= 1 && max_pages >= 1 && ld >= max_pages && (seq || n <= n_seq) &&
         (long long)max_pages * c->d.page <= 0x7ffff000ll;   // keys and the tiles over a sequence's end are 32-bit
}

extern "C" int kq_page_append(kq_pages* c, const kq_append_args* given, void* stream) {
  REQUIRE(c && given, "kq_page_append: null argument");
  kq_append_args own = *given, *a = &own;
  for (long long* x : {&own.k_tok, &own.v_tok, &own.q_tok, &own.o_tok}) *x = stride_of(*x, own.n);
  for (long long* x : {&own.k_head, &own.v_head}) *x = stride_of(*x, c->d.n_kv_heads);
  for (long long* x : {&own.q_head, &own.o_head}) *x = stride_of(*x, own.n_heads);
  REQUIRE(a->n >= 0, "kq_page_append: negative token count");
  REQUIRE(a->src_type == KQ_F32 || a->src_type == KQ_F16 || a->src_type == KQ_BF16, "kq_page_append: rows are f32, f16 or bf16");
  const int es = type_size(a->src_type);
  REQUIRE(rows_ok(a->k, a->k_tok, a->k_head, es) && rows_ok(a->v, a->v_tok, a->v_head, es),
          "kq_page_append: key and value rows must start on 16-byte boundaries");
  REQUIRE(!a->q == !a->q_out && (a->q ? a->n_heads >= 1 : a->n_heads == 0), "kq_page_append: queries need q, q_out and n_heads");
  REQUIRE(!a->q || (rows_ok(a->q, a->q_tok, a->q_head, es) && rows_ok(a->q_out, a->o_tok, a->o_head, es)),
          "kq_page_append: query rows must start on 16-byte boundaries");
  REQUIRE(table_ok(c, a->table, a->seq, a->table_ld, a->n_seq, a->max_pages, a->n) && a->pos, "kq_page_append: bad page table or positions");
  REQUIRE(a->rot >= 0 && a->rot % 16 == 0 && a->rot <= c->d.head_dim, "kq_page_append: rot must be a multiple of 16 up to head_dim");
  REQUIRE(a->rot ? (rows_ok(a->cos_t, a->rope_ld, 0, 4) && rows_ok(a->sin_t, a->rope_ld, 0, 4) && a->rope_ld >= a->rot / 2 && a->n_pos >= 1)
                 : (!a->cos_t && !a->sin_t),
          "kq_page_append: bad rotation table");
  REQUIRE(a->n_heads <= 65535, "kq_page_append: too many heads");
  if (a->n == 0) return KQ_OK;
  CU(cudaSetDevice(c->device));
  AppendParams P;
  P.k = a->k; P.v = a->v; P.q = a->q; P.q_out = a->q_out; P.kc = c->d.k; P.vc = c->d.v;
  P.k_tok = a->k_tok; P.k_head = a->k_head; P.v_tok = a->v_tok; P.v_head = a->v_head;
  P.q_tok = a->q_tok; P.q_head = a->q_head; P.o_tok = a->o_tok; P.o_head = a->o_head;
  P.kp = c->d.k_page; P.kh = c->d.k_head; P.kr = c->d.k_row;
  P.vp = c->d.v_page; P.vh = c->d.v_head; P.vr = c->d.v_row;
  P.ks = c->d.k_scale; P.vs = c->d.v_scale;
  P.T = table_of(c, a->table, a->seq, a->table_ld, a->n_seq, a->max_pages);
  P.pos = a->pos; P.cos_t = a->cos_t; P.sin_t = a->sin_t; P.rope_ld = a->rope_ld;
  P.n_heads = a->n_heads; P.n_kv = c->d.n_kv_heads; P.hd = c->d.head_dim;
  P.rot = a->rot; P.n_pos = a->n_pos; P.err = c->dev.err;
  // AP_DEEP head rows a thread above 64 CTAs an SM (the angles are read once for them), one below. Measured in turn, us with
  // one / three: 48 bf16 rows of 128, 2000 / 4000 / 5000 / 8192 tokens 9.3 / 7.6, 18.7 / 17.9, 24.9 / 25.6, 40.6 / 40.2; 24 fp32
  // rows of 256, 1000 / 2000 / 3000 / 4000 tokens 7.9 / 7.1, 14.2 / 12.4, 22.1 / 22.9, 29.4 / 31.2. Three are faster while a
  // call's rows stay in the L2 and up to 7 % slower beyond: the rule costs up to a fifth below its border, 7 % above.
  const int units = c->d.head_dim / (a->src_type == KQ_F32 ? 8 : 16), rows = a->n_heads + 2 * P.n_kv;
  const int slices = (rows * units + AP_THREADS - 1) / AP_THREADS;
  const bool deep = (long long)a->n * slices > 64ll * c->dev.nsm;
  const dim3 grid((unsigned)a->n, (unsigned)(deep ? (slices + AP_DEEP - 1) / AP_DEEP : slices));
  const AppendFn fn = deep ? append_kernel<AP_DEEP>(a->src_type, c->d.type) : append_kernel<1>(a->src_type, c->d.type);
  CU(launch(fn, grid, AP_THREADS, 0, stream, 1, P));
  return KQ_OK;
}

extern "C" int kq_page_attend(kq_pages* c, const kq_attend_args* given, void* stream) {
  REQUIRE(c && given, "kq_page_attend: null argument");
  kq_attend_args own = *given, *a = &own;
  for (long long* x : {&own.q_tok, &own.o_tok}) *x = stride_of(*x, own.n);
  for (long long* x : {&own.q_head, &own.o_head}) *x = stride_of(*x, own.n_heads);
  REQUIRE(a->n >= 0, "kq_page_attend: negative token count");
  REQUIRE(a->type == KQ_F32 || a->type == KQ_F16 || a->type == KQ_BF16, "kq_page_attend: queries are f32, f16 or bf16");
  const int es = type_size(a->type);
  REQUIRE(rows_ok(a->q, a->q_tok, a->q_head, es) && rows_ok(a->out, a->o_tok, a->o_head, es),
          "kq_page_attend: query and output rows must start on 16-byte boundaries");
  REQUIRE(a->n_heads >= c->d.n_kv_heads && a->n_heads % c->d.n_kv_heads == 0 && a->n_heads <= 65535,
          "kq_page_attend: n_heads must be a multiple of the cache's heads");
  REQUIRE(table_ok(c, a->table, a->seq, a->table_ld, a->n_seq, a->max_pages, a->n) && a->len, "kq_page_attend: bad page table or lengths");
  REQUIRE(a->window >= 0, "kq_page_attend: negative window");
  if (a->n == 0) return KQ_OK;
  CU(cudaSetDevice(c->device));
  AttendParams P;
  P.q = a->q; P.out = a->out; P.q_tok = a->q_tok; P.q_head = a->q_head; P.o_tok = a->o_tok; P.o_head = a->o_head;
  P.kc = c->d.k; P.vc = c->d.v;
  P.kp = c->d.k_page; P.kh = c->d.k_head; P.kr = c->d.k_row;
  P.vp = c->d.v_page; P.vh = c->d.v_head; P.vr = c->d.v_row;
  P.ks = c->d.k_scale; P.vs = c->d.v_scale;
  P.T = table_of(c, a->table, a->seq, a->table_ld, a->n_seq, a->max_pages);
  P.len = a->len; P.n = a->n; P.n_heads = a->n_heads; P.n_kv = c->d.n_kv_heads; P.type = a->type;
  P.window = a->window; P.scale = a->scale; P.err = c->dev.err;
  const int G = a->n_heads / P.n_kv;
  // fp32 queries want fp32 scores: the cache's 16-bit type in two or three terms; so do fp16 queries
  // (11 bits) on a bf16 cache (8 bits)
  const bool prec = a->type == KQ_F32 || (c->d.type == KQ_BF16 && a->type == KQ_F16);
  const AttendKernel k = attend_kernel(c->d.type, c->d.head_dim, G > 8, prec);
  const int heads = G > 8 ? 16 : 8;
  const long long tiles = (((long long)a->max_pages << c->shift) + PA_TILE - 1) / PA_TILE;
  const long long most = (long long)a->n * P.n_kv * ((G + heads - 1) / heads) * tiles;
  const unsigned grid = (unsigned)std::min<long long>(most, std::min(PA_MAX_CTAS, c->dev.nsm * k.per_sm));
  CU(scratch_hold(c->scratch, (cudaStream_t)stream));
  CU(launch(k.fn, dim3(grid), PA_WARPS * 32, k.smem, stream, 1, P, c->scratch->s));
  return KQ_OK;
}

typedef void (*RulesFn)(RuleParams);
static RulesFn rules_kernel(int type, bool deep) {
  if (type == KQ_F32) return deep ? k_logit_rules<float, true> : k_logit_rules<float, false>;
  if (type == KQ_F16) return deep ? k_logit_rules<__half, true> : k_logit_rules<__half, false>;
  return deep ? k_logit_rules<__nv_bfloat16, true> : k_logit_rules<__nv_bfloat16, false>;
}
// Shared memory and cluster sizes above the defaults, allowed once per device (which is current).
static int rules_setup(int device) {
  static std::atomic<bool> done[16];
  if (done[device].load(std::memory_order_acquire)) return KQ_OK;
  const int smem = (KQ_RULES_MAX_VOCAB / RL_CLUSTER + 2 * RL_THREADS * 8) * 4;
  for (int type : {KQ_F32, KQ_F16, KQ_BF16})
    for (bool deep : {false, true}) {
      CU(cudaFuncSetAttribute(rules_kernel(type, deep), cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
      CU(cudaFuncSetAttribute(rules_kernel(type, deep), cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    }
  done[device].store(true, std::memory_order_release);
  return KQ_OK;
}

int kqh_rules_check(const void* args) {
  const kq_rule_args* a = static_cast<const kq_rule_args*>(args);
  REQUIRE(a, "kq_logit_rules: null argument");
  REQUIRE(a->n >= 0 && a->vocab >= 1 && a->vocab <= KQ_RULES_MAX_VOCAB && a->n <= (1 << 26), "kq_logit_rules: bad row count or vocabulary size");
  REQUIRE(a->type == KQ_F32 || a->type == KQ_F16 || a->type == KQ_BF16, "kq_logit_rules: logits are f32, f16 or bf16");
  const int es = type_size(a->type);
  REQUIRE(a->logits && a->out && aligned(a->logits, es) && aligned(a->out, es) && a->in_ld >= a->vocab && a->out_ld >= a->vocab,
          "kq_logit_rules: bad logits or output");
  REQUIRE(a->out != a->logits || a->in_ld == a->out_ld, "kq_logit_rules: in place, both strides must be equal");
  REQUIRE(!a->hist == !a->hist_len && (!a->hist || (a->max_hist >= 0 && a->hist_ld >= a->max_hist)), "kq_logit_rules: bad histories");
  REQUIRE(a->hist || !a->prompt_len, "kq_logit_rules: prompt lengths without histories");
  REQUIRE(!a->bias_id == !a->bias && (a->bias ? (a->n_bias >= 0 && a->bias_ld >= a->n_bias) : a->n_bias == 0), "kq_logit_rules: bad bias lists");
  REQUIRE(a->mask ? (a->n_masks >= 1 && a->mask_ld >= (a->vocab + 31) / 32 && (a->mask_row || a->n <= a->n_masks)) : !a->mask_row,
          "kq_logit_rules: bad masks");
  return KQ_OK;
}
int kqh_logit_rules(const void* args, int device, int* err, void* stream) {
  const kq_rule_args* a = static_cast<const kq_rule_args*>(args);
  KqhDevice dev;
  int rc = kqh_rules_check(a);
  if (rc || (rc = kqh_device(device, &dev)) || a->n == 0) return rc;
  RuleParams P;
  P.in = a->logits; P.out = a->out; P.in_ld = a->in_ld; P.out_ld = a->out_ld; P.best = a->best;
  P.hist = a->hist; P.hist_len = a->hist_len; P.prompt_len = a->prompt_len; P.hist_ld = a->hist_ld;
  P.rep = a->repetition; P.freq = a->frequency; P.pres = a->presence;
  P.bias_id = a->bias_id; P.bias = a->bias; P.bias_ld = a->bias_ld;
  P.mask = a->mask; P.mask_row = a->mask_row; P.mask_ld = a->mask_ld;
  P.n = a->n; P.vocab = a->vocab; P.max_hist = a->max_hist; P.n_bias = a->n_bias; P.n_masks = a->n_masks;
  P.err = err ? err : dev.err;
  // 32-bit counts only where a history may hold more of one id than 14 bits count. The smallest
  // cluster whose CTAs hold at most RL_BYTES, then larger ones while the device has CTAs to spare.
  const bool deep = a->max_hist > (int)RlCount<false>::MOST;
  const int vec = 16 / type_size(a->type), reach = a->vocab + vec - 1, bytes = !P.hist && !P.n_bias ? 0 : deep ? 4 : 2;
  int cl = 1;
  while (cl < RL_CLUSTER && ((long long)reach * bytes > (long long)cl * RL_BYTES ||
                             ((long long)a->n * cl * 2 <= 2 * dev.nsm && reach > cl * RL_THREADS * vec)))
    cl *= 2;
  const int turn = RL_THREADS * vec;
  P.span = (reach + cl * turn - 1) / (cl * turn) * turn;
  if ((rc = rules_setup(device))) return rc;
  CU(launch(rules_kernel(a->type, deep), dim3((unsigned)a->n * (unsigned)cl), RL_THREADS, (size_t)P.span * bytes, stream, cl, P));
  return KQ_OK;
}

extern "C" int kq_logit_rules(const kq_rule_args* a, int device, void* stream) { return kqh_logit_rules(a, device, nullptr, stream); }

// ------------------------------------------------------------------------------ tensor objects
// DLPack's DLTensor (its version 1 ABI).
struct DlTensor {
  void* data;
  int32_t device_type, device_id;   // 2: CUDA
  int32_t ndim;
  uint8_t code, bits;               // 0 int, 1 uint, 2 float, 4 bfloat, 10 float8_e4m3fn
  uint16_t lanes;
  int64_t* shape;
  int64_t* strides;                 // null: dense
  uint64_t byte_offset;
};
typedef int (*DescribeFn)(void*, void*);
static std::atomic<DescribeFn> g_describe;

extern "C" int kq_tensor_source(int (*describe)(void*, void*)) {
  g_describe.store(describe, std::memory_order_release);
  return KQ_OK;
}

typedef int (*CurrentFn)(int, int32_t, void**);
static std::atomic<CurrentFn> g_current;

extern "C" int kq_tensor_stream(int (*current)(int, int32_t, void**)) {
  g_current.store(current, std::memory_order_release);
  return KQ_OK;
}
// `stream`, or the binding's current one on the device where that is asked for.
static bool stream_for(int device, void*& stream) {
  if (stream != KQ_STREAM_CURRENT) return true;
  stream = nullptr;
  const CurrentFn current = g_current.load(std::memory_order_acquire);
  return !current || current(2, device, &stream) == 0;
}

constexpr int T_I32 = 100;
struct Tensor {
  void* p = nullptr;
  int type = -1, device = -1;
  long long n[3] = {0, 0, 0}, s[3] = {0, 0, 0};
};
// The tensor behind `object`, if it is a CUDA tensor of `nd` dimensions without empty ones, dense in the last.
static bool tensor_of(void* object, int nd, Tensor& t) {
  const DescribeFn describe = g_describe.load(std::memory_order_acquire);
  DlTensor d{};
  if (!describe || !object || describe(object, &d) != 0 || d.device_type != 2 || d.ndim != nd || d.lanes != 1 || !d.data) return false;
  t.p = static_cast<char*>(d.data) + d.byte_offset;
  t.device = d.device_id;
  t.type = d.code == 2 && d.bits == 32 ? KQ_F32 : d.code == 2 && d.bits == 16 ? KQ_F16 : d.code == 4 && d.bits == 16 ? KQ_BF16
           : d.code <= 1 && d.bits == 32 ? T_I32 : -1;
  long long dense = 1;
  for (int i = nd - 1; i >= 0; --i) {
    t.n[i] = d.shape[i];
    t.s[i] = d.strides ? d.strides[i] : dense;
    dense *= d.shape[i];
    if (t.n[i] < 1 || t.n[i] > 0x7fffffffll) return false;
  }
  return t.s[nd - 1] == 1 || t.n[nd - 1] == 1;
}
static bool tensor_as(void* object, const Tensor& like, Tensor& t, int nd) {   // the same type, device and shape
  return tensor_of(object, nd, t) && t.type == like.type && t.device == like.device && t.n[0] == like.n[0] &&
         (nd < 2 || t.n[1] == like.n[1]) && (nd < 3 || t.n[2] == like.n[2]);
}
static bool vector_as(void* object, int type, int device, long long n, Tensor& t) {
  return tensor_of(object, 1, t) && t.type == type && t.device == device && t.n[0] == n;
}
#define FITS(cond)                     \
  do {                                 \
    if (!(cond)) return KQ_TENSOR_OTHER; \
  } while (0)

extern "C" int kq_page_append_tensors(kq_pages* c, void* k, void* v, void* table, void* pos, void* seq, void* cos_t, void* sin_t,
                                      void* q, void* q_out, void* stream) {
  FITS(c && !cos_t == !sin_t && !q == !q_out && stream_for(c->device, stream));
  const int dev = c->device;
  Tensor tk, tv, tt, tp, ts, tc, tsn, tq, to;
  FITS(tensor_of(k, 3, tk) && tk.device == dev && tk.n[1] == c->d.n_kv_heads && tk.n[2] == c->d.head_dim && tensor_as(v, tk, tv, 3));
  const long long n = tk.n[0];
  FITS(tensor_of(table, 2, tt) && tt.type == T_I32 && tt.device == dev && vector_as(pos, T_I32, dev, n, tp));
  if (seq) FITS(vector_as(seq, T_I32, dev, n, ts));
  else FITS(n <= tt.n[0]);
  if (cos_t)
    FITS(tensor_of(cos_t, 2, tc) && tc.type == KQ_F32 && tc.device == dev && tensor_as(sin_t, tc, tsn, 2) &&
         (tc.n[0] == 1 || tc.s[0] == tsn.s[0]));
  if (q)
    FITS(tensor_of(q, 3, tq) && tq.type == tk.type && tq.device == dev && tq.n[0] == n && tq.n[2] == tk.n[2] && tensor_as(q_out, tq, to, 3));
  kq_append_args a{};
  a.k = tk.p; a.v = tv.p; a.q = tq.p; a.q_out = to.p;
  a.k_tok = tk.s[0]; a.k_head = tk.s[1]; a.v_tok = tv.s[0]; a.v_head = tv.s[1];
  a.q_tok = tq.s[0]; a.q_head = tq.s[1]; a.o_tok = to.s[0]; a.o_head = to.s[1];
  a.table = static_cast<int32_t*>(tt.p); a.seq = static_cast<int32_t*>(ts.p); a.pos = static_cast<int32_t*>(tp.p);
  a.cos_t = static_cast<float*>(tc.p); a.sin_t = static_cast<float*>(tsn.p);
  a.table_ld = tt.n[0] > 1 ? tt.s[0] : tt.n[1];
  a.rope_ld = tc.n[0] > 1 ? tc.s[0] : tc.n[1];
  a.n = (int)n; a.n_heads = (int)tq.n[1]; a.src_type = tk.type;
  a.n_seq = (int)tt.n[0]; a.max_pages = (int)tt.n[1];
  a.rot = (int)(2 * tc.n[1]); a.n_pos = (int)tc.n[0];
  return kq_page_append(c, &a, stream);
}

extern "C" int kq_page_attend_tensors(kq_pages* c, void* q, void* table, void* len, void* out, void* seq, int window, float scale,
                                      void* stream) {
  FITS(c && stream_for(c->device, stream));
  const int dev = c->device;
  Tensor tq, to, tt, tl, ts;
  FITS(tensor_of(q, 3, tq) && tq.device == dev && tq.n[2] == c->d.head_dim && tensor_as(out, tq, to, 3));
  const long long n = tq.n[0];
  FITS(tensor_of(table, 2, tt) && tt.type == T_I32 && tt.device == dev && vector_as(len, T_I32, dev, n, tl));
  if (seq) FITS(vector_as(seq, T_I32, dev, n, ts));
  else FITS(n <= tt.n[0]);
  kq_attend_args a{};
  a.q = tq.p; a.out = to.p;
  a.q_tok = tq.s[0]; a.q_head = tq.s[1]; a.o_tok = to.s[0]; a.o_head = to.s[1];
  a.table = static_cast<int32_t*>(tt.p); a.seq = static_cast<int32_t*>(ts.p); a.len = static_cast<int32_t*>(tl.p);
  a.table_ld = tt.n[0] > 1 ? tt.s[0] : tt.n[1];
  a.n = (int)n; a.n_heads = (int)tq.n[1]; a.type = tq.type;
  a.n_seq = (int)tt.n[0]; a.max_pages = (int)tt.n[1]; a.window = window; a.scale = scale;
  return kq_page_attend(c, &a, stream);
}

extern "C" int kq_logit_rules_tensors(void* logits, void* out, void* best, void* hist, void* hist_len, void* prompt_len,
                                      void* repetition, void* frequency, void* presence, void* bias_id, void* bias, void* mask,
                                      void* mask_row, void* stream) {
  FITS(!hist == !hist_len && (hist || !prompt_len) && !bias_id == !bias && (mask || !mask_row));
  Tensor tl, to, tb, th, thl, tp, tr, tf, ts, ti, tv, tm, tmr;
  FITS(tensor_of(logits, 2, tl) && tensor_as(out, tl, to, 2));
  const int dev = tl.device;
  const long long n = tl.n[0];
  FITS(stream_for(dev, stream));
  if (best) FITS(vector_as(best, T_I32, dev, n, tb));
  if (hist) FITS(tensor_of(hist, 2, th) && th.type == T_I32 && th.device == dev && th.n[0] == n && vector_as(hist_len, T_I32, dev, n, thl));
  if (prompt_len) FITS(vector_as(prompt_len, T_I32, dev, n, tp));
  if (repetition) FITS(vector_as(repetition, KQ_F32, dev, n, tr));
  if (frequency) FITS(vector_as(frequency, KQ_F32, dev, n, tf));
  if (presence) FITS(vector_as(presence, KQ_F32, dev, n, ts));
  if (bias)
    FITS(tensor_of(bias_id, 2, ti) && ti.type == T_I32 && ti.device == dev && ti.n[0] == n && tensor_of(bias, 2, tv) &&
         tv.type == KQ_F32 && tv.device == dev && tv.n[0] == n && tv.n[1] == ti.n[1] && (n == 1 || tv.s[0] == ti.s[0]));
  if (mask) FITS(tensor_of(mask, 2, tm) && tm.type == T_I32 && tm.device == dev && tm.n[1] >= (tl.n[1] + 31) / 32);
  if (mask_row) FITS(vector_as(mask_row, T_I32, dev, n, tmr));
  kq_rule_args a{};
  auto ld = [](const Tensor& t) { return t.n[0] > 1 ? t.s[0] : t.n[1]; };
  a.logits = tl.p; a.out = to.p; a.in_ld = ld(tl); a.out_ld = ld(to);
  a.best = static_cast<int32_t*>(tb.p);
  a.hist = static_cast<int32_t*>(th.p); a.hist_len = static_cast<int32_t*>(thl.p); a.prompt_len = static_cast<int32_t*>(tp.p);
  a.hist_ld = ld(th);
  a.repetition = static_cast<float*>(tr.p); a.frequency = static_cast<float*>(tf.p); a.presence = static_cast<float*>(ts.p);
  a.bias_id = static_cast<int32_t*>(ti.p); a.bias = static_cast<float*>(tv.p); a.bias_ld = ld(ti);
  a.mask = static_cast<uint32_t*>(tm.p); a.mask_row = static_cast<int32_t*>(tmr.p); a.mask_ld = ld(tm);
  a.n = (int)n; a.vocab = (int)tl.n[1]; a.type = tl.type;
  a.max_hist = (int)th.n[1]; a.n_bias = (int)ti.n[1]; a.n_masks = (int)tm.n[0];
  return kq_logit_rules(&a, dev, stream);
}

std::string kqh_operands(int e) {
  std::string what;
  if (e & KQ_DEV_ERR_BAD_TOKEN) what += " token";
  if (e & KQ_DEV_ERR_BAD_POS) what += " position";
  if (e & KQ_DEV_ERR_BAD_PAGE) what += " page id";
  if (e & KQ_DEV_ERR_BAD_LEN) what += " length";
  if (e & KQ_DEV_ERR_BAD_ROW) what += " row index";
  return what;
}

// Reads and clears an error word in one step: what another stream's kernel flags meanwhile is kept for the next check.
__global__ void k_take_flags(int* word, int* taken) { *taken = atomicExch(word, 0); }

extern "C" int kq_stream_check(int device, void* stream) {
  static std::mutex mu[16];            // of each device's second word
  KqhDevice dev;
  const int rc = kqh_device(device, &dev);
  if (rc) return rc;
  const cudaStream_t s = (cudaStream_t)stream;
  CU(cudaStreamSynchronize(s));        // the long wait, without the lock
  int e = 0;
  {
    std::lock_guard<std::mutex> lk(mu[device]);
    k_take_flags<<<1, 1, 0, s>>>(dev.err, dev.err + 1);
    CU(cudaGetLastError());
    CU(cudaMemcpyAsync(&e, dev.err + 1, sizeof(int), cudaMemcpyDeviceToHost, s));
    CU(cudaStreamSynchronize(s));
  }
  return e ? kqh_error(KQ_ERR_ARG, "an operator met device operands out of range:" + kqh_operands(e)) : KQ_OK;
}
