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

struct kq_pages {
  kq_page_desc d{};
  int device = 0, shift = 0;
  KqhDevice dev{};
  AttendScratch scratch{};
};

// The attention kernel of a cache type, head size, query heads per CTA (8 or 16) and precision.
typedef void (*AttendFn)(AttendParams, AttendScratch);
struct AttendKernel {
  AttendFn fn;
  int smem;
};
template <int CT, int HD, int NT, bool PREC>
static AttendKernel attend_entry() {
  return {k_page_attend<CT, HD, NT, PREC>, PaShape<CT, HD, NT, PREC>::SMEM};
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
template <int ST>
static AppendFn append_of(int cache) {
  return cache == KQ_F16 ? k_page_append<ST, PG_F16> : cache == KQ_BF16 ? k_page_append<ST, PG_BF16> : k_page_append<ST, PG_E4M3>;
}
static AppendFn append_kernel(int src, int cache) {
  return src == KQ_F32 ? append_of<PG_F32>(cache) : src == KQ_F16 ? append_of<PG_F16>(cache) : append_of<PG_BF16>(cache);
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

extern "C" kq_pages* kq_pages_create(const kq_page_desc* d, int device) {
  KqhDevice dev;
  if (pages_check(d) || kqh_device(device, &dev)) return nullptr;
  kq_pages* c = new (std::nothrow) kq_pages;
  if (!c) {
    kqh_error(KQ_ERR_MEMORY, "page handle allocation");
    return nullptr;
  }
  c->d = *d;
  c->device = device;
  c->dev = dev;
  while ((1 << c->shift) < d->page) ++c->shift;
  const size_t part = (size_t)2 * PA_MAX_CTAS * PA_MAX_HEADS * PA_PLD * sizeof(float);
  cudaError_t e = cudaMalloc(&c->scratch.part, part + PA_MAX_CTAS * sizeof(int));
  if (e == cudaSuccess) {
    c->scratch.ticket = reinterpret_cast<int*>(reinterpret_cast<char*>(c->scratch.part) + part);
    e = cudaMemset(c->scratch.ticket, 0, PA_MAX_CTAS * sizeof(int));
  }
  for (int v = 0; v < 4 && e == cudaSuccess; ++v) {
    const AttendKernel k = attend_kernel(d->type, d->head_dim, v & 1, v & 2);
    e = cudaFuncSetAttribute(k.fn, cudaFuncAttributeMaxDynamicSharedMemorySize, k.smem);
  }
  if (e != cudaSuccess) {
    kqh_error(e == cudaErrorMemoryAllocation ? KQ_ERR_MEMORY : KQ_ERR_BACKEND,
              std::string("kq_pages_create: scratch allocation or kernel set-up: ") + cudaGetErrorString(e));
    kq_pages_free(c);
    return nullptr;
  }
  return c;
}

extern "C" void kq_pages_free(kq_pages* c) {
  if (!c) return;
  if (c->scratch.part) {
    cudaSetDevice(c->device);
    cudaFree(c->scratch.part);
  }
  delete c;
}

static PageTable table_of(const kq_pages* c, const int32_t* table, const int32_t* seq, long long ld, int n_seq, int max_pages) {
  return PageTable{table, seq, ld, n_seq, max_pages, c->d.n_pages, c->shift};
}
static bool table_ok(const kq_pages* c, const int32_t* table, const int32_t* seq, long long ld, int n_seq, int max_pages, int n) {
  return table && n_seq >= 1 && max_pages >= 1 && ld >= max_pages && (seq || n <= n_seq) &&
         (long long)max_pages * c->d.page <= 0x7fffffffll;
}

extern "C" int kq_page_append(kq_pages* c, const kq_append_args* a, void* stream) {
  REQUIRE(c && a, "kq_page_append: null argument");
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
  const int units = c->d.head_dim / (a->src_type == KQ_F32 ? 8 : 16), rows = a->n_heads + 2 * P.n_kv;
  const dim3 grid((unsigned)a->n, (unsigned)((rows * units + AP_THREADS - 1) / AP_THREADS));
  CU(launch(append_kernel(a->src_type, c->d.type), grid, AP_THREADS, 0, stream, 1, P));
  return KQ_OK;
}

extern "C" int kq_page_attend(kq_pages* c, const kq_attend_args* a, void* stream) {
  REQUIRE(c && a, "kq_page_attend: null argument");
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
  P.cache_type = c->d.type; P.window = a->window; P.scale = a->scale; P.err = c->dev.err;
  const int G = a->n_heads / P.n_kv;
  // fp32 queries want fp32 scores: the cache's 16-bit type in two or three terms; so do fp16 queries
  // (11 bits) on a bf16 cache (8 bits)
  const bool prec = a->type == KQ_F32 || (c->d.type == KQ_BF16 && a->type == KQ_F16);
  const AttendKernel k = attend_kernel(c->d.type, c->d.head_dim, G > 8, prec);
  const int heads = G > 8 ? 16 : 8;
  const long long tiles = (((long long)a->max_pages << c->shift) + PA_TILE - 1) / PA_TILE;
  const long long most = (long long)a->n * P.n_kv * ((G + heads - 1) / heads) * tiles;
  const int per_sm = k.smem > 110 * 1024 ? 1 : 2;
  const unsigned grid = (unsigned)std::min<long long>(most, std::min(PA_MAX_CTAS, c->dev.nsm * per_sm));
  CU(launch(k.fn, dim3(grid), PA_WARPS * 32, k.smem, stream, 1, P, c->scratch));
  return KQ_OK;
}

typedef void (*RulesFn)(RuleParams);
static RulesFn rules_kernel(int type) {
  return type == KQ_F32 ? k_logit_rules<float> : type == KQ_F16 ? k_logit_rules<__half> : k_logit_rules<__nv_bfloat16>;
}
// Shared memory and cluster sizes above the defaults, allowed once per device (which is current).
static int rules_setup(int device) {
  static std::atomic<bool> done[16];
  if (done[device].load(std::memory_order_acquire)) return KQ_OK;
  const int smem = (KQ_RULES_MAX_VOCAB / RL_CLUSTER + 16) * 8;
  for (int type : {KQ_F32, KQ_F16, KQ_BF16}) {
    CU(cudaFuncSetAttribute(rules_kernel(type), cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    CU(cudaFuncSetAttribute(rules_kernel(type), cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  }
  done[device].store(true, std::memory_order_release);
  return KQ_OK;
}

extern "C" int kq_logit_rules(const kq_rule_args* a, int device, void* stream) {
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
  KqhDevice dev;
  int rc = kqh_device(device, &dev);
  if (rc || a->n == 0) return rc;
  RuleParams P;
  P.in = a->logits; P.out = a->out; P.in_ld = a->in_ld; P.out_ld = a->out_ld; P.best = a->best;
  P.hist = a->hist; P.hist_len = a->hist_len; P.prompt_len = a->prompt_len; P.hist_ld = a->hist_ld;
  P.rep = a->repetition; P.freq = a->frequency; P.pres = a->presence;
  P.bias_id = a->bias_id; P.bias = a->bias; P.bias_ld = a->bias_ld;
  P.mask = a->mask; P.mask_row = a->mask_row; P.mask_ld = a->mask_ld;
  P.n = a->n; P.vocab = a->vocab; P.max_hist = a->max_hist; P.n_bias = a->n_bias; P.n_masks = a->n_masks; P.err = dev.err;
  const RulesFn fn = rules_kernel(a->type);
  // the smallest cluster whose CTAs hold their logits in registers (RL_PRE groups a thread), then larger
  // ones while the device has CTAs to spare
  const int vec = 16 / es, reach = a->vocab + vec - 1;
  int cl = 1;
  while (cl < RL_CLUSTER && (reach > cl * RL_PRE * RL_THREADS * vec || ((long long)a->n * cl * 2 <= dev.nsm && reach > cl * RL_THREADS * vec))) cl *= 2;
  P.span = ((reach + cl - 1) / cl + 15) / 16 * 16;
  const size_t smem = (size_t)P.span * 4 * ((P.hist ? 1 : 0) + (P.n_bias ? 1 : 0));
  if ((rc = rules_setup(device))) return rc;
  CU(launch(fn, dim3((unsigned)a->n * (unsigned)cl), RL_THREADS, smem, stream, cl, P));
  return KQ_OK;
}

extern "C" int kq_stream_check(int device, void* stream) {
  KqhDevice dev;
  const int rc = kqh_device(device, &dev);
  if (rc) return rc;
  CU(cudaStreamSynchronize((cudaStream_t)stream));
  int e = 0;
  CU(cudaMemcpy(&e, dev.err, sizeof(int), cudaMemcpyDeviceToHost));
  if (!e) return KQ_OK;
  CU(cudaMemset(dev.err, 0, sizeof(int)));
  std::string what = "an operator met device operands out of range:";
  if (e & KQ_DEV_ERR_BAD_POS) what += " position";
  if (e & KQ_DEV_ERR_BAD_PAGE) what += " page id";
  if (e & KQ_DEV_ERR_BAD_LEN) what += " length";
  if (e & KQ_DEV_ERR_BAD_ROW) what += " row index";
  return kqh_error(KQ_ERR_ARG, what);
}
