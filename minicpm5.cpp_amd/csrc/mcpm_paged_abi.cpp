// mcpm_paged_abi.cpp -- C ABI of the operators over many sequences: argument
// checks, scratch and launches of the paged cache and the logit rules.
#include <cmath>

#include "mcpm_host.h"
#include "mcpm_paged.h"

using namespace mcpm;

namespace {

// The context's device current for one call, the caller's again after it.
class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    if (hipGetDevice(&old_) != hipSuccess) old_ = device;
    if (old_ != device) status_ = hipSetDevice(device);
    now_ = device;
  }
  ~DeviceScope() {
    if (old_ != now_) (void)hipSetDevice(old_);
  }
  hipError_t status() const { return status_; }

 private:
  int old_ = 0, now_ = 0;
  hipError_t status_ = hipSuccess;
};

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
int elem_bytes(int type) { return type == MCPM_TYPE_F32 ? 4 : 2; }

int view_kv(const mcpm_paged_kv* kv, const char* fn, PagedView& out) {
  if (!kv) return fail(MCPM_ERR_ARG, std::string(fn) + ": null cache");
  if (kv->type != MCPM_TYPE_F32 && kv->type != MCPM_TYPE_F16 && kv->type != MCPM_TYPE_BF16)
    return fail(MCPM_ERR_UNSUPPORTED, std::string(fn) + ": cache type must be F32, F16 or BF16");
  if (!kv->k || !kv->v || !aligned16(kv->k) || !aligned16(kv->v))
    return fail(MCPM_ERR_ARG, std::string(fn) + ": k and v must be 16-byte aligned device memory");
  if (kv->n_pages <= 0 || kv->page_size <= 0 || kv->page_size > PAGED_MAX_PAGE || (kv->page_size & (kv->page_size - 1)))
    return fail(MCPM_ERR_ARG, std::string(fn) + ": page_size must be a power of two up to 65536, n_pages positive");
  if (kv->n_kv_heads <= 0 || kv->n_kv_heads > 65535 || kv->head_dim <= 0 || kv->head_dim > PAGED_MAX_HD || kv->head_dim % 8)
    return fail(MCPM_ERR_ARG, std::string(fn) + ": head_dim must be a multiple of 8 up to 256, n_kv_heads 1 .. 65535");
  const int64_t step = 16 / elem_bytes(kv->type);
  for (const int64_t st : {kv->page_stride, kv->pos_stride, kv->head_stride})
    if (st < kv->head_dim || st % step) return fail(MCPM_ERR_ARG, std::string(fn) + ": strides must be multiples of 16 bytes, at least head_dim");
  if (kv->pos_stride > INT32_MAX || kv->head_stride > INT32_MAX)
    return fail(MCPM_ERR_ARG, std::string(fn) + ": pos_stride and head_stride must be less than 2^31");
  if (!aligned16(kv->weight)) return fail(MCPM_ERR_ARG, std::string(fn) + ": weight must be 16-byte aligned");
  int shift = 0;
  while ((1 << shift) < kv->page_size) ++shift;
  out = PagedView{static_cast<char*>(kv->k), static_cast<char*>(kv->v), kv->weight, kv->page_stride, kv->pos_stride,
                  kv->head_stride, kv->n_pages, shift, kv->page_size - 1, kv->n_kv_heads, kv->head_dim};
  return MCPM_OK;
}

int view_batch(const mcpm_paged_batch* b, bool rows, const char* fn, BatchView& out) {
  if (!b) return fail(MCPM_ERR_ARG, std::string(fn) + ": null batch");
  if (b->n_seq < 0 || b->n_seq > 65535 || b->max_len < 0 || b->max_len > (1 << 30) || b->max_pages < 0)
    return fail(MCPM_ERR_ARG, std::string(fn) + ": bad batch (n_seq 0 .. 65535, max_len up to 2^30)");
  if (b->n_seq && (!b->lens || (b->max_pages && !b->pages)))
    return fail(MCPM_ERR_ARG, std::string(fn) + ": null pages or lens");
  if (rows) {
    if (b->n_rows < 0 || b->max_new < 0) return fail(MCPM_ERR_ARG, std::string(fn) + ": negative rows");
    if (!b->starts && (b->n_rows < b->n_seq || b->max_new < 1) && b->n_seq)
      return fail(MCPM_ERR_ARG, std::string(fn) + ": without starts every sequence has one row");
  }
  out = BatchView{b->pages, b->lens, b->starts, b->n_seq, b->n_rows, b->starts ? b->max_new : 1, b->max_len, b->max_pages};
  if (rows && out.max_new > b->n_rows) out.max_new = b->n_rows;
  return MCPM_OK;
}

int check_rows(const void* p, int64_t stride, int heads, int hd, int type, const char* fn, const char* what) {
  if (!p || !aligned16(p) || stride < static_cast<int64_t>(heads) * hd || stride % (16 / elem_bytes(type)))
    return fail(MCPM_ERR_ARG, std::string(fn) + ": " + what + " rows must be 16-byte aligned, their stride a multiple of 16 bytes "
                                  "and at least heads * head_dim");
  return MCPM_OK;
}

int check_io(int io_type, int kv_type, const char* fn) {
  if (io_type != MCPM_TYPE_F32 && io_type != kv_type)
    return fail(MCPM_ERR_UNSUPPORTED, std::string(fn) + ": rows must be F32 or of the cache's type");
  return MCPM_OK;
}

// The context's scratch for the paged operators.  Growing waits for the stream:
// work already queued may use the old memory.
int ensure_paged_scratch(mcpm_ctx* c, size_t bytes) {
  if (bytes <= c->paged_cap) return MCPM_OK;
  if (c->d_paged) {
    MCPM_HIP(hipStreamSynchronize(c->stream));
    (void)hipFree(c->d_paged);
  }
  c->d_paged = nullptr;
  c->paged_cap = 0;
  MCPM_HIP(hipMalloc(&c->d_paged, bytes));
  c->paged_cap = bytes;
  return MCPM_OK;
}

}  // namespace

extern "C" {

int mcpm_paged_append(mcpm_ctx* c, const mcpm_paged_kv* kv, const mcpm_paged_batch* batch, int io_type, const void* k,
                      const void* v, int64_t kv_stride, void* q, int64_t q_stride, int n_heads, float rope_base) {
  const char* fn = "mcpm_paged_append";
  PagedView kvv;
  BatchView bt;
  int rc = view_kv(kv, fn, kvv);
  if (!rc) rc = view_batch(batch, true, fn, bt);
  if (!rc) rc = check_io(io_type, kv->type, fn);
  if (!rc) rc = check_rows(k, kv_stride, kv->n_kv_heads, kv->head_dim, io_type, fn, "k");
  if (!rc) rc = check_rows(v, kv_stride, kv->n_kv_heads, kv->head_dim, io_type, fn, "v");
  if (!rc && q && n_heads <= 0) rc = fail(MCPM_ERR_ARG, std::string(fn) + ": n_heads must be positive");
  if (!rc && q) rc = check_rows(q, q_stride, n_heads, kv->head_dim, io_type, fn, "q");
  if (!rc && !(rope_base >= 0.0f && std::isfinite(rope_base))) rc = fail(MCPM_ERR_ARG, std::string(fn) + ": bad rope_base");
  if (rc) return rc;
  if (!c) return fail(MCPM_ERR_ARG, std::string(fn) + ": null context");
  if (!bt.n_seq || !bt.n_rows || !bt.max_new) return MCPM_OK;
  DeviceScope dev(c->device);
  MCPM_HIP(dev.status());
  MCPM_HIP(launch_paged_append(kvv, kv->type, bt, io_type, k, v, kv_stride, q, q_stride, n_heads, rope_base, c->n_cu, c->stream));
  return MCPM_OK;
}

int mcpm_paged_attention(mcpm_ctx* c, void* out, int64_t out_stride, const void* q, int64_t q_stride, int io_type,
                         int n_heads, const mcpm_paged_kv* kv, const mcpm_paged_batch* batch, const mcpm_attn_rules* rules) {
  const char* fn = "mcpm_paged_attention";
  PagedView kvv;
  BatchView bt;
  int rc = view_kv(kv, fn, kvv);
  if (!rc) rc = view_batch(batch, true, fn, bt);
  if (!rc) rc = check_io(io_type, kv->type, fn);
  if (!rc && (n_heads <= 0 || n_heads > 65535 || n_heads % kv->n_kv_heads))
    rc = fail(MCPM_ERR_ARG, std::string(fn) + ": n_heads must be a multiple of n_kv_heads");
  if (!rc) rc = check_rows(q, q_stride, n_heads, kv->head_dim, io_type, fn, "q");
  if (!rc) rc = check_rows(out, out_stride, n_heads, kv->head_dim, io_type, fn, "out");
  if (!rc && static_cast<int64_t>(bt.max_new) * n_heads > INT32_MAX)
    rc = fail(MCPM_ERR_ARG, std::string(fn) + ": max_new * n_heads must be less than 2^31");
  if (rc) return rc;
  RuleView rl{};
  if (rules) {
    constexpr float most = 1e38f;  // times log2(e) still finite
    if (!(std::fabs(rules->scale) <= most) || !(rules->softcap >= 0.0f && rules->softcap <= most) || rules->window < 0)
      return fail(MCPM_ERR_ARG, std::string(fn) + ": scale must be finite, softcap and window not negative, none past 1e38");
    if (rules->softcap > 0.0f && !(std::fabs(rules->scale / rules->softcap) <= most))
      return fail(MCPM_ERR_ARG, std::string(fn) + ": scale / softcap must not be past 1e38");
    if (rules->docs && rules->docs_stride < bt.max_len)
      return fail(MCPM_ERR_ARG, std::string(fn) + ": docs_stride is less than max_len");
    rl = RuleView{rules->scale, rules->softcap, rules->window, rules->slopes, rules->prefix, rules->docs, rules->docs_stride};
  }
  if (rl.scale == 0.0f) rl.scale = static_cast<float>(1.0 / std::sqrt(static_cast<double>(kv->head_dim)));
  if (!c) return fail(MCPM_ERR_ARG, std::string(fn) + ": null context");
  if (!bt.n_seq || !bt.n_rows || !bt.max_new) return MCPM_OK;
  DeviceScope dev(c->device);
  MCPM_HIP(dev.status());
  rc = ensure_paged_scratch(c, paged_attention_scratch(kvv, kv->type, bt, rl, io_type, n_heads, c->n_cu));
  if (rc) return rc;
  MCPM_HIP(launch_paged_attention(kvv, kv->type, bt, rl, io_type, out, out_stride, q, q_stride, n_heads, c->d_paged, c->n_cu, c->stream));
  return MCPM_OK;
}

int mcpm_paged_evict(mcpm_ctx* c, const mcpm_paged_kv* kv, const mcpm_paged_batch* batch, int budget, int first, int recent,
                     const int* dst_pages, int max_dst_pages, int* kept, int* dst_lens) {
  const char* fn = "mcpm_paged_evict";
  PagedView kvv;
  BatchView bt;
  int rc = view_kv(kv, fn, kvv);
  if (!rc) rc = view_batch(batch, false, fn, bt);
  if (rc) return rc;
  if (!kv->weight || !dst_pages || !kept || !dst_lens) return fail(MCPM_ERR_ARG, std::string(fn) + ": null weight, dst_pages, kept or dst_lens");
  if (dst_pages == batch->pages || dst_lens == batch->lens)
    return fail(MCPM_ERR_ARG, std::string(fn) + ": dst_pages and dst_lens must be memory of their own");
  if (budget <= 0 || first < 0 || recent < 0 || first > budget - recent)
    return fail(MCPM_ERR_ARG, std::string(fn) + ": first + recent must be within a positive budget");
  if (max_dst_pages <= 0 || (static_cast<int64_t>(max_dst_pages) << kvv.page_shift) < budget)
    return fail(MCPM_ERR_ARG, std::string(fn) + ": dst_pages holds less than budget positions");
  if (!c) return fail(MCPM_ERR_ARG, std::string(fn) + ": null context");
  if (!bt.n_seq) return MCPM_OK;
  DeviceScope dev(c->device);
  MCPM_HIP(dev.status());
  rc = ensure_paged_scratch(c, paged_evict_scratch(kvv, bt, first, recent));
  if (rc) return rc;
  MCPM_HIP(launch_paged_evict(kvv, kv->type, bt, budget, first, recent, dst_pages, max_dst_pages, kept, dst_lens, c->d_paged, c->stream));
  return MCPM_OK;
}

int mcpm_process_logits(mcpm_ctx* c, float* logits, const mcpm_logit_rules* r) {
  const char* fn = "mcpm_process_logits";
  if (!logits || !r) return fail(MCPM_ERR_ARG, std::string(fn) + ": null argument");
  if (r->n_seq < 0 || r->n_seq > 65535 || r->vocab <= 0 || r->vocab > (1 << 30) || r->stride < r->vocab)
    return fail(MCPM_ERR_ARG, std::string(fn) + ": n_seq must be 0 .. 65535, vocab 1 .. 2^30, stride at least vocab");
  if ((r->history != nullptr) != (r->history_starts != nullptr) || (r->bias != nullptr) != (r->bias_ids != nullptr) ||
      (r->bias != nullptr) != (r->bias_starts != nullptr))
    return fail(MCPM_ERR_ARG, std::string(fn) + ": a list and its starts come together");
  if (r->allowed && r->allowed_stride < (static_cast<int64_t>(r->vocab) + 31) / 32)
    return fail(MCPM_ERR_ARG, std::string(fn) + ": allowed_stride is less than the vocabulary's words");
  if (!c) return fail(MCPM_ERR_ARG, std::string(fn) + ": null context");
  if (!r->n_seq) return MCPM_OK;
  DeviceScope dev(c->device);
  MCPM_HIP(dev.status());
  MCPM_HIP(launch_process_logits(logits, *r, c->n_cu, c->stream));
  return MCPM_OK;
}

}  // extern "C"
