// mcpm_paged.h -- the paged cache and its batches as the kernels see them, and
// the launch functions of mcpm_paged.hip, mcpm_paged_attn.hip and
// mcpm_logits.hip.
#pragma once

#include "mcpm_internal.h"

namespace mcpm {

constexpr int PAGED_MAX_HD = 256;
constexpr int PAGED_MAX_PAGE = 65536;

// mcpm_paged_kv with the page size as shift and mask.
struct PagedView {
  char* k;
  char* v;
  float* weight;
  int64_t page_stride, pos_stride, head_stride;  // elements
  int n_pages, page_shift, page_mask, n_kv_heads, hd;
};

struct BatchView {
  const int* pages;
  const int* lens;
  const int* starts;
  int n_seq, n_rows, max_new, max_len, max_pages;
};

struct RuleView {
  float scale, softcap;
  int window;
  const float* slopes;
  const int* prefix;
  const int* docs;
  int64_t docs_stride;
};

// Where positions are in memory: every access of the kernels goes through these,
// whatever the arrays on the device hold.  They also run on the host.
// The positions of sequence b, inside every bound the caller gave.
__host__ __device__ inline int seq_len(const BatchView& bt, const PagedView& kv, int b) {
  const int64_t table = static_cast<int64_t>(bt.max_pages) << kv.page_shift;
  const int cap = table < bt.max_len ? static_cast<int>(table) : bt.max_len;
  const int len = bt.lens[b];
  return len < 0 ? 0 : len < cap ? len : cap;
}

// Rows [r0, r0 + n) of sequence b, inside the buffers; the first row's position
// is len - given, with `given` the row count before any bound.
struct SeqRows {
  int r0, n, given;
};
__host__ __device__ inline SeqRows seq_rows(const BatchView& bt, int b) {
  if (!bt.starts) return SeqRows{b, 1, 1};
  const int r0 = bt.starts[b], r1 = bt.starts[b + 1];
  if (r0 < 0 || r1 <= r0 || r0 >= bt.n_rows) return SeqRows{0, 0, 0};
  const int n = (r1 < bt.n_rows ? r1 : bt.n_rows) - r0;
  return SeqRows{r0, n < bt.max_new ? n : bt.max_new, r1 - r0};
}

// Page of a position below seq_len, or -1 when its number is outside the pool.
__host__ __device__ inline int page_of(const BatchView& bt, const PagedView& kv, int b, int pos) {
  const int p = bt.pages[static_cast<int64_t>(b) * bt.max_pages + (pos >> kv.page_shift)];
  return static_cast<unsigned>(p) < static_cast<unsigned>(kv.n_pages) ? p : -1;
}

// First element of kv head h at a position of a page.
__host__ __device__ inline int64_t elem_of(const PagedView& kv, int page, int pos, int h) {
  return page * kv.page_stride + static_cast<int64_t>(pos & kv.page_mask) * kv.pos_stride + h * kv.head_stride;
}

__host__ __device__ inline float* weight_of(const PagedView& kv, int page, int pos, int h) {
  return kv.weight + (((static_cast<int64_t>(page) * kv.n_kv_heads + h) << kv.page_shift) + (pos & kv.page_mask));
}

// io_type: MCPM_TYPE_F32 or kv_type.
hipError_t launch_paged_append(const PagedView& kv, int kv_type, const BatchView& bt, int io_type, const void* k,
                               const void* v, int64_t kv_stride, void* q, int64_t q_stride, int n_heads,
                               float rope_base, int n_cu, hipStream_t s);

// Bytes of scratch that launch_paged_attention needs.
size_t paged_attention_scratch(const PagedView& kv, int kv_type, const BatchView& bt, const RuleView& rl, int io_type, int n_heads, int n_cu);
hipError_t launch_paged_attention(const PagedView& kv, int kv_type, const BatchView& bt, const RuleView& rl, int io_type,
                                  void* out, int64_t out_stride, const void* q, int64_t q_stride, int n_heads,
                                  void* scratch, int n_cu, hipStream_t s);

// Bytes of scratch that launch_paged_evict needs.
size_t paged_evict_scratch(const PagedView& kv, const BatchView& bt, int first, int recent);
hipError_t launch_paged_evict(const PagedView& kv, int kv_type, const BatchView& bt, int budget, int first, int recent,
                              const int* dst_pages, int max_dst_pages, int* kept, int* dst_lens, void* scratch, hipStream_t s);

hipError_t launch_process_logits(float* logits, const mcpm_logit_rules& r, int n_cu, hipStream_t s);

}  // namespace mcpm
