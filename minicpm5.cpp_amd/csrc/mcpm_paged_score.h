// mcpm_paged_score.h -- what the attention kernels over the paged cache share:
// the rules of a row, its scores, and the split of 32-bit values into terms of
// a 16-bit type.
#pragma once

#include "mcpm_device.h"
#include "mcpm_paged.h"

namespace mcpm {

constexpr float LOG2E = 1.44269504088896340736f;
// The running maximum's start: finite, so that what is not seen (a score of
// -inf) has share 0 and a NaN stays one, and below the scores that 32 bits hold
// but for the last bit of their exponent.
constexpr float MAX_START = -3e38f;

typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

template <typename TC>
struct Half;  // the 16-bit matrix instructions of a type
template <>
struct Half<_Float16> {
  typedef h16x8 V8;
  static __device__ __forceinline__ f32x4 mma16(V8 a, V8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ f32x16 mma32(V8 a, V8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Half<__bf16> {
  typedef b16x8 V8;
  static __device__ __forceinline__ f32x4 mma16(V8 a, V8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ f32x16 mma32(V8 a, V8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};

// Terms that a 32-bit factor takes in products with a cache of type TC, rows
// of type TI.  A half holds 11 bits and a bfloat16 8, so two halves or three
// bfloat16 hold what 24 bits hold to 2^-22 and 2^-24; rows of the cache's own
// type are one term, and their shares p are rounded to it once.
template <typename TC, typename TI>
struct Terms {
  static constexpr int N = sizeof(TI) == 2 ? 1 : sizeof(TC) == 4 ? 1 : __is_same(TC, _Float16) ? 2 : 3;
};

template <typename TC, int N, int M>
__device__ __forceinline__ void split_terms(const float (&x)[M], typename Half<TC>::V8* t) {
  static_assert(M == 8);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float r = x[i];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const TC c = static_cast<TC>(r);
      t[n][i] = c;
      if (n + 1 < N) r -= static_cast<float>(c);
    }
  }
}

// tanh below 0.3 by its series to x^11 (the next term is 2e-9 of it).
constexpr float TANH_SERIES = 0.3f;
__device__ __forceinline__ float tanh_small(float x) {
  const float x2 = x * x;
  float p = -8.8632355299e-3f;
  p = __builtin_fmaf(p, x2, 2.1869488536e-2f);
  p = __builtin_fmaf(p, x2, -5.3968253968e-2f);
  p = __builtin_fmaf(p, x2, 1.3333333333e-1f);
  p = __builtin_fmaf(p, x2, -3.3333333333e-1f);
  return __builtin_fmaf(x * x2, p, x);
}
// Above from exp(-2x) as (1 - e) / (1 + e), whose numerator is exact where it is small.
__device__ __forceinline__ float tanh_f32(float x) {
  const float a = fabsf(x);
  const float e = __builtin_amdgcn_exp2f(a * (-2.0f * LOG2E));
  const float large = (1.0f - e) * __builtin_amdgcn_rcpf(1.0f + e);
  return a < TANH_SERIES ? tanh_small(x) : __builtin_copysignf(large, x);
}

// Scores in units of log2: p = 2^(s - m).  `mul` takes a raw product q.k to the
// score, or to the cap's argument; `cap` is the cap then.
struct ScoreRule {
  float mul, cap;
  bool capped;
};
__device__ __forceinline__ ScoreRule score_rule(const RuleView& rl) {
  const bool capped = rl.softcap > 0.0f;
  return capped ? ScoreRule{rl.scale / rl.softcap, rl.softcap * LOG2E, true} : ScoreRule{rl.scale * LOG2E, 0.0f, false};
}
__device__ __forceinline__ float score_of(const ScoreRule& sr, float dot, float mul) {
  const float s = dot * mul;
  return sr.capped ? sr.cap * tanh_f32(s) : s;
}

// N scores of a lane at once: caps are seldom near, so a wave whose arguments are
// all small takes the series alone.
template <int N, class Dots>
__device__ __forceinline__ void scores_of(const ScoreRule& sr, Dots& s, float mul) {
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] *= mul;
  if (!sr.capped) return;
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) top = fmaxf(top, fabsf(s[i]));
  if (__any(!(top < TANH_SERIES))) {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = sr.cap * tanh_f32(s[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = sr.cap * tanh_small(s[i]);
  }
}

// What a row sees: the positions j with 0 <= j - lo < span whose tag is the row's.  A
// position's tag is its document, 0 without documents; HIDDEN_TAG where its page is
// outside the pool.
constexpr int HIDDEN_TAG = -2;
struct RowRule {
  int lo;
  unsigned span;
  int tag;
};
// pos < 0 (no row, or one before the start) sees nothing, as does a row of no document.
__device__ __forceinline__ RowRule row_rule(const RuleView& rl, int b, int pos, int end) {
  if (pos < 0) return RowRule{0, 0, 0};
  const int tag = rl.docs ? rl.docs[b * rl.docs_stride + pos] : 0;
  const int hi = min(max(pos + 1, rl.prefix ? rl.prefix[b] : 0), end);
  const int lo = rl.window > 0 ? max(pos - rl.window + 1, 0) : 0;
  return RowRule{lo, tag < 0 || hi <= lo ? 0u : static_cast<unsigned>(hi - lo), tag};
}
__device__ __forceinline__ bool in_span(const RowRule& r, int j) { return static_cast<unsigned>(j - r.lo) < r.span; }
// The tag of position j, which has to be below the sequence's length.
__device__ __forceinline__ int tag_of(const RuleView& rl, const BatchView& bt, const PagedView& kv, int b, int j, bool bad_pages) {
  const int tag = rl.docs ? rl.docs[b * rl.docs_stride + j] : 0;
  return bad_pages && page_of(bt, kv, b, j) < 0 ? HIDDEN_TAG : tag;
}

// Positions [lo, hi) that rows at pos0 .. pos1 may see, lo at a multiple of 64.
struct KeyRange {
  int lo, hi;
};
__device__ __forceinline__ KeyRange key_range(const RuleView& rl, int b, int pos0, int pos1, int len) {
  int lo = rl.window > 0 ? max(0, max(pos0, 0) - rl.window + 1) : 0;
  int hi = pos1 + 1;
  if (rl.prefix) hi = max(hi, rl.prefix[b]);
  hi = min(hi, len);
  if (pos1 < 0) hi = 0;
  return KeyRange{lo & ~63, hi};
}

// A call as its kernels see it.  A row block is `block_rows` rows of a sequence
// (new tokens x the kv head's query heads, token by token).  The prompt kernel cuts a
// block's positions into chunks of `chunk`, a work group each; the few-row kernel
// shares them out by the lengths that it finds (few_share).
struct PagedCall {
  PagedView kv;
  BatchView bt;
  RuleView rl;
  const void* q;
  void* out;
  int64_t q_stride, out_stride;
  int n_heads, group, block_rows, n_blocks;  // query heads per kv head; row blocks per (sequence, kv head)
  int chunk, n_splits;  // few rows: work groups wanted, and whether there can be more than one to a block
  bool by_xcd;          // few rows: consecutive parts of the work on one XCD
  float* part_o;    // unnormalised: [seq][new token][head][split][hd]; few rows: [work group][row of the block][hd]
  float2* part_mz;  // the same without [hd]
  float2* row_mz;   // [seq][new token][head]: the rows' own, with weights
  int2* seq_wgs;    // few rows: [seq] the first work group and the chunks of a block
  float* scores;    // few rows with weights: [seq][kv head][row of the sequence][score_len], or null
  int score_len, score_rows;
};

__device__ __forceinline__ int64_t part_index(const PagedCall& a, int b, int t, int head, int split) {
  return ((static_cast<int64_t>(b) * a.bt.max_new + t) * a.n_heads + head) * a.n_splits + split;
}

__device__ __forceinline__ int64_t row_index(const PagedCall& a, int b, int t, int head) {
  return (static_cast<int64_t>(b) * a.bt.max_new + t) * a.n_heads + head;
}

// The positions of a row block.
struct RowBlock {
  int r_end;  // rows of the sequence
  int pos0;   // position of the sequence's first new token
  int first, last;  // positions of the block's first and last row
  KeyRange keys;
};
__device__ __forceinline__ RowBlock row_block(const PagedCall& a, int b, int rb, const SeqRows& sr, int len) {
  const int pos0 = len - sr.given, r_end = sr.n * a.group;
  const int first = pos0 + rb * a.block_rows / a.group;
  const int last = pos0 + (min(rb * a.block_rows + a.block_rows, r_end) - 1) / a.group;
  return RowBlock{r_end, pos0, first, last, key_range(a.rl, b, first, last, len)};
}

// Page offsets of a chunk (a page outside the pool stands at the first one, to be masked);
// whether all of this lane's are in the pool.
__device__ __forceinline__ bool load_page_offsets(const BatchView& bt, const PagedView& kv, int b, int c0, int c1, int64_t* s_off) {
  bool ok = true;
  const int first = c0 >> kv.page_shift, n = ((c1 - 1) >> kv.page_shift) - first + 1;
  for (int i = threadIdx.x; i < n; i += 256) {
    const int page = page_of(bt, kv, b, (first + i) << kv.page_shift);
    s_off[i] = page < 0 ? 0 : page * kv.page_stride;
    ok = ok && page >= 0;
  }
  return ok;
}

// The call's own copy in the kernel's arguments: what the rare ends of a kernel need
// is read again there rather than held in scalar registers through its loops.
__device__ __forceinline__ const PagedCall& call_again() {
  // in the constant address space until the last cast: the loads stay scalar
  const __attribute__((address_space(4))) void* p = (const __attribute__((address_space(4))) void*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const PagedCall*)p;
}

// The plain computation of one row over positions [c0, c1), by the whole work
// group, for values that the matrix products cannot keep apart: a share of 0
// times what a masked place holds.  Returns this lane's element tid of sum
// p v, and (m, z).
template <typename TC, typename TI>
__device__ __forceinline__ float exact_row(const PagedCall& a, int b, int kh, int row, int head, int pos, int c0, int c1, float* s_q,
                                        float* s_p, float* s_red, float2* mz) {
  const PagedView& kv = a.kv;
  const int tid = threadIdx.x, hd = kv.hd;
  __syncthreads();
  if (tid < hd) s_q[tid] = static_cast<float>(static_cast<const TI*>(a.q)[row * a.q_stride + head * hd + tid]);
  __syncthreads();
  const ScoreRule sr = score_rule(a.rl);
  const RowRule rr = row_rule(a.rl, b, pos, c1);
  const float slope = a.rl.slopes ? a.rl.slopes[head] * LOG2E : 0.0f;
  float m = MAX_START, z = 0.0f, o = 0.0f;
  for (int j0 = c0; j0 < c1; j0 += 256) {
    const int j = j0 + tid;
    float s = -__builtin_inff();
    const int page = in_span(rr, j) && tag_of(a.rl, a.bt, kv, b, j, false) == rr.tag ? page_of(a.bt, kv, b, j) : -1;
    if (page >= 0) {
      const TC* k = reinterpret_cast<const TC*>(kv.k) + elem_of(kv, page, j, kh);
      float d = 0.0f;
      for (int i = 0; i < hd; ++i) d = __builtin_fmaf(s_q[i], static_cast<float>(k[i]), d);
      s = score_of(sr, d, sr.mul) - slope * fabsf(static_cast<float>(pos - j));
    }
    float w = wave_max(s);
    if ((tid & 63) == 0) s_red[tid >> 6] = w;
    __syncthreads();
    w = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
    const float mn = fmaxf(m, w), scale = __builtin_amdgcn_exp2f(m - mn);
    m = mn;
    s_p[tid] = __builtin_amdgcn_exp2f(s - m);
    __syncthreads();
    z *= scale;
    o *= scale;
    for (int i = 0; i < min(256, c1 - j0); ++i) {
      const float p = s_p[i];
      if (p == 0.0f) continue;
      z += p;
      if (tid < hd) {
        const int pg = page_of(a.bt, kv, b, j0 + i);  // p != 0: in the pool
        if (pg >= 0) o = __builtin_fmaf(p, static_cast<float>((reinterpret_cast<const TC*>(kv.v) + elem_of(kv, pg, j0 + i, kh))[tid]), o);
      }
    }
    __syncthreads();
  }
  *mz = make_float2(m, z);
  return o;
}

// exact_row for the rows of a block over positions [c0, c1) (the rows that `bad` marks,
// all without it), stored as the block's own were: at part_at(i, t, head) unless final.
template <typename TC, typename TI, class PartAt>
__device__ __forceinline__ void exact_rows(int b, int kh, int rb, int rows, int c0, int c1, bool final, const unsigned char* bad, float* s_q, float* s_p,
                                           float* s_red, const PartAt& part_at) {
  const PagedCall& a = call_again();
  const int tid = threadIdx.x, hd = a.kv.hd;
  const SeqRows sr = seq_rows(a.bt, b);
  const int pos0 = seq_len(a.bt, a.kv, b) - sr.given, r_end = sr.n * a.group;
#pragma unroll 1
  for (int i = 0; i < rows && rb * rows + i < r_end; ++i) {
    if (bad && !bad[i]) continue;
    const int r = rb * rows + i, t = r / a.group, head = kh * a.group + r - t * a.group;
    float2 mz;
    const float o = exact_row<TC, TI>(a, b, kh, sr.r0 + t, head, pos0 + t, c0, c1, s_q, s_p, s_red, &mz);
    const int64_t at = part_at(a, i, t, head);
    if (tid < hd) {
      if (final) static_cast<TI*>(a.out)[(sr.r0 + t) * a.out_stride + head * hd + tid] = static_cast<TI>(mz.y == 0.0f ? 0.0f : o / mz.y);
      else a.part_o[at * hd + tid] = o;
    }
    if (tid == 0) {
      if (a.part_mz) a.part_mz[at] = mz;
      if (final && a.row_mz) a.row_mz[row_index(a, b, t, head)] = mz;
    }
  }
}

// The prompt kernels (mcpm_paged_prompt.hip): row blocks of prompt_block_rows rows.
int prompt_block_rows();
hipError_t launch_attention_prompt(const PagedCall& a, int kv_type, int io_type, hipStream_t s);

}  // namespace mcpm
