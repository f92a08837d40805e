// mcpm_paged_score.h -- what the attention kernels over the paged cache share:
// the rules of a row, its scores, and the split of 32-bit values into terms of
// a 16-bit type.
#pragma once

#include "mcpm_device.h"
#include "mcpm_paged.h"

namespace mcpm {

constexpr float LOG2E = 1.44269504088896340736f;
// The running maximum's start: finite, so that what is not seen (a score of
// -inf) has share 0 and a NaN stays one.
constexpr float MAX_START = -1e30f;

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

// tanh: by its series to x^11 below 0.3 (the next term is 2e-9 of it), from
// exp(2x) above.
__device__ __forceinline__ float tanh_f32(float x) {
  const float a = fabsf(x), x2 = x * x;
  float p = -8.8632355299e-3f;
  p = __builtin_fmaf(p, x2, 2.1869488536e-2f);
  p = __builtin_fmaf(p, x2, -5.3968253968e-2f);
  p = __builtin_fmaf(p, x2, 1.3333333333e-1f);
  p = __builtin_fmaf(p, x2, -3.3333333333e-1f);
  const float small = __builtin_fmaf(x * x2, p, x);
  const float e = __builtin_amdgcn_exp2f(a * (2.0f * LOG2E));
  const float large = 1.0f - 2.0f * __builtin_amdgcn_rcpf(e + 1.0f);
  return a < 0.3f ? small : __builtin_copysignf(large, x);
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

// A row's place under the rules; pos < 0 (no row, or one of no document) sees nothing.
struct RowRule {
  int pos, prefix, window, doc;
};
__device__ __forceinline__ RowRule row_rule(const RuleView& rl, int b, int pos) {
  RowRule r{pos, rl.prefix ? rl.prefix[b] : 0, rl.window > 0 ? rl.window : 0x7fffffff, 0};
  if (rl.docs && pos >= 0) {
    r.doc = rl.docs[b * rl.docs_stride + pos];
    if (r.doc < 0) r.pos = -1;
  }
  if (r.pos < 0) r.prefix = 0;
  return r;
}
// Whether the row sees position j, 0 <= j < the sequence's length.
__device__ __forceinline__ bool seen(const RuleView& rl, const RowRule& r, int b, int j) {
  bool ok = (j <= r.pos) | (j < r.prefix);
  ok &= r.pos - j < r.window;
  if (rl.docs) ok &= rl.docs[b * rl.docs_stride + j] == r.doc;
  return ok;
}

// Positions [lo, hi) that rows at pos0 .. pos1 may see, lo at a multiple of 32.
struct KeyRange {
  int lo, hi;
};
__device__ __forceinline__ KeyRange key_range(const RuleView& rl, int b, int pos0, int pos1, int len) {
  int lo = rl.window > 0 ? max(0, max(pos0, 0) - rl.window + 1) : 0;
  int hi = pos1 + 1;
  if (rl.prefix) hi = max(hi, rl.prefix[b]);
  hi = min(hi, len);
  if (pos1 < 0) hi = 0;
  return KeyRange{lo & ~31, hi};
}

}  // namespace mcpm
