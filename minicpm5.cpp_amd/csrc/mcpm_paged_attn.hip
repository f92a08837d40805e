// mcpm_paged_attn.hip -- attention over the paged cache.
//
//   s_j = scale * q.k_j;  cap: c tanh(s/c);  - slope |i - j|;  seen: see mcpm_attn_rules
//   o = sum_j p_j v_j,  p_j = exp(s_j - m) / z over the seen j;  weight_j += p_j
#include "mcpm_device.h"
#include "mcpm_paged.h"

namespace mcpm {

namespace {

constexpr float NEG_INF = -__builtin_inff();
// The running maximum's start: finite, so that what is not seen (a score of
// -inf) has share 0 and a NaN stays one.
constexpr float MAX_START = -1e30f;

struct RowRule {
  int pos, prefix, doc;
  const int* docs;
};

__device__ __forceinline__ RowRule row_rule(const RuleView& rl, int b, int pos) {
  RowRule r{pos, rl.prefix ? rl.prefix[b] : 0, 0, rl.docs ? rl.docs + b * rl.docs_stride : nullptr};
  if (r.docs) r.doc = r.docs[pos];
  return r;
}

__device__ __forceinline__ bool seen(const RuleView& rl, const RowRule& r, int j) {
  if (j > r.pos && j >= r.prefix) return false;
  if (rl.window > 0 && r.pos - j >= rl.window) return false;
  return !r.docs || (r.doc >= 0 && r.docs[j] == r.doc);
}

__device__ __forceinline__ float rule_score(const RuleView& rl, float slope, float dot, int pos, int j) {
  float s = dot * rl.scale;
  if (rl.softcap > 0.0f) s = rl.softcap * tanhf(s / rl.softcap);
  return s - slope * fabsf(static_cast<float>(pos - j));
}

template <typename TC>
__device__ __forceinline__ float dot_row(const float* q, const TC* k, int hd) {
  float a = 0.0f;
  for (int d = 0; d < hd; ++d) a = __builtin_fmaf(q[d], static_cast<float>(k[d]), a);
  return a;
}

// One work group per (new token, query head): 256 positions at a time, a lane
// each for the scores, then a lane per output element for the sum over v.
template <typename TC, typename TI>
__global__ void __launch_bounds__(256) k_paged_attention(PagedView kv, BatchView bt, RuleView rl, TI* __restrict__ out,
                                                         int64_t out_stride, const TI* __restrict__ q, int64_t q_stride,
                                                         int n_heads, float2* __restrict__ mz) {
  __shared__ float s_q[PAGED_MAX_HD], s_p[256], s_red[4];
  const int h = blockIdx.x, t = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, hd = kv.hd;
  const SeqRows sr = seq_rows(bt, b);
  if (t >= sr.n) return;
  const int row = sr.r0 + t, len = seq_len(bt, kv, b), pos = len - sr.given + t;
  const int kh = h / (n_heads / kv.n_kv_heads);
  if (tid < hd) s_q[tid] = static_cast<float>(q[row * q_stride + h * hd + tid]);
  __syncthreads();
  float m = MAX_START, z = 0.0f, o = 0.0f;
  if (pos >= 0) {
    const RowRule rr = row_rule(rl, b, pos);
    const float slope = rl.slopes ? rl.slopes[h] : 0.0f;
    for (int j0 = 0; j0 < len; j0 += 256) {
      const int j = j0 + tid;
      float s = NEG_INF;
      if (j < len && seen(rl, rr, j)) {
        const int page = page_of(bt, kv, b, j);
        if (page >= 0)
          s = rule_score(rl, slope, dot_row(s_q, reinterpret_cast<const TC*>(kv.k) + elem_of(kv, page, j, kh), hd), pos, j);
      }
      float w = wave_max(s);
      if ((tid & 63) == 0) s_red[tid >> 6] = w;
      __syncthreads();
      w = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
      const float mn = fmaxf(m, w);
      {
        const float scale = expf(m - mn);
        m = mn;
        s_p[tid] = expf(s - m);
        __syncthreads();
        z *= scale;
        o *= scale;
        for (int i = 0; i < min(256, len - j0); ++i) {
          const float p = s_p[i];
          if (p == 0.0f) continue;
          z += p;
          if (tid < hd) {
            const int page = page_of(bt, kv, b, j0 + i);
            o = __builtin_fmaf(p, static_cast<float>((reinterpret_cast<const TC*>(kv.v) + elem_of(kv, page, j0 + i, kh))[tid]), o);
          }
        }
      }
      __syncthreads();
    }
  }
  if (tid < hd) out[row * out_stride + h * hd + tid] = static_cast<TI>(z == 0.0f ? 0.0f : o / z);
  if (mz && tid == 0) mz[static_cast<int64_t>(row) * n_heads + h] = make_float2(m, z);
}

// weight of a position: a lane sums its shares over the rows and heads, in order.
template <typename TC, typename TI>
__global__ void __launch_bounds__(256) k_paged_weight(PagedView kv, BatchView bt, RuleView rl, const TI* __restrict__ q,
                                                      int64_t q_stride, int n_heads, const float2* __restrict__ mz) {
  const int j = blockIdx.x * 256 + threadIdx.x, kh = blockIdx.y, b = blockIdx.z, hd = kv.hd;
  const int len = seq_len(bt, kv, b), G = n_heads / kv.n_kv_heads;
  const SeqRows sr = seq_rows(bt, b);
  if (j >= len) return;
  const int page = page_of(bt, kv, b, j);
  if (page < 0) return;
  const TC* k = reinterpret_cast<const TC*>(kv.k) + elem_of(kv, page, j, kh);
  float sum = 0.0f;
  for (int t = 0; t < sr.n; ++t) {
    const int pos = len - sr.given + t;
    if (pos < 0) continue;
    const RowRule rr = row_rule(rl, b, pos);
    if (!seen(rl, rr, j)) continue;
    for (int h = kh * G; h < kh * G + G; ++h) {
      const int64_t row = sr.r0 + t;
      float a = 0.0f;
      for (int d = 0; d < hd; ++d) a = __builtin_fmaf(static_cast<float>(q[row * q_stride + h * hd + d]), static_cast<float>(k[d]), a);
      const float2 r = mz[row * n_heads + h];
      if (r.y != 0.0f) sum += expf(rule_score(rl, rl.slopes ? rl.slopes[h] : 0.0f, a, pos, j) - r.x) / r.y;
    }
  }
  *weight_of(kv, page, j, kh) += sum;
}

template <typename TC, typename TI>
hipError_t attention(const PagedView& kv, const BatchView& bt, const RuleView& rl, void* out, int64_t out_stride,
                     const void* q, int64_t q_stride, int n_heads, void* scratch, hipStream_t s) {
  float2* mz = kv.weight ? static_cast<float2*>(scratch) : nullptr;
  hipLaunchKernelGGL((k_paged_attention<TC, TI>), dim3(n_heads, bt.max_new, bt.n_seq), dim3(256), 0, s, kv, bt, rl,
                     static_cast<TI*>(out), out_stride, static_cast<const TI*>(q), q_stride, n_heads, mz);
  if (hipError_t e = hipGetLastError(); e != hipSuccess || !mz) return e;
  hipLaunchKernelGGL((k_paged_weight<TC, TI>), dim3((bt.max_len + 255) / 256, kv.n_kv_heads, bt.n_seq), dim3(256), 0, s,
                     kv, bt, rl, static_cast<const TI*>(q), q_stride, n_heads, mz);
  return hipGetLastError();
}

}  // namespace

size_t paged_attention_scratch(const PagedView& kv, const BatchView& bt, int n_heads, int) {
  return kv.weight ? static_cast<size_t>(bt.n_rows) * n_heads * sizeof(float2) : 0;
}

hipError_t launch_paged_attention(const PagedView& kv, int kv_type, const BatchView& bt, const RuleView& rl, int io_type,
                                  void* out, int64_t out_stride, const void* q, int64_t q_stride, int n_heads,
                                  void* scratch, int, hipStream_t s) {
  const bool f32 = io_type == MCPM_TYPE_F32;
  if (kv_type == MCPM_TYPE_F32) return attention<float, float>(kv, bt, rl, out, out_stride, q, q_stride, n_heads, scratch, s);
  if (kv_type == MCPM_TYPE_F16)
    return f32 ? attention<_Float16, float>(kv, bt, rl, out, out_stride, q, q_stride, n_heads, scratch, s)
               : attention<_Float16, _Float16>(kv, bt, rl, out, out_stride, q, q_stride, n_heads, scratch, s);
  return f32 ? attention<__bf16, float>(kv, bt, rl, out, out_stride, q, q_stride, n_heads, scratch, s)
             : attention<__bf16, __bf16>(kv, bt, rl, out, out_stride, q, q_stride, n_heads, scratch, s);
}

}  // namespace mcpm
