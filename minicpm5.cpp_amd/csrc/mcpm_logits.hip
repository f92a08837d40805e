// mcpm_logits.hip -- the rules on logits that come before sampling: penalties
// for ids of the history, biases, a mask of allowed ids (mcpm_process_logits).
//
//   c > 0:  l <- (l > 0 ? l / rep : l * rep) - (freq * c + pres)
//   listed: l <- l + bias;   not allowed: l <- -inf
//
// One work group per (sequence, LG_TILE ids): it counts the history's ids that
// fall into its tile and finds the last bias entry of each in LDS (integer
// atomics, so no order of arrival changes a result), then passes once over the
// tile's logits.  No scratch in device memory and one launch.
#include "mcpm_device.h"
#include "mcpm_paged.h"

namespace mcpm {

namespace {

constexpr int LG_TILE = 4096;
constexpr int LG_T = 256;

__global__ void __launch_bounds__(LG_T) k_process_logits(float* __restrict__ logits, const mcpm_logit_rules r) {
  __shared__ unsigned cnt[LG_TILE];
  __shared__ unsigned last[LG_TILE];
  const int b = blockIdx.y, id0 = blockIdx.x * LG_TILE, tid = threadIdx.x;
  const int n = min(LG_TILE, r.vocab - id0);
  for (int i = tid; i < LG_TILE; i += LG_T) cnt[i] = last[i] = 0;
  __syncthreads();
  if (r.history)
    for (int i = r.history_starts[b] + tid; i < r.history_starts[b + 1]; i += LG_T) {
      const unsigned o = static_cast<unsigned>(r.history[i] - id0);
      if (o < static_cast<unsigned>(n)) atomicAdd(&cnt[o], 1u);
    }
  const int b0 = r.bias ? r.bias_starts[b] : 0;
  if (r.bias)
    for (int i = b0 + tid; i < r.bias_starts[b + 1]; i += LG_T) {
      const unsigned o = static_cast<unsigned>(r.bias_ids[i] - id0);
      if (o < static_cast<unsigned>(n)) atomicMax(&last[o], static_cast<unsigned>(i - b0) + 1);
    }
  __syncthreads();
  const float rep = r.repetition ? r.repetition[b] : 1.0f;
  const float pres = r.presence ? r.presence[b] : 0.0f, freq = r.frequency ? r.frequency[b] : 0.0f;
  float* row = logits + b * r.stride + id0;
  const uint32_t* ok = r.allowed ? r.allowed + b * r.allowed_stride + id0 / 32 : nullptr;
  for (int i = tid; i < n; i += LG_T) {
    float l = row[i];
    const unsigned c = cnt[i], e = last[i];
    if (c) l = (l > 0.0f ? l / rep : l * rep) - (freq * static_cast<float>(c) + pres);
    if (e) l += r.bias[b0 + e - 1];
    if (ok && !((ok[i >> 5] >> (i & 31)) & 1)) l = -__builtin_inff();
    row[i] = l;
  }
}

}  // namespace

hipError_t launch_process_logits(float* logits, const mcpm_logit_rules& r, hipStream_t s) {
  hipLaunchKernelGGL(k_process_logits, dim3((r.vocab + LG_TILE - 1) / LG_TILE, r.n_seq), dim3(LG_T), 0, s, logits, r);
  return hipGetLastError();
}

}  // namespace mcpm
